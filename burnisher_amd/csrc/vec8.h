// Eight neighbouring values of a row, the unit that the kernels of whole rows load and store.
#pragma once

#include "common.h"

namespace bh {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(bf16_t v) { return bf2f(v); }

// Eight values at column `col` of a row (its address `p` is that of `col`), zero from column `cols` on. Memory takes 16 bytes
// at the alignment of a value, so rows of any stride load alike (8192 x 4607 bf16: 27 us, value by value 52).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t col, int64_t cols, float (&v)[8]) {
    if (col + 8 <= cols) {
        if constexpr (sizeof(T) == 2) {
            typedef u32x4_t Any __attribute__((aligned(2)));
            const u32x4_t w = *reinterpret_cast<const Any*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
            typedef f32x4_t Any __attribute__((aligned(4)));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f32x4_t r = *reinterpret_cast<const Any*>(p + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * i + e] = r[e];
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = col + e < cols ? value(p[e]) : 0.0f;
}

// Eight values as they lie in memory until they are used (four registers of bf16, eight of fp32), at any alignment.
template <typename T>
struct Packed8 {
    static constexpr int kWords = sizeof(T) == 2 ? 4 : 8;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* p) {
        typedef u32x4_t Any __attribute__((aligned(2)));
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const u32x4_t r = reinterpret_cast<const Any*>(p)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * i + e] = r[e];
        }
    }
    // The last 8 - skip of a row of fewer than eight values, p where the first would be.
    __device__ __forceinline__ void load_from(const T* p, int skip) {
        uint32_t bits[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (sizeof(T) == 2) bits[e] = e >= skip ? p[e] : 0u;
            else bits[e] = e >= skip ? __float_as_uint(p[e]) : 0u;
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = sizeof(T) == 2 ? bits[2 * i % 8] | bits[(2 * i + 1) % 8] << 16 : bits[i];
    }
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        else return __uint_as_float(w[e]);
    }
};

// Those of columns below `cols`, each rounded once.
template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t col, int64_t cols, const float (&v)[8]) {
    if (col + 8 <= cols) {
        if constexpr (sizeof(T) == 2) {
            typedef u32x4_t Any __attribute__((aligned(2)));
            *reinterpret_cast<Any*>(p) = u32x4_t{f2bf2(v[0], v[1]), f2bf2(v[2], v[3]), f2bf2(v[4], v[5]), f2bf2(v[6], v[7])};
        } else {
            typedef f32x4_t Any __attribute__((aligned(4)));
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<Any*>(p + 4 * i) = f32x4_t{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + e < cols) {
            if constexpr (sizeof(T) == 2) p[e] = f2bf(v[e]);
            else p[e] = v[e];
        }
}

}  // namespace bh
