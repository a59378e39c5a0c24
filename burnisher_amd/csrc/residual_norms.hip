// The norm of a block's output, its gate and scale into the residual stream, and the norm before the next block:
//   n = post(x),  r = residual_scale * residual + branch_scale * gate * n,  out = pre(r) * (1 + scale) + shift.
// One pass: a row's values stay in registers from their load to their last use, both norms' statistics included, so x and
// residual are read once and r and out written once. Statistics are fp32; a variance is the mean square of the
// differences to the mean, in a second pass over the registers, so a large mean costs no digits. r goes into the
// second norm before it is rounded.
//
// Bound by HBM for wide rows (4096 x 4096 bf16: 29 us, 4.6 TB/s); rows of 1152 columns with gate, scale and shift, 8192 of them
// in 17.6 us (4.3 TB/s), are bound by vector instructions too, 45 an element, which is why a row's address and a
// modulation's row are scalar and no lane has a path of its own. One row of 4096: 3.4 us, a launch.
#include "common.h"
#include "vec8.h"

#include <algorithm>
#include <type_traits>

namespace bh {
namespace {

struct NormsArgs {
    const void* x;
    const void* residual;
    void* residual_out;
    void* out;
    int64_t ld_x, ld_res, ld_res_out, ld_out;
    int64_t rows;
    int cols;
    float each;   // 1 / cols
    bool few;     // rows and mod_rows below 2^32: a 64-bit division cost 2 of 20 us at 8192 x 1152
    bh_residual_norms f;
};

constexpr int kMostWaves = 16;

// Sum over a wave: within 16 lanes by data-parallel moves, then across the four rows of 16.
__device__ __forceinline__ float wave_sum(float v) {
    auto moved = [](float x, auto control) {
        return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(x), decltype(control)::value, 0xf, 0xf, true));
    };
    v += moved(v, std::integral_constant<int, 0xB1>{});    // the neighbour
    v += moved(v, std::integral_constant<int, 0x4E>{});    // the other pair of four
    v += moved(v, std::integral_constant<int, 0x141>{});   // the other four of eight
    v += moved(v, std::integral_constant<int, 0x140>{});   // the other eight of 16
    v += moved(v, std::integral_constant<int, 0x142>{});   // the row of 16 before, into each
    v += moved(v, std::integral_constant<int, 0x143>{});   // the first half's sum, into the second
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// Sum over the `waves` waves of a row; `slot` has a place for each.
__device__ __forceinline__ float row_sum(float v, int waves, float* slot) {
    v = wave_sum(v);
    if (waves == 1) return v;
    __syncthreads();   // the last sum has been read
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
    for (int w = 1; w < waves; ++w) v += slot[w];
    return v;
}

// The columns of a thread's vectors: eight from `col` on, of which the first `skip` are another's. A row's last vector ends with
// the row, so that every load is whole and no lane goes a way of its own (tails loaded value by value: 17.0 us instead of
// 11 for 1155 rows of 2001 fp32 columns); threads past the row take its last vector and own nothing of it.
template <int V>
struct Columns {
    int col[V], skip[V];
    bool ragged;   // rows end inside a vector
    bool tiny;     // a row of fewer than eight columns: col is below zero, and only what is owned may be loaded
    __device__ __forceinline__ Columns(int thread, int threads, int cols) : ragged((cols & 7) != 0), tiny(cols < 8) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int want = (i * threads + thread) * 8;
            col[i] = min(want, cols - 8);
            skip[i] = min(want - col[i], 8);
        }
    }
    template <typename T>
    __device__ __forceinline__ Packed8<T> load(const T* row, int i) const {
        Packed8<T> v;
        if (tiny) v.load_from(row + col[i], skip[i]);
        else v.load(row + col[i]);
        return v;
    }
    template <typename T>
    __device__ __forceinline__ void store(T* row, int i, const float (&v)[8]) const {
        if (skip[i] == 0) {
            store8(row + col[i], 0, 8, v);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e >= skip[i]) {
                if constexpr (sizeof(T) == 2) row[col[i] + e] = f2bf(v[e]);
                else row[col[i] + e] = v[e];
            }
    }
};

// A parameter's columns: with HELD loaded ahead, all of a row's latencies at once, else where they are used. Null: none.
template <typename T, int V, bool HELD>
struct Parameter {
    const T* p;
    const Columns<V>& c;
    Packed8<T> held[HELD ? V : 1];
    __device__ __forceinline__ Parameter(const void* at, int64_t offset, const Columns<V>& columns)
        : p(at ? static_cast<const T*>(at) + offset : nullptr), c(columns) {
        if constexpr (HELD)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (p) held[i] = c.load(p, i);
    }
    __device__ __forceinline__ explicit operator bool() const { return p != nullptr; }
    __device__ __forceinline__ Packed8<T> operator[](int i) const {
        if constexpr (HELD) return held[i];
        else return c.load(p, i);
    }
};

// norm(v) * (offset + weight) + bias, in place; `each` is 1 / columns; what another thread owns is left out of the sums.
template <int V, typename P>
__device__ __forceinline__ void norm(float (&v)[V][8], int kind, const P& weight, const P& bias, float eps, float offset, float each,
                                     const Columns<V>& c, int waves, float* slot) {
    if (kind == BH_NORM_NONE) return;
    // over what the thread owns: all of a vector or nothing where rows are whole vectors
    auto owned = [&](auto term) {
        float sum = 0.f;
        if (c.ragged) {
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = e >= c.skip[i] ? term(v[i][e], sum) : sum;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float part = sum;
#pragma unroll
                for (int e = 0; e < 8; ++e) part = term(v[i][e], part);
                sum = c.skip[i] == 0 ? part : sum;
            }
        }
        return row_sum(sum, waves, slot) * each;
    };
    if (kind == BH_NORM_LAYER) {
        const float mean = owned([](float x, float sum) { return sum + x; });
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] -= mean;
    }
    const float inv = rsqrtf(owned([](float x, float sum) { return __builtin_fmaf(x, x, sum); }) + eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= inv;
        if (weight) {
            const auto w = weight[i];
            if (offset == 0.f)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] *= w[e];
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] *= offset + w[e];
        }
        if (bias) {
            const auto b = bias[i];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] += b[e];
        }
    }
}

// A row to the blockDim.x threads of one y, V times eight columns each; with HELD and V above 1 those are one wave.
template <typename T, typename R, int V, bool HELD>
__global__ void __launch_bounds__(HELD && V > 1 ? 256 : 64 * kMostWaves) k_residual_norms(NormsArgs a) {
    __shared__ float slots[4][kMostWaves];
    const int waves = blockDim.x / 64;
    const int y = __builtin_amdgcn_readfirstlane(threadIdx.y);   // a wave has one row, so its addresses are scalar
    float* slot = slots[y];
    const int64_t number = group_index() * blockDim.y;
    if (number >= a.rows) return;
    const int64_t mine = number + y, row = min(mine, a.rows - 1);   // a row past the last takes part in the barriers
    const bool kept = mine < a.rows;
    const Columns<V> c(threadIdx.x, blockDim.x, a.cols);
    Packed8<T> px[V];
    Packed8<R> pr[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        px[i] = c.load(static_cast<const T*>(a.x) + row * a.ld_x, i);
        pr[i] = c.load(static_cast<const R*>(a.residual) + row * a.ld_res, i);
    }
    const bh_residual_norms& f = a.f;
    const int64_t mod = f.gate || f.scale || f.shift ? (a.few ? static_cast<uint32_t>(row) / static_cast<uint32_t>(f.mod_rows) : row / f.mod_rows) * f.ld_mod : 0;
    using P = Parameter<T, V, HELD>;
    const P post_w(f.post_weight, 0, c), post_b(f.post_bias, 0, c), gate(f.gate, mod, c);
    float x[V][8], r[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = px[i][e];
    norm<V>(x, f.post_norm, post_w, post_b, f.post_eps, f.weight_offset, a.each, c, waves, slot);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (gate) {
            const auto g = gate[i];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] *= g[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) r[i][e] = __builtin_fmaf(f.branch_scale, x[i][e], f.residual_scale * pr[i][e]);
        if (a.residual_out && kept) c.store(static_cast<R*>(a.residual_out) + row * a.ld_res_out, i, r[i]);
    }
    if (!a.out) return;
    const P pre_w(f.pre_weight, 0, c), pre_b(f.pre_bias, 0, c), scale(f.scale, mod, c), shift(f.shift, mod, c);
    norm<V>(r, f.pre_norm, pre_w, pre_b, f.pre_eps, f.weight_offset, a.each, c, waves, slot);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (scale) {
            const auto m = scale[i];
#pragma unroll
            for (int e = 0; e < 8; ++e) r[i][e] *= 1.0f + m[e];
        }
        if (shift) {
            const auto m = shift[i];
#pragma unroll
            for (int e = 0; e < 8; ++e) r[i][e] += m[e];
        }
        if (kept) c.store(static_cast<T*>(a.out) + row * a.ld_out, i, r[i]);
    }
}

template <typename T, typename R, int V, bool HELD>
void launch(const NormsArgs& a, hipStream_t s) {
    const int threads = ((a.cols + 8 * V - 1) / (8 * V) + 63) / 64 * 64, rows = std::max(1, 256 / threads);
    k_residual_norms<T, R, V, HELD><<<grid_of((a.rows + rows - 1) / rows, threads * rows), dim3(threads, rows), 0, s>>>(a);
}

// Rows of up to 1024 columns to a wave, without a barrier (8192 rows of 768 bf16 columns 12.8 us, to two waves 14.1); up to
// 1536 where the stream is bf16 too (1152 columns 17.6, to three waves 19.6; with an fp32 stream the registers of three
// vectors cost more, 1280 columns 27.9 against 27.0); wider ones to as many waves as make a vector each (2048 columns
// 31.8, four vectors of one wave 34.7).
template <typename T, typename R>
void by_width(const NormsArgs& a, hipStream_t s) {
    const int vectors = (a.cols + 7) / 8;
    if (vectors <= 64) return launch<T, R, 1, true>(a, s);
    if (vectors <= 128) return launch<T, R, 2, true>(a, s);
    if constexpr (sizeof(R) == 2)
        if (vectors <= 192) return launch<T, R, 3, true>(a, s);
    if (vectors <= 64 * kMostWaves) return launch<T, R, 1, true>(a, s);
    if (vectors <= 128 * kMostWaves) return launch<T, R, 2, false>(a, s);
    launch<T, R, 4, false>(a, s);
}

}  // namespace

void launch_residual_norms(const void* x, int64_t ld_x, const void* residual, int64_t ld_res, void* residual_out,
                           int64_t ld_res_out, void* out, int64_t ld_out, int64_t rows, int64_t cols,
                           const bh_residual_norms& f, bool residual_f32, bool f32, hipStream_t s) {
    const NormsArgs a{x, residual, residual_out, out, ld_x, ld_res, ld_res_out, ld_out, rows, static_cast<int>(cols), 1.0f / static_cast<float>(cols),
                      rows < (int64_t{1} << 32) && f.mod_rows < (int64_t{1} << 32), f};
    require(rows < (int64_t{1} << 40), "residual_norms: too many rows");
    if (f32) by_width<float, float>(a, s);
    else if (residual_f32) by_width<bf16_t, float>(a, s);
    else by_width<bf16_t, bf16_t>(a, s);
    launch_check("residual_norms");
}

}  // namespace bh
