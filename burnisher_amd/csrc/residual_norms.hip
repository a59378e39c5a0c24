// The norm of a block's output, its gate and scale into the residual stream, and the norm before the next block:
//   n = post(x),  r = residual_scale * residual + branch_scale * gate * n,  out = pre(r) * (1 + scale) + shift.
// One pass: a row's values stay in registers from their load to their last use, both norms' statistics included, so x and
// residual are read once and r and out written once. Statistics are fp32; a variance is the mean square of the
// differences to the mean, in a second pass over the registers, so a large mean costs no digits. r goes into the
// second norm before it is rounded.
//
// Bound by HBM.
#include "common.h"
#include "vec8.h"

#include <algorithm>

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
    bh_residual_norms f;
};

// Sum over the threads of a row.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    if constexpr (THREADS > 64) {
        constexpr int kWaves = THREADS / 64;
        __syncthreads();   // the last sum has been read
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += slot[w];
    }
    return v;
}

// norm(v) * (offset + weight) + bias, in place; columns from `cols` on are zeros and stay out of the sums.
template <typename T, int THREADS, int V>
__device__ __forceinline__ void norm(float (&v)[V][8], int kind, const void* weight, const void* bias, float eps, float offset,
                                     int cols, int thread, float* slot) {
    if (kind == BH_NORM_NONE) return;
    if (kind == BH_NORM_LAYER) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += v[i][e];
        const float mean = row_sum<THREADS>(sum, slot) / cols;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = (i * THREADS + thread) * 8 + e < cols ? v[i][e] - mean : 0.f;
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(v[i][e], v[i][e], sum);
    const float inv = 1.0f / sqrtf(row_sum<THREADS>(sum, slot) / cols + eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int col = (i * THREADS + thread) * 8;
        if (col >= cols) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= inv;
        if (weight) {
            float w[8];
            load8(static_cast<const T*>(weight) + col, col, cols, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] *= offset + w[e];
        }
        if (bias) {
            float b[8];
            load8(static_cast<const T*>(bias) + col, col, cols, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] += b[e];
        }
    }
}

template <typename T, typename R, int THREADS, int V>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) k_residual_norms(NormsArgs a) {
    __shared__ float slot[16];
    constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
    const int thread = threadIdx.x % THREADS;
    const int64_t row = group_index() * kRows + threadIdx.x / THREADS;
    if (row >= a.rows) return;
    float x[V][8], r[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int col = (i * THREADS + thread) * 8;
        load8(static_cast<const T*>(a.x) + row * a.ld_x + col, col, a.cols, x[i]);
        load8(static_cast<const R*>(a.residual) + row * a.ld_res + col, col, a.cols, r[i]);
    }
    const bh_residual_norms& f = a.f;
    const bool modulated = f.gate || f.scale || f.shift;
    const int64_t mod = modulated ? row / f.mod_rows * f.ld_mod : 0;
    norm<T, THREADS, V>(x, f.post_norm, f.post_weight, f.post_bias, f.post_eps, f.weight_offset, a.cols, thread, slot);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int col = (i * THREADS + thread) * 8;
        if (col >= a.cols) continue;
        if (f.gate) {
            float g[8];
            load8(static_cast<const T*>(f.gate) + mod + col, col, a.cols, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] *= g[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) r[i][e] = __builtin_fmaf(f.branch_scale, x[i][e], f.residual_scale * r[i][e]);
        if (a.residual_out) store8(static_cast<R*>(a.residual_out) + row * a.ld_res_out + col, col, a.cols, r[i]);
        if (col + 8 > a.cols)
#pragma unroll
            for (int e = 0; e < 8; ++e) r[i][e] = col + e < a.cols ? r[i][e] : 0.f;
    }
    if (!a.out) return;
    norm<T, THREADS, V>(r, f.pre_norm, f.pre_weight, f.pre_bias, f.pre_eps, f.weight_offset, a.cols, thread, slot);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int col = (i * THREADS + thread) * 8;
        if (col >= a.cols) continue;
        float m[8];
        if (f.scale) {
            load8(static_cast<const T*>(f.scale) + mod + col, col, a.cols, m);
#pragma unroll
            for (int e = 0; e < 8; ++e) r[i][e] *= 1.0f + m[e];
        }
        if (f.shift) {
            load8(static_cast<const T*>(f.shift) + mod + col, col, a.cols, m);
#pragma unroll
            for (int e = 0; e < 8; ++e) r[i][e] += m[e];
        }
        store8(static_cast<T*>(a.out) + row * a.ld_out + col, col, a.cols, r[i]);
    }
}

template <typename T, typename R, int THREADS, int V>
void launch(const NormsArgs& a, hipStream_t s) {
    constexpr int threads = THREADS < 256 ? 256 : THREADS, rows = threads / THREADS;
    k_residual_norms<T, R, THREADS, V><<<grid_of((a.rows + rows - 1) / rows, threads), threads, 0, s>>>(a);
}

template <typename T, typename R>
void by_width(const NormsArgs& a, hipStream_t s) {
    if (a.cols <= 2048) launch<T, R, 64, 4>(a, s);
    else if (a.cols <= 8192) launch<T, R, 256, 4>(a, s);
    else launch<T, R, 1024, 4>(a, s);
}

}  // namespace

void launch_residual_norms(const void* x, int64_t ld_x, const void* residual, int64_t ld_res, void* residual_out,
                           int64_t ld_res_out, void* out, int64_t ld_out, int64_t rows, int64_t cols,
                           const bh_residual_norms& f, bool residual_f32, bool f32, hipStream_t s) {
    const NormsArgs a{x, residual, residual_out, out, ld_x, ld_res, ld_res_out, ld_out, rows, static_cast<int>(cols), f};
    require(rows < (int64_t{1} << 40), "residual_norms: too many rows");
    if (f32) by_width<float, float>(a, s);
    else if (residual_f32) by_width<bf16_t, float>(a, s);
    else by_width<bf16_t, bf16_t>(a, s);
    launch_check("residual_norms");
}

}  // namespace bh
