// The matrix product of two e4m3 matrices with a scale per block of 128 along K:
//   out[m, n] = act(sum over blocks j of sa[j, m] * sb[n / 128, j] * sum over k in block j of A[m, k] B[n, k] + bias[n])
// Rows of A and B are fp8_row_bytes(k) apart, zero from k on.
#include "common.h"

namespace bh {
namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

struct Fp8Args {
    const uint8_t* a;
    const float* sa;     // [blocks, m]
    const uint8_t* b;
    const float* sb;     // [n / 128, blocks]
    const void* bias;    // [n] in the output's type, or null
    void* out;           // [m, n]
    int64_t m, n, ld;    // ld: row bytes of a and b
    int blocks;
    int act;
};

__device__ __forceinline__ float ld_out(const float* p) { return *p; }
__device__ __forceinline__ float ld_out(const bf16_t* p) { return bf2f(*p); }
__device__ __forceinline__ void st_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void st_out(bf16_t* p, float v) { *p = f2bf(v); }

// gelu-tanh as x / (1 + exp(-2u)) and SiLU: both keep their relative accuracy where the result is tiny.
__device__ __forceinline__ float activate(float x, int act) {
    if (act == 1) {
        const float u = 0.7978845608028654f * (x + 0.044715f * x * x * x);
        return x / (1.0f + expf(-2.0f * u));
    }
    if (act == 2) return x / (1.0f + expf(-x));
    return x;
}

// Sixteen codes (16 bytes) as two bf16 operands: every e4m3 value is a bf16 value.
__device__ __forceinline__ void widen16(const uint4& c, bf16x8_t (&f)[2]) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, false);
        const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, true);
        bf16x8_t& d = f[i >> 1];
        const int o = (i & 1) * 4;
        d[o] = lo[0]; d[o + 1] = lo[1]; d[o + 2] = hi[0]; d[o + 3] = hi[1];
    }
}

// The product of one block of 128: lane (l, h) = (lane % 16, lane / 16) holds the same 32 of the block's
// columns of row l of either operand (`x0`, `x1`), so their order within the block does not matter.
// EXACT: through bf16 operands, whose products and sums are fp32; otherwise through the 8-bit matrix
// instruction.
template <bool EXACT>
__device__ __forceinline__ f32x4_t block_product(const uint4& x0, const uint4& x1, const uint4& y0, const uint4& y1) {
    f32x4_t d = {0.f, 0.f, 0.f, 0.f};
    if constexpr (EXACT) {
        bf16x8_t x[2], y[2];
        widen16(x0, x);
        widen16(y0, y);
#pragma unroll
        for (int i = 0; i < 2; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], y[i], d, 0, 0, 0);
        widen16(x1, x);
        widen16(y1, y);
#pragma unroll
        for (int i = 0; i < 2; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], y[i], d, 0, 0, 0);
    } else {
        const i32x8_t x = {static_cast<int>(x0.x), static_cast<int>(x0.y), static_cast<int>(x0.z), static_cast<int>(x0.w),
                           static_cast<int>(x1.x), static_cast<int>(x1.y), static_cast<int>(x1.z), static_cast<int>(x1.w)};
        const i32x8_t y = {static_cast<int>(y0.x), static_cast<int>(y0.y), static_cast<int>(y0.z), static_cast<int>(y0.w),
                           static_cast<int>(y1.x), static_cast<int>(y1.y), static_cast<int>(y1.z), static_cast<int>(y1.w)};
        d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, d, 0, 0, 0, 0, 0, 0);
    }
    return d;
}

// 16 bytes of a row at `off`, zeros past the row's end.
__device__ __forceinline__ uint4 chunk(const uint8_t* row, int64_t off, int64_t ld) {
    return off < ld ? *reinterpret_cast<const uint4*>(row + off) : make_uint4(0, 0, 0, 0);
}

// Workgroup: 16 columns x 16 MT rows; its waves take every kWaves-th block of K and their sums meet in LDS.
constexpr int kWaves = 8;

template <int MT, bool EXACT, typename OUT>
__global__ void __launch_bounds__(kWaves * 64) k_gemm_fp8_rows(Fp8Args a) {
    __shared__ float part[kWaves][MT][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, h = lane >> 4;
    const int64_t tiles_n = (a.n + 15) / 16;
    const int64_t n0 = blockIdx.x % tiles_n * 16, m0 = blockIdx.x / tiles_n * 16 * MT;
    const uint8_t* brow = a.b + min(n0 + l, a.n - 1) * a.ld;
    const float* sb = a.sb + n0 / 128 * a.blocks;
    int64_t m[MT];
    f32x4_t acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        m[i] = min(m0 + i * 16 + l, a.m - 1);
        acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    for (int j = wave; j < a.blocks; j += kWaves) {
        const int64_t off = static_cast<int64_t>(j) * 128 + h * 32;
        const uint4 b0 = chunk(brow, off, a.ld), b1 = chunk(brow, off + 16, a.ld);
        const float s = sb[j];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint8_t* arow = a.a + m[i] * a.ld;
            const f32x4_t d = block_product<EXACT>(b0, b1, chunk(arow, off, a.ld), chunk(arow, off + 16, a.ld));
            const float sc = s * a.sa[j * a.m + m[i]];
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[i][t] = __builtin_fmaf(d[t], sc, acc[i][t]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)   // lane (l, h): columns 4h .. 4h + 3 of row l
#pragma unroll
        for (int t = 0; t < 4; ++t) part[wave][i][l][h * 4 + t] = acc[i][t];
    __syncthreads();
    OUT* out = static_cast<OUT*>(a.out);
    const OUT* bias = static_cast<const OUT*>(a.bias);
    for (int e = threadIdx.x; e < MT * 256; e += kWaves * 64) {
        const int i = e >> 8, r = (e >> 4) & 15, c = e & 15;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v += part[w][i][r][c];
        const int64_t row = m0 + i * 16 + r, col = n0 + c;
        if (row >= a.m || col >= a.n) continue;
        if (bias) v += ld_out(bias + col);
        st_out(out + row * a.n + col, activate(v, a.act));
    }
}

}  // namespace

int64_t gemm_fp8_workspace_floats(int64_t, int64_t, int64_t) { return 0; }

void launch_gemm_fp8(const uint8_t* a, const float* sa, const uint8_t* b, const float* sb, const void* bias, void* out,
                     int64_t m, int64_t n, int64_t k, int act, bool f32, float*, int64_t, hipStream_t s) {
    Fp8Args p{a, sa, b, sb, bias, out, m, n, fp8_row_bytes(k), static_cast<int>((k + 127) / 128), act};
    ProfileScope ps(K_GEMM, s, 2.0 * m * n * k);
    const int mt = m > 32 ? 4 : m > 16 ? 2 : 1;
    const int64_t grid = (n + 15) / 16 * ((m + 16 * mt - 1) / (16 * mt));
    require(grid < (int64_t{1} << 31), "gemm_fp8: the output is too large");
    auto launch = [&](void (*kernel)(Fp8Args)) { kernel<<<static_cast<unsigned>(grid), kWaves * 64, 0, s>>>(p); };
    if (mt == 1) launch(f32 ? &k_gemm_fp8_rows<1, true, float> : &k_gemm_fp8_rows<1, false, bf16_t>);
    else if (mt == 2) launch(f32 ? &k_gemm_fp8_rows<2, true, float> : &k_gemm_fp8_rows<2, false, bf16_t>);
    else launch(f32 ? &k_gemm_fp8_rows<4, true, float> : &k_gemm_fp8_rows<4, false, bf16_t>);
    launch_check("gemm_fp8");
}

}  // namespace bh
