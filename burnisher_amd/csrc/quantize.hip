// Quantising a matrix to 8-bit floating point (e4m3), one fp32 scale per block of 128 values of a row
// (activations) or per 128 x 128 block (weights):
//   scale = max(amax, 2^-96) / 448,  code = e4m3(x * (448 / max(amax, 2^-96))),  amax = max |x| of the block.
// 448 is e4m3's largest value, so a block's largest magnitude becomes +-448. The scale and the factor
// are each one IEEE division, the product is rounded to fp32 and then to e4m3 (to nearest even): the
// second rounding is the format's, half an e4m3 step (2^-4 of the value); the first moves a value by
// 2^-24 and matters at a tie only. The floor keeps the factor finite for a block of zeros, whose codes
// are zeros. A block that holds an infinity or a NaN gets that as its scale (the maximum is taken over
// the magnitudes' bits, where both lie above every finite value), so whatever is multiplied with it
// becomes NaN instead of a finite wrong number.
//
// Bound by HBM: each value is read once into registers, where the maximum is found before the codes
// are written. Measured (call to call): 128 x 128 blocks of a 10240 x 4096 fp32 matrix 38.7 us, 5.4 TB/s;
// rows of a 600 x 10240 bf16 matrix 6.0 us, 18.8 MB at 3.1 TB/s, of which a launch is 3.5; one row of 4096
// 5.2 us, the call itself.
#include "common.h"
#include "vec8.h"

#include <algorithm>

namespace bh {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr uint32_t kAmaxFloorBits = 0x0f800000u;   // 2^-96
constexpr int kThreads = 256;

// The magnitudes' largest bit pattern of eight values (NaN above infinity above the finite ones).
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
    return m;
}

// Over the 16 lanes of a row's block.
__device__ __forceinline__ uint32_t max16(uint32_t m) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), d, 64)));
    return m;
}

// The codes of eight values from column `col`; columns from `cols` on are zero whatever the factor.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float factor, int64_t col, int64_t cols) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float* f = v + 4 * h;
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * factor, f[1] * factor, 0, false);
        w[h] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[2] * factor, f[3] * factor, r, true));
    }
    if (col + 8 > cols) {
        const int64_t keep = max(cols - col, static_cast<int64_t>(0)) * 8;   // bits
        w[0] = keep >= 32 ? w[0] : w[0] & ((1u << keep) - 1);
        w[1] = keep <= 32 ? 0 : w[1] & ((1u << (keep - 32)) - 1);
    }
    return make_uint2(w[0], w[1]);
}

// Workgroup: 16 rows x 512 columns. A wave takes four rows, its 64 lanes a row's 512 columns (eight
// values each, 16 lanes a block), all four rows' loads before the first maximum. The scales are laid
// out [block of columns, row] and leave through LDS, 16 consecutive rows a block.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_quantize_rows(const T* __restrict__ x, int64_t ld, uint8_t* __restrict__ q,
                                                            int64_t ld_q, float* __restrict__ scales, int64_t rows,
                                                            int64_t cols, int64_t col_blocks) {
    __shared__ float s[4][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int64_t id = group_index(), cb = id % col_blocks, r0 = id / col_blocks * 16;
    if (r0 >= rows) return;
    const int64_t col = cb * 512 + lane * 8;
    float v[4][8];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t row = r0 + wave * 4 + r;
        const int64_t lim = row < rows ? cols : 0;
        load8<T>(x + min(row, rows - 1) * ld + col, col, lim, v[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t row = r0 + wave * 4 + r;
        const float amax = __uint_as_float(max(max16(amax8(v[r])), kAmaxFloorBits));
        if (row < rows && col < ld_q)
            *reinterpret_cast<uint2*>(q + row * ld_q + col) = codes8(v[r], __fdiv_rn(kE4m3Max, amax), col, cols);
        if ((lane & 15) == 0) s[g][wave * 4 + r] = __fdiv_rn(amax, kE4m3Max);
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (t < 64) {
        const int64_t block = cb * 4 + (t >> 4), row = r0 + (t & 15);
        if (row < rows && block * 128 < cols) scales[block * rows + row] = s[t >> 4][t & 15];
    }
}

// Workgroup: one 128 x 128 block, 64 values a thread in registers.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_quantize_blocks(const T* __restrict__ x, int64_t ld, uint8_t* __restrict__ q,
                                                              int64_t ld_q, float* __restrict__ scales, int64_t rows,
                                                              int64_t cols, int64_t col_blocks) {
    __shared__ uint32_t s[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t id = group_index(), cb = id % col_blocks, rb = id / col_blocks;
    if (rb * 128 >= rows) return;
    const int64_t col = cb * 128 + (lane & 15) * 8, row0 = rb * 128 + wave * 4 + (lane >> 4);
    float v[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int64_t row = row0 + p * 16;
        load8<T>(x + min(row, rows - 1) * ld + col, col, row < rows ? cols : 0, v[p]);
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) m = max(m, amax8(v[p]));
    m = max16(m);
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16, 64)));
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32, 64)));
    if (lane == 0) s[wave] = m;
    __syncthreads();
    const float amax = __uint_as_float(max(max(max(s[0], s[1]), max(s[2], s[3])), kAmaxFloorBits));
    const float factor = __fdiv_rn(kE4m3Max, amax);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int64_t row = row0 + p * 16;
        if (row < rows && col < ld_q) *reinterpret_cast<uint2*>(q + row * ld_q + col) = codes8(v[p], factor, col, cols);
    }
    if (threadIdx.x == 0) scales[rb * col_blocks + cb] = __fdiv_rn(amax, kE4m3Max);
}

template <typename T>
void quantize(const T* x, int64_t ld, uint8_t* q, float* scales, int64_t rows, int64_t cols, bool blocks, hipStream_t s) {
    const int64_t ld_q = fp8_row_bytes(cols);
    const int64_t col_blocks = blocks ? (cols + 127) / 128 : (cols + 511) / 512;
    const int64_t grid = col_blocks * (blocks ? (rows + 127) / 128 : (rows + 15) / 16);
    require(grid < (int64_t{1} << 31), "quantize_fp8: the matrix is too large");
    auto* kernel = blocks ? &k_quantize_blocks<T> : &k_quantize_rows<T>;
    kernel<<<grid_of(grid, kThreads), kThreads, 0, s>>>(x, ld, q, ld_q, scales, rows, cols, col_blocks);
    launch_check("quantize_fp8");
}

}  // namespace

void launch_quantize_fp8(const void* x, int64_t ld, uint8_t* q, float* scales, int64_t rows, int64_t cols, bool blocks,
                         bool f32, hipStream_t s) {
    if (f32) quantize(static_cast<const float*>(x), ld, q, scales, rows, cols, blocks, s);
    else quantize(static_cast<const bf16_t*>(x), ld, q, scales, rows, cols, blocks, s);
}

}  // namespace bh
