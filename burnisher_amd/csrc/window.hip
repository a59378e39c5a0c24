// Sliding-window attention with first tokens that stay visible, over grouped heads:
//   out[b, i, h] = sum_j softmax_j(scale * q[b, i, h] . k[b, j, h / group]) v[b, j, h / group]
// over the keys j < kv_lens[b] that query i, at position p = q_starts[b] + i, sees:
//   j <= p + right and (j >= p - left or j < sinks).
// A query that sees no key gives zeros.
//
// The heads of a group read the same keys, so they are rows of one tile: row r of (batch row, key head)
// is token r / group, head r % group of the group, and rows of one tile share a narrow window. The
// workgroup walks the keys that one of its rows sees and no others: whole blocks outside are never
// loaded, and of a block's 64 keys those that no row sees are replaced by one that is seen, so what lies
// there (the unwritten end of a cache, a NaN) never enters a product.
//
// Both products run on v_mfma_f32_16x16x32_bf16 in transposed tiles, S^T = K Q^T and O^T += V^T P^T: two
// accumulator tiles of the first are one operand of the second, and V^T comes out of row-major V by the
// transposing LDS read, which gives a lane four keys of one column.
#include "common.h"

#include <algorithm>
#include <cmath>

namespace bh {
namespace {

constexpr int kThreads = 256;
constexpr int kKeys = 64;      // keys per block
constexpr float kLog2e = 1.4426950408889634f;

typedef __attribute__((address_space(3))) const char* lds_ptr;
typedef short s16x4_t __attribute__((ext_vector_type(4)));

struct WindowArgs {
    const bf16_t* q;
    const bf16_t* k;
    const bf16_t* v;
    bf16_t* out;
    const int32_t* kv_lens;
    const int32_t* q_starts;
    int64_t ld_q, ld_kv, ld_o;
    int B, H, KH, group, Sq, Skv, D;
    int left, right, sinks;
    int tiles;    // row tiles per (batch row, key head)
    float c;      // scale * log2(e)
};

// Four keys of column (lane % 16), keys 4 (lane / 16) .. + 3 of a 16-key tile: lane i of a 16-lane group
// passes the address of columns 4 (i % 4) .. + 3 of key i / 4.
__device__ __forceinline__ s16x4_t read_transposed(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(reinterpret_cast<uintptr_t>((lds_ptr)p)));
}

template <int DT>
__global__ void __launch_bounds__(kThreads) k_window(WindowArgs a) {
    constexpr int KS = (DT + 1) / 2;              // K = 32 steps of the score product
    constexpr int kPitch = DT * 32 + 16;          // LDS bytes of a key
    constexpr int kChunks = DT * 2;               // 16-byte chunks of a key
    __shared__ __attribute__((aligned(16))) char smem[2 * kKeys * kPitch];
    char* ks_ = smem;
    char* vs_ = smem + kKeys * kPitch;

    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, c16 = lane & 15;
    const int tile = blockIdx.x % a.tiles, bk = blockIdx.x / a.tiles, kh = bk % a.KH, b = bk / a.KH;
    const int rows = a.group * a.Sq;
    const int r0 = tile * 64, r1 = min(r0 + 64, rows) - 1;

    const int64_t len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.Skv) : a.Skv;
    const int64_t start = a.q_starts ? a.q_starts[b] : a.Skv - a.Sq;
    // the keys that some row of the tile sees: [0, near) and [lo, hi)
    const int64_t p0 = start + r0 / a.group, p1 = start + r1 / a.group;
    const int64_t hi = max(min(len, a.right < 0 ? len : p1 + a.right + 1), int64_t{0});
    int64_t lo = a.left < 0 ? 0 : min(max(p0 - a.left, int64_t{0}), hi);
    const int64_t near = min(static_cast<int64_t>(a.sinks), lo);
    const int nb1 = static_cast<int>((near + kKeys - 1) / kKeys), nb = nb1 + static_cast<int>((hi - lo + kKeys - 1) / kKeys);

    const int row = r0 + wave * 16 + c16;          // this lane's query
    const int64_t pos = start + min(row, rows - 1) / a.group;
    const int64_t see_hi = min(hi, a.right < 0 ? hi : pos + a.right + 1), see_lo = a.left < 0 ? 0 : pos - a.left;
    const int head = kh * a.group + min(row, rows - 1) % a.group;
    const int64_t token = static_cast<int64_t>(b) * a.Sq + min(row, rows - 1) / a.group;

    bf16x8_t qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int d0 = ks * 32 + g * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[ks][e] = static_cast<__bf16>(0.0f);
        if (d0 < a.D) qf[ks] = *reinterpret_cast<const bf16x8_t*>(a.q + token * a.ld_q + static_cast<int64_t>(head) * a.D + d0);
    }
    f32x4_t o[DT];
#pragma unroll
    for (int e = 0; e < DT; ++e) o[e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float row_max = -3.4028235e38f, row_sum = 0.f;   // finite, so that a masked score's weight is exp2(-inf) = 0

    for (int j = 0; j < nb; ++j) {
        const int64_t base = j < nb1 ? static_cast<int64_t>(j) * kKeys : lo + static_cast<int64_t>(j - nb1) * kKeys;
        const int64_t end = j < nb1 ? near : hi;
        __syncthreads();
        for (int i = tid; i < kKeys * kChunks; i += kThreads) {
            const int key = i / kChunks, ch = i % kChunks;
            const int64_t off = (static_cast<int64_t>(b) * a.Skv + min(base + key, end - 1)) * a.ld_kv +
                                static_cast<int64_t>(kh) * a.D + ch * 8;
            uint4 rk = make_uint4(0, 0, 0, 0), rv = rk;
            if (ch * 8 < a.D) {
                rk = *reinterpret_cast<const uint4*>(a.k + off);
                rv = *reinterpret_cast<const uint4*>(a.v + off);
            }
            *reinterpret_cast<uint4*>(ks_ + key * kPitch + ch * 16) = rk;
            *reinterpret_cast<uint4*>(vs_ + key * kPitch + ch * 16) = rv;
        }
        __syncthreads();
        // S^T: s[t] holds keys base + 16 t + 4 g + r of this lane's query
        f32x4_t s[4];
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8_t kf;
#pragma unroll
                for (int e = 0; e < 8; ++e) kf[e] = static_cast<__bf16>(0.0f);
                if (ks * 32 + g * 8 < DT * 16)
                    kf = *reinterpret_cast<const bf16x8_t*>(ks_ + (t * 16 + c16) * kPitch + ks * 64 + g * 16);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[ks], s[t], 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t kv = base + t * 16 + g * 4 + r;
                const bool seen = kv < end && kv < see_hi && (kv >= see_lo || kv < a.sinks);
                s[t][r] = seen ? s[t][r] * a.c : -INFINITY;
                mx = fmaxf(mx, s[t][r]);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(row_max, mx), alpha = exp2f(row_max - m_new);
        row_max = m_new;
        row_sum *= alpha;
#pragma unroll
        for (int e = 0; e < DT; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[e][r] *= alpha;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float p = exp2f(s[t][r] - m_new);
                row_sum += p;
                s[t][r] = p;
            }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            bf16x8_t pf;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pf[r] = static_cast<__bf16>(s[2 * c][r]);
                pf[4 + r] = static_cast<__bf16>(s[2 * c + 1][r]);
            }
            const char* vrow = vs_ + (c * 32 + g * 4 + (c16 >> 2)) * kPitch + (c16 & 3) * 8;
#pragma unroll
            for (int e = 0; e < DT; ++e) {
                const s16x4_t v0 = read_transposed(vrow + e * 32), v1 = read_transposed(vrow + 16 * kPitch + e * 32);
                typedef short s16x8_t __attribute__((ext_vector_type(8)));
                const s16x8_t vv = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vv), pf, o[e], 0, 0, 0);
            }
        }
    }
    row_sum += __shfl_xor(row_sum, 16, 64);
    row_sum += __shfl_xor(row_sum, 32, 64);
    if (row >= rows) return;
    const float rl = row_sum == 0.f ? 0.f : 1.0f / row_sum;
    bf16_t* dst = a.out + token * a.ld_o + static_cast<int64_t>(head) * a.D;
#pragma unroll
    for (int e = 0; e < DT; ++e) {
        const int d = e * 16 + g * 4;
        if (d >= a.D) continue;
        const uint2 w = make_uint2(f2bf2(o[e][0] * rl, o[e][1] * rl), f2bf2(o[e][2] * rl, o[e][3] * rl));
        *reinterpret_cast<uint2*>(dst + d) = w;
    }
}

}  // namespace

int64_t attention_window_workspace_floats(const WindowShape&) { return 0; }

void launch_attention_window(const bf16_t* q, const bf16_t* k, const bf16_t* v, bf16_t* out, const WindowShape& sh,
                             const int32_t* kv_lens, const int32_t* q_starts, float*, int64_t, hipStream_t s) {
    WindowArgs a;
    a.q = q; a.k = k; a.v = v; a.out = out;
    a.kv_lens = kv_lens; a.q_starts = q_starts;
    a.ld_q = sh.ld_q; a.ld_kv = sh.ld_kv; a.ld_o = sh.ld_o;
    a.B = static_cast<int>(sh.batch); a.H = static_cast<int>(sh.heads); a.KH = static_cast<int>(sh.kv_heads);
    a.group = a.H / a.KH;
    a.Sq = static_cast<int>(sh.q_len); a.Skv = static_cast<int>(sh.kv_len); a.D = static_cast<int>(sh.head_dim);
    a.left = sh.left; a.right = sh.right; a.sinks = sh.sinks;
    a.c = sh.scale * kLog2e;
    const int64_t rows = static_cast<int64_t>(a.group) * a.Sq, tiles = (rows + 63) / 64;
    a.tiles = static_cast<int>(tiles);
    const int64_t grid = tiles * a.B * a.KH;
    const unsigned gr = static_cast<unsigned>(grid);
    const int dt = (a.D + 15) / 16;
    ProfileScope ps(sh.q_len == sh.kv_len ? K_ATTN_SELF : K_ATTN_CROSS, s, 0);
    if (dt <= 2) k_window<2><<<gr, kThreads, 0, s>>>(a);
    else if (dt <= 4) k_window<4><<<gr, kThreads, 0, s>>>(a);
    else if (dt <= 5) k_window<5><<<gr, kThreads, 0, s>>>(a);
    else if (dt <= 6) k_window<6><<<gr, kThreads, 0, s>>>(a);
    else k_window<8><<<gr, kThreads, 0, s>>>(a);
    launch_check("attention_window");
}

}  // namespace bh
