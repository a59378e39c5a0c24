// Causal linear attention with a decay for each key head:
//   S_t = decay * S_{t-1} + k_t (outer) v_t,  out_t = scale * q_t . S_t.
#include "common.h"

#include <algorithm>
#include <cmath>

namespace bh {
namespace {

constexpr int kThreads = 256;

struct LinearArgs {
    const bf16_t* q;
    const bf16_t* k;
    const bf16_t* v;
    bf16_t* out;
    const float* log_decay;
    const int32_t* lens;
    const float* state_in;
    float* state_out;
    int64_t ld_q, ld_k, ld_v, ld_o;
    int B, H, KH, group, N, D, E;
    int slices;   // of the value columns
    float scale;
};

// A head's log decay: at most 0, and finite, so that no step times it is a NaN.
__device__ __forceinline__ float log_decay_of(const LinearArgs& a, int kh) { return fmaxf(fminf(a.log_decay[kh], 0.f), -1e6f); }

// Times decay^n, log of it `x`. A factor from a half on is applied as S + (decay^n - 1) S, so that one near 1 keeps its
// digits over many steps: rounded itself, it would be off by 2^-25 the same way each time.
struct Fade {
    float by, keep;
    __device__ __forceinline__ explicit Fade(float x) : by(x > -0.69f ? expm1f(x) : expf(x)), keep(x > -0.69f ? 1.f : 0.f) {}
    __device__ __forceinline__ float operator()(float s) const { return __builtin_fmaf(s, by, s * keep); }
};

// Token after token: a workgroup holds 32 columns of a state, thread (d, c) rows d + 32 p, columns 4 c .. 4 c + 3.
__global__ void __launch_bounds__(kThreads) k_linear_tokens(LinearArgs a) {
    __shared__ float part[2][4][32];
    const int64_t number = group_index();
    if (number >= static_cast<int64_t>(a.B) * a.KH * a.slices) return;
    const int slice = static_cast<int>(number % a.slices), kh = static_cast<int>(number / a.slices % a.KH);
    const int64_t b = number / a.slices / a.KH;
    const int wave = threadIdx.x >> 6, d0 = threadIdx.x >> 3, e = slice * 32 + (threadIdx.x & 7) * 4;
    const bool mine = e < a.E;
    const int n = a.lens ? min(max(a.lens[b], 0), a.N) : a.N;
    const Fade fade(log_decay_of(a, kh));
    const int64_t state = (b * a.KH + kh) * a.D * a.E + e;
    f32x4_t s[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int d = d0 + 32 * p;
        s[p] = a.state_in && mine && d < a.D ? *reinterpret_cast<const f32x4_t*>(a.state_in + state + static_cast<int64_t>(d) * a.E)
                                             : f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    int turn = 0;
    for (int t = 0; t < a.N; ++t) {
        const int64_t row = b * a.N + t;
        if (t >= n) {
            if (threadIdx.x < 8 && mine)
                for (int g = 0; g < a.group; ++g)
                    *reinterpret_cast<uint2*>(a.out + row * a.ld_o + static_cast<int64_t>(kh * a.group + g) * a.E + e) = make_uint2(0, 0);
            continue;
        }
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = mine ? bf2f(a.v[row * a.ld_v + static_cast<int64_t>(kh) * a.E + e + c]) : 0.f;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int d = d0 + 32 * p;
            const float k = d < a.D ? bf2f(a.k[row * a.ld_k + static_cast<int64_t>(kh) * a.D + d]) : 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) s[p][c] = __builtin_fmaf(k, v[c], fade(s[p][c]));
        }
        for (int g = 0; g < a.group; ++g, turn ^= 1) {
            const int head = kh * a.group + g;
            f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int d = d0 + 32 * p;
                const float q = d < a.D ? bf2f(a.q[row * a.ld_q + static_cast<int64_t>(head) * a.D + d]) : 0.f;
#pragma unroll
                for (int c = 0; c < 4; ++c) o[c] = __builtin_fmaf(q, s[p][c], o[c]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int x = 8; x < 64; x <<= 1) o[c] += __shfl_xor(o[c], x, 64);
            if ((threadIdx.x & 63) < 8) *reinterpret_cast<f32x4_t*>(&part[turn][wave][(threadIdx.x & 7) * 4]) = o;
            __syncthreads();
            if (threadIdx.x < 8 && mine) {
                f32x4_t total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; ++w) total += *reinterpret_cast<const f32x4_t*>(&part[turn][w][threadIdx.x * 4]);
                *reinterpret_cast<uint2*>(a.out + row * a.ld_o + static_cast<int64_t>(head) * a.E + e) =
                    make_uint2(f2bf2(total[0] * a.scale, total[1] * a.scale), f2bf2(total[2] * a.scale, total[3] * a.scale));
            }
        }
    }
    if (a.state_out && mine)
#pragma unroll
        for (int p = 0; p < 4; ++p)
            if (d0 + 32 * p < a.D) *reinterpret_cast<f32x4_t*>(a.state_out + state + static_cast<int64_t>(d0 + 32 * p) * a.E) = s[p];
}

}  // namespace

int64_t attention_linear_workspace_floats(const LinearShape&) { return 0; }

bh_attention_linear_plan attention_linear_plan(const LinearShape& sh, bool, int) {
    return bh_attention_linear_plan{1, 1, sh.batch * sh.kv_heads * ((sh.value_dim + 31) / 32)};
}

void launch_attention_linear(const bf16_t* q, const bf16_t* k, const bf16_t* v, bf16_t* out, const LinearShape& sh,
                             const float* log_decay, const int32_t* lens, const float* state_in, float* state_out, float*,
                             hipStream_t s) {
    LinearArgs a;
    a.q = q; a.k = k; a.v = v; a.out = out;
    a.log_decay = log_decay; a.lens = lens;
    a.state_in = state_in; a.state_out = state_out;
    a.ld_q = sh.ld_q; a.ld_k = sh.ld_k; a.ld_v = sh.ld_v; a.ld_o = sh.ld_o;
    a.B = static_cast<int>(sh.batch); a.H = static_cast<int>(sh.heads); a.KH = static_cast<int>(sh.kv_heads);
    a.group = a.H / a.KH;
    a.N = static_cast<int>(sh.seq_len); a.D = static_cast<int>(sh.head_dim); a.E = static_cast<int>(sh.value_dim);
    a.slices = (a.E + 31) / 32;
    a.scale = sh.scale;
    ProfileScope ps(K_ATTN_SELF, s, 2.0 * sh.batch * sh.seq_len * (sh.heads + sh.kv_heads) * sh.head_dim * sh.value_dim);
    const int64_t groups = sh.batch * sh.kv_heads * a.slices;
    k_linear_tokens<<<grid_of(groups, kThreads), kThreads, 0, s>>>(a);
    launch_check("attention_linear");
}

}  // namespace bh
