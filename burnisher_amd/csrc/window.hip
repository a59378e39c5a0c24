// Sliding-window attention with first tokens that stay visible, over grouped heads:
//   out[b, i, h] = sum_j softmax_j(scale * q[b, i, h] . k[b, j, h / group]) v[b, j, h / group]
// over the keys j < kv_lens[b] that query i, at position p = q_starts[b] + i, sees:
//   j <= p + right and (j >= p - left or j < sinks).
// A query that sees no key gives zeros.
//
// The heads of a group read the same keys, so they are rows of one tile: row r of (batch row, key head)
// is token r / group, head r % group of the group, and the rows of a tile share a narrow window. A
// workgroup walks the keys that one of its rows sees and no others: first those below `sinks`, then the
// window, in blocks from its first key on. Of a last block's keys those past the window's end are loaded as
// the last one that is seen, so what lies there (the unwritten end of a cache, a NaN) never enters a product.
//
// Both products run on v_mfma_f32_16x16x32_bf16 in transposed tiles, S^T = K Q^T and O^T += V^T P^T: two
// accumulator tiles of the first are one operand of the second, so P stays in registers, and V^T comes out of
// row-major V by the transposing LDS read, which gives a lane four keys of one column. K and V go to LDS by
// direct loads, a key a row of an odd number of 16-byte chunks (K: the 16 rows of a fragment read then start in
// different banks) or twice an odd number (V: the eight rows of half a transposing read do).
//
// The softmax keeps a running maximum in log2 units, moved only when a score of the wave exceeds it by more
// than 8: any fixed value gives the same result after the division, and this bounds a weight by 2^8. Weights are
// rounded to bf16 for the second product (2^-8 of each); the scores, their sums and the output sums are fp32.
#include "common.h"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace bh {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.4028235e38f;   // a maximum before any score: finite, so exp2(-inf - it) is 0
constexpr float kSlack = 8.0f;

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

struct WindowArgs {
    const bf16_t* q;
    const bf16_t* k;
    const bf16_t* v;
    bf16_t* out;
    const int32_t* kv_lens;
    const int32_t* q_starts;
    float* part;   // split keys: [splits][rows of all][D] sums, then [splits][rows of all][2] maxima and denominators
    int64_t ld_q, ld_kv, ld_o;
    int B, H, KH, group, Sq, Skv, D;
    int left, right, sinks;
    int tiles;     // row tiles per (batch row, key head)
    int splits;
    float c;       // scale * log2(e)
};

__host__ __device__ constexpr int k_pitch(int chunks) { return chunks | 1; }
__host__ __device__ constexpr int v_pitch(int chunks) { return (chunks + 1) / 4 * 4 + 2; }

__device__ __forceinline__ int clamp_to(int64_t v, int lo, int hi) {
    return static_cast<int>(min(max(v, static_cast<int64_t>(lo)), static_cast<int64_t>(hi)));
}

__device__ __forceinline__ uint32_t lds_address(const char* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)(p)));
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// Lane L's 16 bytes at base + off land at LDS address lds + 16 L (`base` and `lds` uniform). Inline assembly so
// that the compiler does not wait for these loads by itself: s_waitcnt below covers them.
__device__ __forceinline__ void dma16(const void* base, uint32_t off, const char* lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds_address(lds)), "v"(off), "s"(base)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// Four keys of column (lane % 16): lane i of a 16-lane group passes the address of columns 4 (i % 4) .. + 3 of the
// group's key i / 4.
__device__ __forceinline__ s16x4_t read_transposed(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(lds_address(p)));
}

// ---- which keys a tile of rows walks -----------------------------------------------------------------

// Keys [0, near) and [lo, hi): all that a row of tokens first .. last of batch row b sees.
struct Keys {
    int len, near, lo, hi;
    int64_t start;
    __device__ __forceinline__ Keys(const WindowArgs& a, int b, int first, int last) {
        len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.Skv) : a.Skv;
        start = a.q_starts ? a.q_starts[b] : a.Skv - a.Sq;
        hi = see_hi(a, last);
        lo = min(see_lo(a, first), hi);
        near = min(a.sinks, lo);
    }
    // Token i sees [see_lo, see_hi), and of the keys below `sinks` those below see_hi.
    __device__ __forceinline__ int see_hi(const WindowArgs& a, int i) const {
        return a.right < 0 ? len : clamp_to(start + i + a.right + 1, 0, len);
    }
    __device__ __forceinline__ int see_lo(const WindowArgs& a, int i) const {
        return a.left < 0 ? 0 : clamp_to(start + i - a.left, 0, len);
    }
};

// Block j of N keys: keys base .. base + N - 1, of which those from `end` on are none of the tile's.
template <int N>
struct Blocks {
    int nb1, n, near, lo, hi;
    __device__ __forceinline__ explicit Blocks(const Keys& k) : near(k.near), lo(k.lo), hi(k.hi) {
        nb1 = (near + N - 1) / N;
        n = nb1 + (hi - lo + N - 1) / N;
    }
    __device__ __forceinline__ int base(int j) const { return j < nb1 ? j * N : lo + (j - nb1) * N; }
    __device__ __forceinline__ int end(int j) const { return j < nb1 ? near : hi; }
};

// One operand's 16-byte chunks of a block: chunk 64 n + lane of the LDS image is column id % pitch of key id / pitch;
// pad columns repeat the key's last chunk.
template <int PITCH>
__device__ __forceinline__ uint32_t chunk_offset(int n, int lane, int chunks, int last_key, uint32_t ld_bytes) {
    const uint32_t id = n * 64 + lane, key = id / PITCH, col = id - key * PITCH;
    return min(key, static_cast<uint32_t>(last_key)) * ld_bytes + min(col, static_cast<uint32_t>(chunks - 1)) * 16;
}

// ---- a wave's state: QT tiles of 16 rows, lane (g, c) = (lane / 16, lane % 16) holds row c of each ------

template <int DT, int QT>
struct Rows {
    static constexpr int KS = (DT + 1) / 2;   // K = 32 steps of the score product
    bf16x8_t q[QT][KS];
    f32x4_t o[DT][QT];                        // o[e][u][r]: column 16 e + 4 g + r
    float top[QT], sum[QT];                   // the running maximum; this lane's part of the denominator
    int lo[QT], hi[QT];                       // the row's window

    __device__ __forceinline__ void init(const WindowArgs& a, const Keys& keys, int b, int kh, int row0, int rows, int lane) {
        const int g = lane >> 4, c = lane & 15;
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            const int row = min(row0 + u * 16 + c, rows - 1), token = row / a.group, head = kh * a.group + row % a.group;
            lo[u] = keys.see_lo(a, token);
            hi[u] = keys.see_hi(a, token);
            const bf16_t* src = a.q + (static_cast<int64_t>(b) * a.Sq + token) * a.ld_q + static_cast<int64_t>(head) * a.D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = ks * 32 + g * 8;
                const bf16x8_t f = *reinterpret_cast<const bf16x8_t*>(src + min(d, a.D - 8));
#pragma unroll
                for (int e = 0; e < 8; ++e) q[u][ks][e] = d < a.D ? f[e] : static_cast<__bf16>(0.0f);
            }
            top[u] = kLowest;
            sum[u] = 0.f;
#pragma unroll
            for (int e = 0; e < DT; ++e) o[e][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }

    // Scores, weights and output sums of 16 T keys (T even) from `base` on in the LDS images at kp and vp. `masked`: some row
    // sees only some of them.
    template <int T>
    __device__ __forceinline__ void step(const char* kp, const char* vp, int kpitch, int vpitch, int D, int base, int end,
                                         int sinks, bool masked, float c_, int lane) {
        const int g = lane >> 4, c = lane & 15;
        f32x4_t s[T][QT];
#pragma unroll
        for (int t = 0; t < T; ++t) {
#pragma unroll
            for (int u = 0; u < QT; ++u) s[t][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(kp + (t * 16 + c) * kpitch + min(ks * 64 + g * 16, D * 2 - 16));
                if (ks == KS - 1)   // past head_dim the query is zero, and so must the key be: it may hold a NaN
#pragma unroll
                    for (int e = 0; e < 8; ++e) kf[e] = ks * 32 + g * 8 < D ? kf[e] : static_cast<__bf16>(0.0f);
#pragma unroll
                for (int u = 0; u < QT; ++u) s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[u][ks], s[t][u], 0, 0, 0);
            }
        }
        if (masked) {
#pragma unroll
            for (int u = 0; u < QT; ++u) {
                const int first = lo[u] - base, last = min(hi[u], end) - base, near = sinks - base;
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = t * 16 + g * 4 + r;
                        if (!(j < last && (j >= first || j < near))) s[t][u][r] = -INFINITY;
                    }
            }
        }
        float mx[QT];
        bool move = false;
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            mx[u] = -INFINITY;
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx[u] = fmaxf(mx[u], s[t][u][r]);
            mx[u] *= c_;
            move |= mx[u] > top[u] + kSlack;
        }
        if (__any(move)) {
#pragma unroll
            for (int u = 0; u < QT; ++u) {
                float m = fmaxf(mx[u], __shfl_xor(mx[u], 16, 64));
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                m = fmaxf(m, top[u]);
                const float alpha = exp2f(top[u] - m);
                top[u] = m;
                sum[u] *= alpha;
#pragma unroll
                for (int e = 0; e < DT; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[e][u][r] *= alpha;
            }
        }
#pragma unroll
        for (int u = 0; u < QT; ++u)
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][u][r], c_, -top[u]));
                    sum[u] += p;
                    s[t][u][r] = p;
                }
        const char* vrow = vp + (g * 4 + (c >> 2)) * vpitch + (c & 3) * 8;
#pragma unroll
        for (int h = 0; h < T / 2; ++h) {
            bf16x8_t p[QT];
#pragma unroll
            for (int u = 0; u < QT; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[u][r] = static_cast<__bf16>(s[2 * h][u][r]);
                    p[u][4 + r] = static_cast<__bf16>(s[2 * h + 1][u][r]);
                }
#pragma unroll
            for (int e = 0; e < DT; ++e) {
                const char* at = vrow + h * 32 * vpitch + e * 32;
                const s16x8_t v = __builtin_shufflevector(read_transposed(at), read_transposed(at + 16 * vpitch), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int u = 0; u < QT; ++u)
                    o[e][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), p[u], o[e][u], 0, 0, 0);
            }
        }
    }

    __device__ __forceinline__ float denominator(int u) const {
        float l = sum[u] + __shfl_xor(sum[u], 16, 64);
        return l + __shfl_xor(l, 32, 64);
    }
};

// Whether a wave whose rows' windows run from [lo0, hi0) (its first token's) to [lo1, hi1) (its last's) sees something
// of keys base .. base + N - 1, and whether all its rows see all of them.
template <int N>
__device__ __forceinline__ bool sees_some(int base, int end, int lo0, int hi1, int sinks) {
    return base < min(end, hi1) && (base + N > lo0 || base < sinks);
}
template <int N>
__device__ __forceinline__ bool sees_all(int base, int end, int lo1, int hi0, int sinks) {
    return base + N <= min(end, hi0) && (base >= lo1 || base + N <= sinks);
}

// ---- many rows: 128 a workgroup, 32 a wave; K and V in blocks of 64 keys that its four waves share ------

constexpr int kKeys = 64;

template <int DT, int QT>
__global__ void __launch_bounds__(kThreads, 2) k_window_many(WindowArgs a) {
    constexpr int kChunks = DT * 2, KP = k_pitch(kChunks), VP = v_pitch(kChunks);   // for the widest head_dim here
    constexpr int kStage = kKeys * 16 * (KP + VP);
    constexpr int kItems = (KP + VP + 3) / 4;       // loads a wave issues per block
    __shared__ __attribute__((aligned(1024))) char smem[2 * kStage];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int T = a.tiles * a.B * a.KH;
    int id = blockIdx.x;
    if ((T & 7) == 0) id = (id & 7) * (T >> 3) + (id >> 3);   // neighbouring tiles, which share keys, on one XCD
    const int tile = id % a.tiles, bk = id / a.tiles, kh = bk % a.KH, b = bk / a.KH;
    const int rows = a.group * a.Sq, row0 = tile * (64 * QT), row1 = min(row0 + 64 * QT, rows) - 1;
    const Keys keys(a, b, row0 / a.group, row1 / a.group);
    const Blocks<kKeys> blocks(keys);

    Rows<DT, QT> w;
    const int w0 = row0 + wave * (16 * QT), w1 = min(w0 + 16 * QT, rows) - 1;
    w.init(a, keys, b, kh, w0, rows, lane);
    const bool any = w0 < rows;
    const int t0 = min(w0, rows - 1) / a.group, t1 = max(w1, 0) / a.group;
    const int lo0 = keys.see_lo(a, t0), lo1 = keys.see_lo(a, t1), hi0 = keys.see_hi(a, t0), hi1 = keys.see_hi(a, t1);

    const uint32_t ld_bytes = static_cast<uint32_t>(a.ld_kv) * 2;
    const int chunks = a.D / 8;
    const int64_t first = static_cast<int64_t>(b) * a.Skv * a.ld_kv + static_cast<int64_t>(kh) * a.D;
    // item i of a wave: LDS rows of 1 KiB 4 i + wave, K's first, then V's
    uint32_t off[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int n = i * 4 + wave;
        off[i] = n < KP ? chunk_offset<KP>(n, lane, chunks, kKeys - 1, ld_bytes)
                        : chunk_offset<VP>(n - KP, lane, chunks, kKeys - 1, ld_bytes);
    }
    auto load = [&](int j) {
        char* stage = smem + (j & 1) * kStage;
        const int base = blocks.base(j), last = blocks.end(j) - base - 1;
        const bf16_t *k = a.k + first + static_cast<int64_t>(base) * a.ld_kv, *v = a.v + first + static_cast<int64_t>(base) * a.ld_kv;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int n = i * 4 + wave;
            if (n >= KP + VP) continue;
            uint32_t o = off[i];
            if (last < kKeys - 1)
                o = n < KP ? chunk_offset<KP>(n, lane, chunks, last, ld_bytes) : chunk_offset<VP>(n - KP, lane, chunks, last, ld_bytes);
            dma16(n < KP ? k : v, o, stage + n * 1024);
        }
    };
    if (blocks.n > 0) load(0);
    for (int j = 0; j < blocks.n; ++j) {
        // block j has landed, for everyone behind the barrier, and everyone has read block j - 1
        asm volatile("" ::: "memory");
        s_waitcnt<0, 0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (j + 1 < blocks.n) load(j + 1);
        const int base = blocks.base(j), end = blocks.end(j);
        if (!any || !sees_some<kKeys>(base, end, lo0, hi1, a.sinks)) continue;
        const char* stage = smem + (j & 1) * kStage;
        w.template step<4>(stage, stage + KP * 1024, KP * 16, VP * 16, a.D, base, end, a.sinks,
                           !sees_all<kKeys>(base, end, lo1, hi0, a.sinks), a.c, lane);
    }
    const int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        const float l = w.denominator(u);
        const int row = w0 + u * 16 + c;
        if (row >= rows) continue;
        const float rl = l == 0.f ? 0.f : 1.0f / l;
        bf16_t* dst = a.out + (static_cast<int64_t>(b) * a.Sq + row / a.group) * a.ld_o +
                      static_cast<int64_t>(kh * a.group + row % a.group) * a.D;
#pragma unroll
        for (int e = 0; e < DT; ++e) {
            const int d = e * 16 + g * 4;
            if (d < a.D)
                *reinterpret_cast<uint2*>(dst + d) = make_uint2(f2bf2(w.o[e][u][0] * rl, w.o[e][u][1] * rl),
                                                                f2bf2(w.o[e][u][2] * rl, w.o[e][u][3] * rl));
        }
    }
}

// ---- few rows: 16 a workgroup, whose waves take pieces of 32 keys in turn, each through LDS of its own -----
//
// Bound by the keys' bytes: a wave waits only for its own loads, two pieces in flight, and the waves' sums meet
// at the end. With `splits` the keys go to several workgroups, whose partial results k_window_join sums.

constexpr int kPiece = 32;

template <int DT>
__global__ void __launch_bounds__(kThreads, 1) k_window_few(WindowArgs a) {
    constexpr int kChunks = DT * 2, KP = k_pitch(kChunks), VP = v_pitch(kChunks);
    constexpr int kK = (KP + 1) / 2, kItems = kK + VP / 2;   // loads per piece: 32 rows of KP and of VP chunks
    constexpr int kStage = kItems * 1024;
    static_assert(kItems <= 60, "vmcnt");
    __shared__ __attribute__((aligned(1024))) char smem[4 * 2 * kStage];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int split = blockIdx.x % a.splits, id = blockIdx.x / a.splits;
    const int tile = id % a.tiles, bk = id / a.tiles, kh = bk % a.KH, b = bk / a.KH;
    const int rows = a.group * a.Sq, row0 = tile * 16, row1 = min(row0 + 16, rows) - 1;
    const int t0 = row0 / a.group, t1 = row1 / a.group;
    const Keys keys(a, b, t0, t1);
    const Blocks<kPiece> pieces(keys);
    const int j0 = static_cast<int>(static_cast<int64_t>(split) * pieces.n / a.splits) + wave;
    const int j1 = static_cast<int>(static_cast<int64_t>(split + 1) * pieces.n / a.splits);
    const int lo1 = keys.see_lo(a, t1), hi0 = keys.see_hi(a, t0);

    Rows<DT, 1> w;
    const uint32_t ld_bytes = static_cast<uint32_t>(a.ld_kv) * 2;
    const int chunks = a.D / 8;
    const int64_t first = static_cast<int64_t>(b) * a.Skv * a.ld_kv + static_cast<int64_t>(kh) * a.D;
    uint32_t off[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i)
        off[i] = i < kK ? chunk_offset<KP>(i, lane, chunks, kPiece - 1, ld_bytes)
                        : chunk_offset<VP>(i - kK, lane, chunks, kPiece - 1, ld_bytes);
    char* own = smem + wave * 2 * kStage;
    auto load = [&](int j, int slot) {
        const int base = pieces.base(j), last = pieces.end(j) - base - 1;
        const bf16_t *k = a.k + first + static_cast<int64_t>(base) * a.ld_kv, *v = a.v + first + static_cast<int64_t>(base) * a.ld_kv;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            uint32_t o = off[i];
            if (last < kPiece - 1)
                o = i < kK ? chunk_offset<KP>(i, lane, chunks, last, ld_bytes) : chunk_offset<VP>(i - kK, lane, chunks, last, ld_bytes);
            dma16(i < kK ? k : v, o, own + slot * kStage + i * 1024);
        }
    };
    if (j0 < j1) load(j0, 0);
    w.init(a, keys, b, kh, row0, rows, lane);
    if (j0 + 4 < j1) load(j0 + 4, 1);
    int slot = 0;
    for (int j = j0; j < j1; j += 4) {
        // this wave's piece j has landed; the next may be on its way
        asm volatile("" ::: "memory");
        if (j + 4 < j1) s_waitcnt<kItems, 0>();
        else s_waitcnt<0, 0>();
        asm volatile("" ::: "memory");
        const int base = pieces.base(j), end = pieces.end(j);
        const char* stage = own + slot * kStage;
        w.template step<2>(stage, stage + kK * 1024, KP * 16, VP * 16, a.D, base, end, a.sinks,
                           !sees_all<kPiece>(base, end, lo1, hi0, a.sinks), a.c, lane);
        if (j + 8 < j1) {   // into the piece that was just read
            asm volatile("" ::: "memory");
            s_waitcnt<63, 0>();
            asm volatile("" ::: "memory");
            load(j + 8, slot);
        }
        slot ^= 1;
    }
    // the four waves' rows: maximum, denominator and sums
    constexpr int kRow = DT * 16 + 4;   // floats
    static_assert(4 * 16 * kRow * 4 <= 4 * 2 * kStage, "the sums fit where the keys were");
    const float l = w.denominator(0);
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
    const int g = lane >> 4, c = lane & 15;
    float* mine = sums + (wave * 16 + c) * kRow;
    if (g == 0) {
        mine[DT * 16] = w.top[0];
        mine[DT * 16 + 1] = l;
    }
#pragma unroll
    for (int e = 0; e < DT; ++e) *reinterpret_cast<f32x4_t*>(mine + e * 16 + g * 4) = w.o[e][0];
    __syncthreads();
    const int r = threadIdx.x >> 4, row = row0 + r;
    if (row >= rows) return;
    float m = kLowest, total = 0.f, scale[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, sums[(k * 16 + r) * kRow + DT * 16]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        scale[k] = exp2f(sums[(k * 16 + r) * kRow + DT * 16] - m);
        total += scale[k] * sums[(k * 16 + r) * kRow + DT * 16 + 1];
    }
    const int64_t all = static_cast<int64_t>(a.B) * a.KH * rows, at = static_cast<int64_t>(bk) * rows + row;
    const float rl = total == 0.f ? 0.f : 1.0f / total;
    bf16_t* dst = a.out + (static_cast<int64_t>(b) * a.Sq + row / a.group) * a.ld_o +
                  static_cast<int64_t>(kh * a.group + row % a.group) * a.D;
    for (int d = (threadIdx.x & 15) * 4; d < a.D; d += 64) {
        f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) v += *reinterpret_cast<const f32x4_t*>(sums + (k * 16 + r) * kRow + d) * scale[k];
        if (a.splits == 1) *reinterpret_cast<uint2*>(dst + d) = make_uint2(f2bf2(v[0] * rl, v[1] * rl), f2bf2(v[2] * rl, v[3] * rl));
        else *reinterpret_cast<f32x4_t*>(a.part + (split * all + at) * a.D + d) = v;
    }
    if (a.splits > 1 && (threadIdx.x & 15) == 0) {
        float* ml = a.part + a.splits * all * a.D + (split * all + at) * 2;
        ml[0] = m;
        ml[1] = total;
    }
}

// The splits' results of a row: 32 lanes a row, four columns each.
__global__ void __launch_bounds__(kThreads) k_window_join(WindowArgs a) {
    const int rows = a.group * a.Sq;
    const int64_t all = static_cast<int64_t>(a.B) * a.KH * rows;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int d = (threadIdx.x & 31) * 4;
    if (at >= all || d >= a.D) return;
    const float* ml = a.part + a.splits * all * a.D;
    float m = kLowest, total = 0.f;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[(s * all + at) * 2]);
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const float f = exp2f(ml[(s * all + at) * 2] - m);
        total += f * ml[(s * all + at) * 2 + 1];
        v += *reinterpret_cast<const f32x4_t*>(a.part + (s * all + at) * a.D + d) * f;
    }
    const float rl = total == 0.f ? 0.f : 1.0f / total;
    const int row = static_cast<int>(at % rows), bk = static_cast<int>(at / rows), kh = bk % a.KH, b = bk / a.KH;
    bf16_t* dst = a.out + (static_cast<int64_t>(b) * a.Sq + row / a.group) * a.ld_o +
                  static_cast<int64_t>(kh * a.group + row % a.group) * a.D;
    *reinterpret_cast<uint2*>(dst + d) = make_uint2(f2bf2(v[0] * rl, v[1] * rl), f2bf2(v[2] * rl, v[3] * rl));
}

int device_cus() {
    static std::atomic<int> cus[64] = {};
    int dev = 0;
    hip_check(hipGetDevice(&dev), "hipGetDevice");
    require(dev >= 0 && dev < 64, "attention_window: device index out of range");
    int n = cus[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        hip_check(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev), "hipDeviceGetAttribute");
        require(n > 0, "attention_window: device reports no compute units");
        cus[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

struct Plan {
    bool many;
    int splits;
};
Plan plan(const WindowShape& sh, bool may_split) {
    const int64_t cus = device_cus(), group = sh.heads / sh.kv_heads, rows = group * sh.q_len;
    const int64_t many = sh.batch * sh.kv_heads * ((rows + 127) / 128);
    if (many * 2 >= cus) return {true, 1};
    // the keys that 16 rows see at most, in pieces
    const int64_t tokens = (15 + group) / group;
    int64_t keys = sh.kv_len;
    if (sh.left >= 0 && sh.right >= 0) keys = std::min(keys, static_cast<int64_t>(sh.left) + sh.right + tokens + sh.sinks);
    const int64_t few = sh.batch * sh.kv_heads * ((rows + 15) / 16), pieces = (keys + kPiece - 1) / kPiece;
    const int64_t splits = may_split ? std::min(std::max<int64_t>(1, 2 * cus / few), std::max<int64_t>(1, pieces / 8)) : 1;
    return {false, static_cast<int>(std::min<int64_t>(splits, 64))};
}

template <int DT>
void launch(const WindowArgs& a0, const Plan& how, int64_t grid, hipStream_t s) {
    WindowArgs a = a0;
    if (how.many) k_window_many<DT, 2><<<static_cast<unsigned>(grid), kThreads, 0, s>>>(a);
    else k_window_few<DT><<<static_cast<unsigned>(grid), kThreads, 0, s>>>(a);
}

}  // namespace

int64_t attention_window_workspace_floats(const WindowShape& sh) {
    const Plan how = plan(sh, true);
    if (how.splits == 1) return 0;
    return how.splits * sh.batch * sh.heads * sh.q_len * (sh.head_dim + 2);
}

void launch_attention_window(const bf16_t* q, const bf16_t* k, const bf16_t* v, bf16_t* out, const WindowShape& sh,
                             const int32_t* kv_lens, const int32_t* q_starts, float* ws, hipStream_t s) {
    WindowArgs a;
    a.q = q; a.k = k; a.v = v; a.out = out;
    a.kv_lens = kv_lens; a.q_starts = q_starts;
    a.part = ws;
    a.ld_q = sh.ld_q; a.ld_kv = sh.ld_kv; a.ld_o = sh.ld_o;
    a.B = static_cast<int>(sh.batch); a.H = static_cast<int>(sh.heads); a.KH = static_cast<int>(sh.kv_heads);
    a.group = a.H / a.KH;
    a.Sq = static_cast<int>(sh.q_len); a.Skv = static_cast<int>(sh.kv_len); a.D = static_cast<int>(sh.head_dim);
    a.left = sh.left; a.right = sh.right; a.sinks = sh.sinks;
    a.c = sh.scale * kLog2e;
    const Plan how = plan(sh, ws != nullptr);
    const int64_t rows = static_cast<int64_t>(a.group) * a.Sq, per = how.many ? 128 : 16, tiles = (rows + per - 1) / per;
    a.tiles = static_cast<int>(tiles);
    a.splits = how.splits;
    const int64_t grid = tiles * sh.batch * sh.kv_heads * how.splits;
    require(grid < (int64_t{1} << 31), "attention_window: too many queries");
    ProfileScope ps(sh.q_len == sh.kv_len ? K_ATTN_SELF : K_ATTN_CROSS, s, 0);
    const int dt = (a.D + 15) / 16;
    if (dt <= 2) launch<2>(a, how, grid, s);
    else if (dt <= 4) launch<4>(a, how, grid, s);
    else if (dt <= 5) launch<5>(a, how, grid, s);
    else if (dt <= 6) launch<6>(a, how, grid, s);
    else launch<8>(a, how, grid, s);
    launch_check("attention_window");
    if (how.splits > 1) {
        const int64_t all = rows * sh.batch * sh.kv_heads;
        k_window_join<<<static_cast<unsigned>((all + 7) / 8), kThreads, 0, s>>>(a);
        launch_check("attention_window");
    }
}

}  // namespace bh
