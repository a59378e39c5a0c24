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
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
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
    f32x4_t sum[QT];                          // the denominator, from a row of ones beside V^T: the matrix cores add it up
    float top[QT];                            // the running maximum
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
            sum[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < DT; ++e) o[e][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }

    // The scores of 16 keys, rows 16 t .. of the LDS image at kp: lane (g, c) has keys 16 t + 4 g + r of row c. Past
    // head_dim the query is zero, against the key's last chunk again.
    __device__ __forceinline__ void scores(f32x4_t (&s)[QT], int t, const char* kp, int kpitch, int D, int lane) const {
        const int g = lane >> 4, c = lane & 15;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(kp + (t * 16 + c) * kpitch + min(ks * 64 + g * 16, D * 2 - 16));
#pragma unroll
            for (int u = 0; u < QT; ++u)
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[u][ks], ks == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : s[u], 0, 0, 0);
        }
    }
    // Those of keys from `base` on that a row does not see become -inf.
    template <int T>
    __device__ __forceinline__ void mask(f32x4_t (&s)[T][QT], int base, int end, int sinks, int lane) const {
        const int g = lane >> 4;
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            const int first = lo[u] - base, last = min(hi[u], end) - base, near = sinks - base;
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = t * 16 + g * 4 + r;
                    const bool seen = (j < last) & ((j >= first) | (j < near));
                    s[t][u][r] = seen ? s[t][u][r] : -INFINITY;
                }
        }
    }
    // The largest of this lane's scores of each row, in the maximum's units.
    template <int T>
    __device__ __forceinline__ void largest(float (&mx)[QT], const f32x4_t (&s)[T][QT], float c_) const {
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            mx[u] = -INFINITY;
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx[u] = fmaxf(mx[u], s[t][u][r]);
            mx[u] *= c_;
        }
    }
    // Moves the maximum, and with it the sums, where a score exceeds it by more than the slack.
    __device__ __forceinline__ void raise(const float (&mx)[QT]) {
        bool move = false;
#pragma unroll
        for (int u = 0; u < QT; ++u) move |= mx[u] > top[u] + kSlack;
        if (!__any(move)) return;
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            float m = fmaxf(mx[u], __shfl_xor(mx[u], 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            m = fmaxf(m, top[u]);
            const float alpha = exp2f(top[u] - m);
            top[u] = m;
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[u][r] *= alpha;
#pragma unroll
            for (int e = 0; e < DT; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[e][u][r] *= alpha;
        }
    }
    // The weights of a score tile, in bf16: half an operand of the output product.
    __device__ __forceinline__ u32x2_t weights(const f32x4_t& s, int u, float c_) const {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c_, -top[u]));
        return u32x2_t{f2bf2(w[0], w[1]), f2bf2(w[2], w[3])};
    }
    static __device__ __forceinline__ bf16x8_t operand(u32x2_t x, u32x2_t y) {
        return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3));
    }
    // The output sums and denominators, V's image at vp.
    template <int T>
    __device__ __forceinline__ void accumulate(const bf16x8_t (&p)[T / 2][QT], const char* vp, int vpitch, int lane) {
        const int g = lane >> 4, c = lane & 15;
        bf16x8_t ones;
#pragma unroll
        for (int e = 0; e < 8; ++e) ones[e] = static_cast<__bf16>(1.0f);
        const char* vrow = vp + (g * 4 + (c >> 2)) * vpitch + (c & 3) * 8;
#pragma unroll
        for (int h = 0; h < T / 2; ++h) {
#pragma unroll
            for (int e = 0; e < DT; ++e) {
                const char* at = vrow + h * 32 * vpitch + e * 32;
                const s16x8_t v = __builtin_shufflevector(read_transposed(at), read_transposed(at + 16 * vpitch), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int u = 0; u < QT; ++u)
                    o[e][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), p[h][u], o[e][u], 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < QT; ++u) sum[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[h][u], sum[u], 0, 0, 0);
        }
    }
};

// Whether rows whose windows run from [., hi0) (their first token's) to [lo1, .) (their last's) see all of keys
// base .. base + N - 1.
template <int N>
__device__ __forceinline__ bool sees_all(int base, int end, int lo1, int hi0, int sinks) {
    return base + N <= min(end, hi0) && (base >= lo1 || base + N <= sinks);
}

// ---- many rows: 128 a workgroup, 32 a wave; K and V in blocks of 64 keys that its four waves share --------
//
// Two workgroups a CU (three up to head_dim 64), each with two slots in LDS for K and for V; deeper rings, tiles of 256
// rows and 32 x 32 x 16 products were no faster. What bounds it: the vector instructions, 32 exponentials and about 75
// others a lane and block, run beside the matrix ones only in part, and a block's loads wait for each other while they are
// issued (600 of 3200 to 4500 cycles, five wait states a load among them that dma16_at no longer has; put between the
// products they cost more registers than that). Without the
// exponentials a call takes 8 to 15% less; finding the maximum among the output product's matrix instructions, or acting on
// it behind the barrier, gained nothing. Which blocks a wave sees, and sees whole, are ranges found before the loop, and
// whole blocks load without a branch a load: at head_dim 64 388 -> 340 us. Measured (2 x 16384 tokens of 16 heads, window
// 1024 to either side): head_dim 64 339 us (780 TFLOP/s), 72 445 (its columns are computed as 80 and 96), 128 576 (930);
// 2 x 4096 tokens of 32 / 8 heads of 128, window 1023 back, 158 to 178; 2 x 300 of 64 heads of 64, 128 either side, 15.

constexpr int kKeys = 64, kManyRows = 128;

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) k_window_many(WindowArgs a) {
    constexpr int QT = 2, kChunks = DT * 2, KP = k_pitch(kChunks), VP = v_pitch(kChunks);   // for the widest head_dim here
    constexpr int kKBytes = kKeys * 16 * KP, kVBytes = kKeys * 16 * VP;
    constexpr int kItems = (KP + VP + 3) / 4;   // loads a wave issues per block, at most
    __shared__ __attribute__((aligned(1024))) char kmem[2 * kKBytes], vmem[2 * kVBytes];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int T = a.tiles * a.B * a.KH;
    const int64_t number = group_index();
    if (number >= T) return;
    int id = static_cast<int>(number);
    if ((T & 7) == 0) id = (id & 7) * (T >> 3) + (id >> 3);   // neighbouring tiles, which share keys, on one XCD
    const int tile = id % a.tiles, bk = id / a.tiles, kh = bk % a.KH, b = bk / a.KH;
    const int rows = a.group * a.Sq, row0 = tile * kManyRows, row1 = min(row0 + kManyRows, rows) - 1;
    const Keys keys(a, b, row0 / a.group, row1 / a.group);
    const Blocks<kKeys> blocks(keys);

    Rows<DT, QT> w;
    const int w0 = row0 + wave * (16 * QT), w1 = min(w0 + 16 * QT, rows) - 1;
    w.init(a, keys, b, kh, w0, rows, lane);
    const int t0 = min(w0, rows - 1) / a.group, t1 = max(w1, 0) / a.group;
    const int lo0 = keys.see_lo(a, t0), lo1 = keys.see_lo(a, t1), hi0 = keys.see_hi(a, t0);
    const int hi1 = w0 < rows ? keys.see_hi(a, t1) : 0;   // a wave without rows sees nothing

    const uint32_t ld_bytes = static_cast<uint32_t>(a.ld_kv) * 2;
    const int chunks = a.D / 8;
    const int64_t first = static_cast<int64_t>(b) * a.Skv * a.ld_kv + static_cast<int64_t>(kh) * a.D;
    // A block's loads are the KP rows of 1 KiB of K's LDS image and then V's VP: row 4 i + wave is wave's i-th, the last
    // one of some waves only. K of one block goes with V of the block before it.
    uint32_t off[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int n = i * 4 + wave;
        off[i] = n < KP ? chunk_offset<KP>(n, lane, chunks, kKeys - 1, ld_bytes) : chunk_offset<VP>(n - KP, lane, chunks, kKeys - 1, ld_bytes);
    }
    uint32_t off_last[kItems - KP / 4];   // V's of the last block, which ends inside it in most calls
#pragma unroll
    for (int i = KP / 4; i < kItems; ++i) {
        const int last = blocks.n > 0 ? blocks.end(blocks.n - 1) - blocks.base(blocks.n - 1) - 1 : 0;
        off_last[i - KP / 4] = chunk_offset<VP>(max(i * 4 + wave - KP, 0), lane, chunks, min(last, kKeys - 1), ld_bytes);
    }
    const bf16_t *k0 = a.k + first, *v0 = a.v + first;
    auto key_offset = [&](int base) { return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(base)) * ld_bytes / 2); };
    // K of block jk and V of block jv (jv < 0: not), where there are such blocks. Keys past a block's end: K's are masked, so
    // they may be read where there is memory; V's are the last one again.
    auto load = [&](int jk, int jv) {
        const int kb = blocks.base(jk), vb = blocks.base(max(jv, 0)), k_last = blocks.end(jk) - kb - 1, v_last = blocks.end(max(jv, 0)) - vb - 1;
        const bf16_t *k = k0 + key_offset(kb), *v = v0 + key_offset(vb);
        const char *kl = kmem + (jk & 1) * kKBytes, *vl = vmem + (jv & 1) * kVBytes - KP * 1024;
        const bool with_k = jk < blocks.n, with_v = (jv >= 0) & (jv < blocks.n), k_whole = kb + kKeys <= a.Skv;
        if (with_k & with_v & k_whole & (v_last >= kKeys - 1)) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                const int n = i * 4 + wave;
                if (i * 4 + 3 < KP + VP || n < KP + VP) dma16_at(n < KP ? k : v, off[i], (n < KP ? kl : vl) + n * 1024);
            }
            return;
        }
        if ((jv < 0) & k_whole) {
#pragma unroll
            for (int i = 0; i * 4 < KP; ++i)
                if (i * 4 + wave < KP) dma16_at(k, off[i], kl + (i * 4 + wave) * 1024);
            return;
        }
        if (!with_k & (jv == blocks.n - 1)) {
#pragma unroll
            for (int i = KP / 4; i < kItems; ++i) {
                const int n = i * 4 + wave;
                if (n >= KP && n < KP + VP) dma16_at(v, off_last[i - KP / 4], vl + n * 1024);
            }
            return;
        }
#pragma unroll 1
        for (int n = with_k ? wave : KP + (wave + 3 * KP) % 4; n < (with_v ? KP + VP : KP); n += 4) {
            if (n < KP) dma16_at(k, chunk_offset<KP>(n, lane, chunks, min(k_last, kKeys - 1), ld_bytes), kl + n * 1024);
            else dma16_at(v, chunk_offset<VP>(n - KP, lane, chunks, min(v_last, kKeys - 1), ld_bytes), vl + n * 1024);
        }
    };
    auto join = [&]() {   // this wave's loads have landed and its reads are done; behind the barrier everyone's
        asm volatile("" ::: "memory");
        s_waitcnt<0, 0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    f32x4_t s[4][QT];
    float mx[QT];
    // The wave's blocks, as ranges of their numbers: those of which some row sees some key, and those of which every row
    // sees every key (at least those that the ranges hold), before the window and in it.
    const int lo = blocks.lo, hi = blocks.hi, nb1 = blocks.nb1;
    const int seen_near = (min(blocks.near, hi1) + kKeys - 1) / kKeys, whole_near = min(blocks.near, hi0) / kKeys;
    const int seen0 = nb1 + (a.sinks > lo ? 0 : max(lo0 - lo, 0) / kKeys), seen1 = nb1 + (max(min(hi, hi1) - lo, 0) + kKeys - 1) / kKeys;
    const int whole0 = nb1 + (max(lo1 - lo, 0) + kKeys - 1) / kKeys, whole1 = nb1 + max(min(hi, hi0) - lo, 0) / kKeys;
    auto seen = [&](int j) { return (j < seen_near) | ((j >= seen0) & (j < seen1)); };
    auto maximum = [&](int j) {
        if (!((j < whole_near) | ((j >= whole0) & (j < whole1)))) w.template mask<4>(s, blocks.base(j), blocks.end(j), a.sinks, lane);
        w.template largest<4>(mx, s, a.c);
        w.raise(mx);
    };
    if (blocks.n > 0) {
        load(0, -1);
        join();
        load(1, 0);
#pragma unroll
        for (int t = 0; t < 4; ++t) w.scores(s[t], t, kmem, KP * 16, a.D, lane);
        maximum(0);
    }
    // Block j's weights beside block j + 1's score product, which takes their place tile by tile, then block j's output
    // product. Behind the barrier K of block j + 1 and V of block j have landed, and K of block j and V of block j - 1
    // have been read. Scores that no row of the wave sees are -inf here, so a block that it does not see adds nothing.
    for (int j = 0; j < blocks.n; ++j) {
        join();
        load(j + 2, j + 1);
        if (!(seen(j) | seen(j + 1))) continue;
        const char* kp = kmem + ((j + 1) & 1) * kKBytes;   // behind the last block: scores that nobody uses
        u32x2_t half[4][QT];
        bf16x8_t p[2][QT];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int u = 0; u < QT; ++u) half[t][u] = w.weights(s[t][u], u, a.c);
            w.scores(s[t], t, kp, KP * 16, a.D, lane);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < QT; ++u) p[h][u] = w.operand(half[2 * h][u], half[2 * h + 1][u]);
        w.template accumulate<4>(p, vmem + (j & 1) * kVBytes, VP * 16, lane);
        if (j + 1 < blocks.n) maximum(j + 1);
    }
    const int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        const float l = w.sum[u][0];
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

// ---- few rows: 16 QT a workgroup, whose waves take pieces of 32 keys in turn, each through LDS of its own ----
//
// Bound by the keys' bytes: a wave waits only for its own loads, two pieces in flight, and the waves' sums meet
// at the end. With `splits` the keys go to several workgroups, whose partial results k_window_join sums (4.8 us for
// 512 rows of 128 in two splits: a launch). 16 sequences of one token, 32 / 8 heads of 128, window 4095 back in up
// to 8192 keys: 54 us with the join, 5.0 TB/s. 4 x 64 tokens of the same heads, on 32-row tiles: 46 us (52 when each load
// waited for its base).

constexpr int kPiece = 32;

template <int DT, int QT>
__global__ void __launch_bounds__(kThreads, 1) k_window_few(WindowArgs a) {
    constexpr int kChunks = DT * 2, KP = k_pitch(kChunks), VP = v_pitch(kChunks);
    constexpr int kK = (KP + 1) / 2, kItems = kK + VP / 2;   // loads per piece: 32 rows of KP and of VP chunks
    constexpr int kStage = kItems * 1024;
    static_assert(kItems <= 60, "vmcnt");
    __shared__ __attribute__((aligned(1024))) char smem[4 * 2 * kStage];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int T = a.tiles * a.splits * a.B * a.KH;
    const int64_t number = group_index();
    if (number >= T) return;
    int id = static_cast<int>(number);
    if ((T & 7) == 0) id = (id & 7) * (T >> 3) + (id >> 3);   // tiles that read the same keys on one XCD
    const int tile = id % a.tiles, split = id / a.tiles % a.splits, bk = id / a.tiles / a.splits, kh = bk % a.KH, b = bk / a.KH;
    const int rows = a.group * a.Sq, row0 = tile * (16 * QT), row1 = min(row0 + 16 * QT, rows) - 1;
    const int t0 = row0 / a.group, t1 = row1 / a.group;
    const Keys keys(a, b, t0, t1);
    const Blocks<kPiece> pieces(keys);
    const int j0 = static_cast<int>(static_cast<int64_t>(split) * pieces.n / a.splits) + wave;
    const int j1 = static_cast<int>(static_cast<int64_t>(split + 1) * pieces.n / a.splits);
    const int lo1 = keys.see_lo(a, t1), hi0 = keys.see_hi(a, t0);

    Rows<DT, QT> w;
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
        char* to = own + slot * kStage;
        if (last >= kPiece - 1) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) dma16_at(i < kK ? k : v, off[i], to + i * 1024);
            return;
        }
#pragma unroll 1
        for (int i = 0; i < kItems; ++i)
            dma16_at(i < kK ? k : v, i < kK ? chunk_offset<KP>(i, lane, chunks, last, ld_bytes) : chunk_offset<VP>(i - kK, lane, chunks, last, ld_bytes),
                  to + i * 1024);
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
        f32x4_t s[2][QT];
        float mx[QT];
        bf16x8_t p[1][QT];
#pragma unroll
        for (int t = 0; t < 2; ++t) w.scores(s[t], t, stage, KP * 16, a.D, lane);
        if (!sees_all<kPiece>(base, end, lo1, hi0, a.sinks)) w.template mask<2>(s, base, end, a.sinks, lane);
        w.template largest<2>(mx, s, a.c);
        w.raise(mx);
#pragma unroll
        for (int u = 0; u < QT; ++u) p[0][u] = w.operand(w.weights(s[0][u], u, a.c), w.weights(s[1][u], u, a.c));
        w.template accumulate<2>(p, stage + kK * 1024, VP * 16, lane);
        if (j + 8 < j1) {   // into the piece that was just read
            asm volatile("" ::: "memory");
            s_waitcnt<63, 0>();
            asm volatile("" ::: "memory");
            load(j + 8, slot);
        }
        slot ^= 1;
    }
    // the four waves' rows: maximum, denominator and sums
    constexpr int kRows = 16 * QT, kRow = DT * 16 + 4;   // floats
    static_assert(4 * kRows * kRow * 4 <= 4 * 2 * kStage, "the sums fit where the keys were");
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
    const int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        float* mine = sums + (wave * kRows + u * 16 + c) * kRow;
        if (g == 0) {
            mine[DT * 16] = w.top[u];
            mine[DT * 16 + 1] = w.sum[u][0];
        }
#pragma unroll
        for (int e = 0; e < DT; ++e) *reinterpret_cast<f32x4_t*>(mine + e * 16 + g * 4) = w.o[e][u];
    }
    __syncthreads();
    const int64_t all = static_cast<int64_t>(a.B) * a.KH * rows;
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        const int r = u * 16 + (threadIdx.x >> 4), row = row0 + r;
        if (row >= rows) return;
        float m = kLowest, total = 0.f, scale[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) m = fmaxf(m, sums[(k * kRows + r) * kRow + DT * 16]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            scale[k] = exp2f(sums[(k * kRows + r) * kRow + DT * 16] - m);
            total += scale[k] * sums[(k * kRows + r) * kRow + DT * 16 + 1];
        }
        const int64_t at = static_cast<int64_t>(bk) * rows + row;
        const float rl = total == 0.f ? 0.f : 1.0f / total;
        bf16_t* dst = a.out + (static_cast<int64_t>(b) * a.Sq + row / a.group) * a.ld_o +
                      static_cast<int64_t>(kh * a.group + row % a.group) * a.D;
        for (int d = (threadIdx.x & 15) * 4; d < a.D; d += 64) {
            f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k) v += *reinterpret_cast<const f32x4_t*>(sums + (k * kRows + r) * kRow + d) * scale[k];
            if (a.splits == 1) *reinterpret_cast<uint2*>(dst + d) = make_uint2(f2bf2(v[0] * rl, v[1] * rl), f2bf2(v[2] * rl, v[3] * rl));
            else *reinterpret_cast<f32x4_t*>(a.part + (split * all + at) * a.D + d) = v;
        }
        if (a.splits > 1 && (threadIdx.x & 15) == 0) {
            float* ml = a.part + a.splits * all * a.D + (split * all + at) * 2;
            ml[0] = m;
            ml[1] = total;
        }
    }
}

// The splits' results of a row: 32 lanes a row, four columns each.
__global__ void __launch_bounds__(kThreads) k_window_join(WindowArgs a) {
    const int rows = a.group * a.Sq;
    const int64_t all = static_cast<int64_t>(a.B) * a.KH * rows;
    const int64_t at = group_index() * 8 + (threadIdx.x >> 5);
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

// How a call runs: k_window_many, or k_window_few on tiles of 16 `few` rows with the keys in `splits`. The estimates, in
// us, were checked on 30 shapes on one MI355X (head_dim 32 to 128, 4 to 16384 rows of 77 to 16384 keys), each on every
// kernel and split that fits it: what they choose is within 6% of the fastest on 27, and 9 to 13% above it on 8 x 4 tokens
// of 16 / 4 heads against 3000 keys (eight splits 13.4 to 17.5, four 12.0 to 16.0). Beside 3.5 a workgroup,
//  - many: a block of 64 keys costs 0.62 + 0.006 head_dim alone on a CU, 0.5 + 0.014 beside another workgroup;
//  - few: a piece of 32 keys for each of the four waves costs 0.35 + 0.005 head_dim on 16 rows and 0.3 + 0.009 on 32, one
//    workgroup a CU (two up to head_dim 64), and no less in all than reading the keys at
//    5.2 TB/s (a quarter more on fewer workgroups than CUs);
//  - a join costs 3 + 0.25 a split and its partial results at 3 TB/s.
// 16 sequences of a token each, 32 / 8 heads of 128, 4096 keys: two splits 58 us, none 64, k_window_many 87. Four times
// 64 tokens of the same: 32-row tiles 46, 16-row 63, k_window_many 83. 2 x 64 heads of 300 tokens, head_dim 64:
// k_window_many 14.8, 32-row tiles 23. (64-row tiles were never ahead of these.)
struct Plan {
    int few;      // 0: k_window_many
    int splits;
};
Plan plan(const WindowShape& sh, bool may_split, int64_t cus) {
    const int64_t group = sh.heads / sh.kv_heads, rows = group * sh.q_len, heads = sh.batch * sh.kv_heads;
    const double D = static_cast<double>(sh.head_dim);
    auto keys = [&](int64_t n) {   // that n rows see at most
        if (sh.left < 0 || sh.right < 0) return sh.kv_len;
        const int64_t tokens = std::min((n + group - 2) / group + 1, sh.q_len);
        return std::min<int64_t>(sh.kv_len, int64_t{sh.left} + sh.right + tokens + sh.sinks);
    };
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    Plan best{0, 1};
    double least = 1e30;
    if (rows > 16) {
        const int64_t groups = heads * up(rows, kManyRows);
        const double blocks = static_cast<double>(up(keys(kManyRows), kKeys));
        least = groups <= cus ? 3.5 + blocks * (0.62 + 0.006 * D) : up(groups, 2 * cus) * (3.5 + blocks * (0.5 + 0.014 * D));
    }
    for (int few : {1, 2}) {
        if (few > 1 && rows <= 16) continue;
        const int64_t pieces = up(keys(16 * few), kPiece);
        const double step = few == 1 ? 0.35 + 0.005 * D : 0.3 + 0.009 * D;
        for (int s = 1; s == 1 || (may_split && s <= 32 && 4 * s <= pieces); s *= 2) {
            const int64_t groups = heads * up(rows, 16 * few) * s, at_once = cus * (sh.head_dim <= 64 ? 2 : 1);
            const double bytes = static_cast<double>(heads) * keys(rows) * D * 4;
            double cost = std::max(up(groups, at_once) * (3.5 + up(pieces, 4 * s) * step), bytes / 5.2e6 * (groups < cus ? 1.25 : 1.0));
            if (s > 1) cost += 3 + 0.25 * s + s * static_cast<double>(heads) * rows * (D + 2) * 8 / 3e6;
            if (cost < least) {
                least = cost;
                best = Plan{few, s};
            }
        }
    }
    return best;
}

int tile_rows(const Plan& how) { return how.few == 0 ? kManyRows : 16 * how.few; }

template <int DT>
void launch(const WindowArgs& a, const Plan& how, int64_t grid, hipStream_t s) {
    const dim3 n = grid_of(grid, kThreads);
    if (how.few == 0) k_window_many<DT><<<n, kThreads, 0, s>>>(a);
    else if (how.few == 1) k_window_few<DT, 1><<<n, kThreads, 0, s>>>(a);
    else k_window_few<DT, 2><<<n, kThreads, 0, s>>>(a);
}

}  // namespace

int64_t attention_window_workspace_floats(const WindowShape& sh) {
    const Plan how = plan(sh, true, device_cus());
    if (how.splits == 1) return 0;
    return how.splits * sh.batch * sh.heads * sh.q_len * (sh.head_dim + 2);
}

bh_attention_window_plan attention_window_plan(const WindowShape& sh, bool may_split, int cus) {
    const Plan how = plan(sh, may_split, cus > 0 ? cus : device_cus());
    const int64_t rows = sh.heads / sh.kv_heads * sh.q_len, per = tile_rows(how), tiles = (rows + per - 1) / per;
    return bh_attention_window_plan{static_cast<int>(per), how.splits, tiles * sh.batch * sh.kv_heads * how.splits};
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
    const Plan how = plan(sh, ws != nullptr, device_cus());
    const int64_t rows = static_cast<int64_t>(a.group) * a.Sq, per = tile_rows(how), tiles = (rows + per - 1) / per;
    a.tiles = static_cast<int>(tiles);
    a.splits = how.splits;
    const int64_t grid = tiles * sh.batch * sh.kv_heads * how.splits;
    require(grid < (int64_t{1} << 31), "attention_window: too many queries");
    // the operations of windows that lie inside the sequence; the lengths themselves are on the device
    const int64_t seen = sh.left < 0 || sh.right < 0 ? sh.kv_len : std::min(sh.kv_len, int64_t{sh.left} + sh.right + 1 + sh.sinks);
    ProfileScope ps(sh.q_len == sh.kv_len ? K_ATTN_SELF : K_ATTN_CROSS, s, 4.0 * sh.batch * sh.heads * sh.q_len * seen * sh.head_dim);
    const int dt = (a.D + 15) / 16;
    if (dt <= 2) launch<2>(a, how, grid, s);
    else if (dt <= 4) launch<4>(a, how, grid, s);
    else if (dt <= 5) launch<5>(a, how, grid, s);
    else if (dt <= 6) launch<6>(a, how, grid, s);
    else launch<8>(a, how, grid, s);
    launch_check("attention_window");
    if (how.splits > 1) {
        const int64_t all = rows * sh.batch * sh.kv_heads;
        k_window_join<<<grid_of((all + 7) / 8, kThreads), kThreads, 0, s>>>(a);
        launch_check("attention_window");
    }
}

}  // namespace bh
