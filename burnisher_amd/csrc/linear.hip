// Causal linear attention with a decay for each key head:
//   S_t = decay * S_{t-1} + k_t (outer) v_t,  out_t = scale * q_t . S_t.
//
// Tokens by the chunk of C = 32: with S the state before the chunk, i and j tokens of it,
//   out_i = scale * (decay^(i + 1) q_i . S + sum_{j <= i} decay^(i - j) (q_i . k_j) v_j)
//   S'    = decay^C S + sum_j decay^(C - 1 - j) k_j (outer) v_j,
// four matrix products, all on v_mfma_f32_16x16x32_bf16. A workgroup's waves share a chunk of q, k and v in LDS and
// each keep 16 or 32 columns of the state in accumulators for all chunks; every wave computes the chunk's
// scores anew (12 of its 100 matrix instructions at 128 x 128). Products are formed transposed, S and out^T from V^T, so
// that two accumulator tiles of 16 rows, of scores or state, are one operand of the next product. The order of its
// 32 columns is followed by the other operand: tokens 4 g + r, then 16 + 4 g + r for lane group g (v); the state's
// rows are dealt to its tiles so that theirs is 8 g .. 8 g + 7, 16 bytes of q.
//
// Scores and states are fp32 and enter the output's products as sums of two bf16 values (16 bits, where the output
// keeps 8); decay^(C - 1 - j) v_j enters the state's as three (24 bits), since a state lives on. q, k and v are bf16.
//
// Few heads do not fill the device, so a long sequence is cut into segments: a first launch adds up each one's own state
// from k and v, a second runs over the segments' states, and in a third each segment starts from its own.
//
// What bounds it: one token of 16 sequences, 32 states of 128 x 128 each, their bytes (14.9 us, 4.5 TB/s). Chunks, the
// instructions of few waves: at 128 x 128 a chunk takes 2.3 us alone on a CU, two 3.9, where matrix (100, 1600 cycles) and vector
// instructions (361) of two waves of a SIMD overlap little, and issuing a wave's six direct loads takes 500 to 800 cycles of 6500.
// Two heads at once take 152 and 430 instead of 200 and 722: 2 x 4096 tokens of 32 / 8 heads of 128 71 to 74 us (83 with one where it
// took 71), 51 of it the third launch; 65536 tokens of 16 heads of 128 350 to 361 us, bound by bytes: k and v twice, 106 us of it
// the first launch (4.9 TB/s), 15 the second; 2 x 300 of 64 heads of 64 16.7 us. Ranges are over sixteen runs on several cards.
#include "common.h"

#include <algorithm>
#include <atomic>
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
    int slices;      // of the value columns (token after token)
    // [batch * kv_heads][1 + (segments - 1) * pieces][D][E]: place m + 1 first takes the own state of piece m, and then
    // place n * pieces the state before segment n
    float* states;
    int segments, pieces, length;   // of a sequence, of a segment, tokens of a piece (a multiple of kChunk)
    int first_state;        // the first segment's: 0 zeros, 1 state_in, 2 states
    int turns;              // that a workgroup takes its query heads in, one after the other: 1, or enough for the group
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

// ---- chunks ------------------------------------------------------------------------------------------

constexpr int kChunk = 32;
constexpr float kLog2e = 1.4426950408889634f;

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// 16-byte chunks of a row of an LDS image, a power of two; chunk n of row r stands at place n ^ turn(r), r / (16 / P) with
// its bits rotated by BY. Rows c of one chunk (a fragment: 16 bytes a lane, eight lanes at a time) then lie in different
// banks. Of the transposing reads, eight rows at a time, those of two whole chunks (v: BY 1) do too; those of half of four
// chunks each (k: BY 2), whose order lets a fragment be one read, meet in pairs.
constexpr int places(int steps) { return steps == 1 ? 4 : steps == 2 ? 8 : 16; }
template <int P, int BY>
__device__ __forceinline__ int turn(int row) {
    constexpr int bits = P == 4 ? 2 : P == 8 ? 3 : 4, by = BY % bits;
    const int q = (row & 15) / (16 / P);
    return ((q << by) | (q >> (bits - by))) & (P - 1);
}

// Byte offset that lane `lane` of load n of an image brings from memory: rows from last_row on repeat it, chunks from
// `chunks` on the last one.
template <int P, int BY>
__device__ __forceinline__ uint32_t source(int n, int lane, int chunks, int last_row, uint32_t ld_bytes) {
    const int id = n * 64 + lane, row = id / P, chunk = (id % P) ^ turn<P, BY>(row);
    return static_cast<uint32_t>(min(row, last_row)) * ld_bytes + static_cast<uint32_t>(min(chunk, chunks - 1)) * 16;
}

__device__ __forceinline__ s16x4_t read_transposed(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(lds_address(p)));
}
__device__ __forceinline__ bf16x8_t pair(u32x2_t x, u32x2_t y) {
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3));
}
__device__ __forceinline__ f32x4_t product(bf16x8_t a, bf16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// The bf16 nearest to each value, and what is left of the values: v - h as v + (h, h') . (-1, 0), the dot product of a pair,
// exact here (h is within a factor of two of v), which takes h from its pair as it is.
struct Split {
    uint32_t first, second;   // (-1, 0) and (0, -1); opaque, since an inline -1 would stand for the second
    __device__ __forceinline__ Split() : first(0x0000bf80u), second(0xbf800000u) { asm volatile("" : "+s"(first), "+s"(second)); }
    __device__ __forceinline__ u32x2_t operator()(f32x4_t& v) const {
        u32x2_t h = {f2bf2(v[0], v[1]), f2bf2(v[2], v[3])};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t word = h[i];   // a value: the cast of a vector's element takes its first
            const bf16x2_t p = __builtin_bit_cast(bf16x2_t, word);
            v[2 * i] = __builtin_amdgcn_fdot2_f32_bf16(p, __builtin_bit_cast(bf16x2_t, first), v[2 * i], false);
            v[2 * i + 1] = __builtin_amdgcn_fdot2_f32_bf16(p, __builtin_bit_cast(bf16x2_t, second), v[2 * i + 1], false);
        }
        return h;
    }
};

// STEPS: of 32 columns of q and k; TILES: of 16 value columns a wave. A workgroup walks a segment from the state before it
// for HEADS query heads of a group at once, which have the state in common. With none it adds up a piece's own state from
// k and v, from its end back, so that weights only fall and the walk ends where they are zero, and what it read last is
// what the next launch reads first.
template <int STEPS, int TILES, int WAVES, int HEADS>
__global__ void __launch_bounds__(WAVES * 64, 2) k_linear_chunks(LinearArgs a) {
    constexpr int P = places(STEPS), PV = places(WAVES * TILES / 2), DT = 2 * STEPS;
    constexpr bool OUT = HEADS > 0;
    constexpr int kLoadsQ = HEADS * (P / 2), kLoadsK = P / 2, kLoads = kLoadsQ + kLoadsK + PV / 2;   // of 1 KiB
    constexpr int kItems = (kLoads + WAVES - 1) / WAVES;                                             // a wave's
    // Two workgroups fit a CU. Two stages instead of three: 4 x 2400 tokens of 64 heads of 64, one workgroup a CU, 108 us for 85, but
    // 2 x 300 15.9 for 16.9 and 8 x 2400 147 for 163. Two heads of 128 at once in three stages, alone on a CU, lost 4 to 10%.
    constexpr int kStage = kLoads * 1024, kStages = 3 * kStage <= 80 * 1024 ? 3 : 2;
    __shared__ __attribute__((aligned(1024))) char smem[kStages * kStage];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int per = OUT ? a.group / (HEADS * a.turns) : 1, segments = OUT ? a.segments : (a.segments - 1) * a.pieces;
    const int64_t number = group_index();
    const int T = a.B * a.KH * segments * per;
    if (number >= T) return;
    int id = static_cast<int>(number);
    if ((T & 7) == 0) id = (id & 7) * (T >> 3) + (id >> 3);   // heads of a group, which share keys, on one XCD
    const int at = id % per, segment = id / per % segments;
    const int64_t bk = id / per / segments;
    const int length = OUT ? a.length * a.pieces : a.length, first = segment * length;
    const int kh = static_cast<int>(bk) % a.KH;
    const int64_t b = static_cast<int>(bk) / a.KH;
    const int n = a.lens ? min(max(a.lens[b], 0), a.N) : a.N, last_segment = n > 0 ? (n - 1) / (a.length * a.pieces) : 0;
    if (!OUT && segment >= last_segment * a.pieces) return;
    const float log_decay = log_decay_of(a, kh), rate = log_decay * kLog2e;
    const int count = min(max(n - first, 0), length);
    // a weight below 2^-150 is zero
    const int chunks = OUT ? (count + kChunk - 1) / kChunk : min(length / kChunk, static_cast<int>(1.f + 150.f / fmaxf(-rate * kChunk, 1e-6f)));
    const int column = wave * TILES * 16;   // the wave's first value column
    const bool active = column < a.E;
    auto column_of = [&](int x, int i) { return column + (TILES == 2 ? (i >> 2) * 8 + x * 4 + (i & 3) : i); };   // row or column i of tile x

    const uint32_t ldq = static_cast<uint32_t>(a.ld_q) * 2, ldk = static_cast<uint32_t>(a.ld_k) * 2, ldv = static_cast<uint32_t>(a.ld_v) * 2;
    const int dc = a.D / 8, ec = a.E / 8;
    auto offset = [&](int m, int last_row) {
        return m < kLoadsQ             ? source<P, 2>(m % (P / 2), lane, dc, last_row, ldq)
               : m < kLoadsQ + kLoadsK ? source<P, 2>(m - kLoadsQ, lane, dc, last_row, ldk)
                                       : source<PV, TILES>(m - kLoadsQ - kLoadsK, lane, ec, last_row, ldv);
    };
    uint32_t off[kItems];   // (a wave beyond the last load repeats it)
#pragma unroll
    for (int i = 0; i < kItems; ++i) off[i] = offset(min(i * WAVES + wave, kLoads - 1), kChunk - 1);
    const int64_t row0 = b * a.N + first;
    const bf16_t* k0 = a.k + row0 * a.ld_k + static_cast<int64_t>(kh) * a.D;
    const bf16_t* v0 = a.v + row0 * a.ld_v + static_cast<int64_t>(kh) * a.E;

    // where this lane's fragments start in an image: chunk g of row c (of q and k), and of row 4 g + c / 4, transposed, half
    // of chunk c % 4 (k, and v in two tiles, whose columns are dealt as the state's rows) or a quarter of chunks 0 and 1
    const int trow = 4 * g + (c >> 2);
    const int frag = c * P * 16 + (g ^ turn<P, 2>(c)) * 16;
    const int kt = trow * P * 16 + ((c & 3) ^ turn<P, 2>(trow)) * 16;
    const int vt = TILES == 2 ? trow * PV * 16 + ((c & 3) ^ turn<PV, 2>(trow)) * 16
                              : trow * PV * 16 + (((c & 3) >> 1) ^ turn<PV, 1>(trow)) * 16 + (c & 1) * 8;

    const Split take_bf16;
    // powers of the decay: token j of the fragment's order before the chunk's end, and (times scale) query c of a tile
    // against the keys of its own tile, of the one before, and the state
    float to_end[8], own[4], before[4], since[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) to_end[e] = exp2f(rate * (kChunk - 1 - ((e & 4) * 4 + 4 * g + (e & 3))));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int gap = c - 4 * g - r;
        own[r] = gap >= 0 ? exp2f(rate * gap) * a.scale : 0.f;
        before[r] = exp2f(rate * (16 + gap)) * a.scale;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) since[u] = exp2f(rate * (16 * u + c + 1)) * a.scale;

    for (int turn_of = 0; turn_of < (OUT ? a.turns : 1); ++turn_of) {
        const int member = (at + turn_of) * HEADS, head = kh * a.group + member;   // the first
        const bf16_t* q0 = OUT ? a.q + row0 * a.ld_q + static_cast<int64_t>(head) * a.D : nullptr;
        auto load = [&](int j) {
            const int64_t t = OUT ? j * kChunk : length - (j + 1) * kChunk;
            const int rows = OUT ? count - j * kChunk : kChunk;
            const bf16_t *q = q0 + t * a.ld_q, *k = k0 + t * a.ld_k, *v = v0 + t * a.ld_v;
            const char* to = smem + j % kStages * kStage;
            auto from = [&](int m) { return m < kLoadsQ ? q + m / (P / 2) * a.D : m < kLoadsQ + kLoadsK ? k : v; };
            if (rows >= kChunk) {
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    const int m = min(i * WAVES + wave, kLoads - 1);
                    dma16_at(from(m), off[i], to + m * 1024);
                }
                return;
            }
#pragma unroll 1
            for (int i = 0; i < kItems; ++i) {
                const int m = min(i * WAVES + wave, kLoads - 1);
                dma16_at(from(m), offset(m, rows - 1), to + m * 1024);
            }
        };
        if (chunks > 0) load(0);
        if (kStages == 3 && chunks > 1) load(1);

        // s[t][x][r]: row 32 (t / 2) + 8 g + 4 (t % 2) + r, column column_of(x, c)
        f32x4_t s[DT][TILES];
        const float* start = nullptr;
        if (OUT) {
            const int64_t size = static_cast<int64_t>(a.D) * a.E;
            if (segment > 0 || a.first_state == 2) start = a.states + (bk * (1 + (a.segments - 1) * a.pieces) + segment * a.pieces) * size;
            else if (a.first_state == 1) start = a.state_in + bk * size;
        }
        int from = lane;   // opaque, as below
        asm volatile("" : "+v"(from));
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int x = 0; x < TILES; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = t / 2 * 32 + (from >> 4) * 8 + t % 2 * 4 + r, e = column_of(x, from & 15);
                    s[t][x][r] = start && d < a.D && e < a.E ? start[d * a.E + e] : 0.f;
                }

        // The state is `faded` times what the accumulators hold: its decay is put off, as a factor of what is added, until
        // it comes to 2^-8 since `age` tokens. Applied in every chunk it took 128 of 662 vector instructions.
        int age = 0;
        float faded = 1.f;
        typedef uint32_t out_t __attribute__((ext_vector_type(2 * TILES)));
        out_t done[OUT ? HEADS : 1][2];   // the last chunk's outputs, columns column_of(0, 4 g) on of query c: they leave behind the next barrier
        auto store = [&](int j, int rows) {
            const int e = column_of(0, g * 4);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = u * 16 + c;
                typedef out_t Any __attribute__((aligned(8)));
                if (e < a.E && i < rows)
#pragma unroll
                    for (int h = 0; h < HEADS; ++h)
                        *reinterpret_cast<Any*>(a.out + (row0 + j * kChunk + i) * a.ld_o + static_cast<int64_t>(head + h) * a.E + e) = done[h][u];
            }
        };
        for (int j = 0; j < chunks; ++j) {
            // this wave's loads of chunk j have landed, those of chunk j + 1 may be on their way; behind the barrier
            // everyone's have, and chunk j - 1 has been read
            asm volatile("" ::: "memory");
            if (kStages == 3 && j + 1 < chunks) s_waitcnt<kItems, 0>();
            else s_waitcnt<0, 0>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const int rows = min(count - j * kChunk, kChunk);
            const char* image = smem + j % kStages * kStage;
            const char *qi = image, *ki = image + kLoadsQ * 1024, *vi = ki + kLoadsK * 1024;
            auto read_keys = [&](int t) {   // transposed
                const char* p = ki + (kt ^ (t / 2 * 64)) + t % 2 * 8;
                return __builtin_bit_cast(
                    bf16x8_t, __builtin_shufflevector(read_transposed(p), read_transposed(p + 16 * P * 16), 0, 1, 2, 3, 4, 5, 6, 7));
            };
            auto read_values = [&](int x) {
                const char* p = vi + (vt ^ (column / 8 * 16)) + x * 8;
                return __builtin_bit_cast(
                    bf16x8_t, __builtin_shufflevector(read_transposed(p), read_transposed(p + 16 * PV * 16), 0, 1, 2, 3, 4, 5, 6, 7));
            };
            if (OUT && j > 0) store(j - 1, kChunk);
            if (!active) {
                if (j + kStages - 1 < chunks) load(j + kStages - 1);
                continue;
            }
            // the transposed operands are read ahead of what comes before them: 8 x 2048 tokens of 32 heads of 64 74 us instead of 77
            bf16x8_t v[TILES], keys[2][2];   // keys: [pair of tiles % 2][tile]
            auto read_first = [&]() {
#pragma unroll
                for (int x = 0; x < TILES; ++x) v[x] = read_values(x);
#pragma unroll
                for (int y = 0; y < 2; ++y) keys[0][y] = read_keys(y);
            };
            if constexpr (OUT) {
                // by 32 rows of the state: scores of key tile y against query tile u >= y, and the state's part of the outputs
                const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
                __builtin_amdgcn_s_setprio(1);   // before the other wave's loads and values: 2 x 4096 tokens of 32 / 8 heads of 128, one at once, 84 us, without 88
                f32x4_t o[HEADS][TILES][2], score[HEADS][3];   // (0, 0), (0, 1), (1, 1)
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    bf16x8_t q[HEADS][2], kk[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int h = 0; h < HEADS; ++h) {
                            u32x4_t f = *reinterpret_cast<const u32x4_t*>(qi + (h * 32 + u * 16) * P * 16 + (frag ^ (k * 64)));
                            if (k == STEPS - 1 && k * 4 + g >= dc) f = u32x4_t{0, 0, 0, 0};   // past head_dim
                            q[h][u] = __builtin_bit_cast(bf16x8_t, f);
                        }
                        kk[u] = *reinterpret_cast<const bf16x8_t*>(ki + u * 16 * P * 16 + (frag ^ (k * 64)));
                    }
                    if (k + 1 == STEPS) read_first();
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        score[h][0] = product(kk[0], q[h][0], k == 0 ? zero : score[h][0]);
                        score[h][1] = product(kk[0], q[h][1], k == 0 ? zero : score[h][1]);
                        score[h][2] = product(kk[1], q[h][1], k == 0 ? zero : score[h][2]);
                    }
#pragma unroll
                    for (int x = 0; x < TILES; ++x) {
                        f32x4_t lo = s[2 * k][x], hi = s[2 * k + 1][x];
                        const u32x2_t l1 = take_bf16(lo), h1 = take_bf16(hi);
                        const bf16x8_t one = pair(l1, h1);
                        const bf16x8_t two = pair(u32x2_t{f2bf2(lo[0], lo[1]), f2bf2(lo[2], lo[3])}, u32x2_t{f2bf2(hi[0], hi[1]), f2bf2(hi[2], hi[3])});
#pragma unroll
                        for (int h = 0; h < HEADS; ++h)
#pragma unroll
                            for (int u = 0; u < 2; ++u) o[h][x][u] = product(one, q[h][u], k == 0 ? zero : o[h][x][u]);
#pragma unroll
                        for (int h = 0; h < HEADS; ++h)
#pragma unroll
                            for (int u = 0; u < 2; ++u) o[h][x][u] = product(two, q[h][u], o[h][x][u]);
                    }
                }
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float by = since[u] * faded;
#pragma unroll
                        for (int x = 0; x < TILES; ++x)
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[h][x][u][r] *= by;
                    }
                    // the chunk's own
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        score[h][0][r] *= own[r];
                        score[h][1][r] *= before[r];
                        score[h][2][r] *= own[r];
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f32x4_t lo = score[h][u], hi = u == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : score[h][2];
                        const u32x2_t l1 = take_bf16(lo), h1 = take_bf16(hi);
                        const bf16x8_t one = pair(l1, h1);
                        const bf16x8_t two = pair(u32x2_t{f2bf2(lo[0], lo[1]), f2bf2(lo[2], lo[3])}, u32x2_t{f2bf2(hi[0], hi[1]), f2bf2(hi[2], hi[3])});
#pragma unroll
                        for (int x = 0; x < TILES; ++x) {
                            o[h][x][u] = product(v[x], one, o[h][x][u]);
                            o[h][x][u] = product(v[x], two, o[h][x][u]);
                            done[h][u][2 * x] = f2bf2(o[h][x][u][0], o[h][x][u][1]);
                            done[h][u][2 * x + 1] = f2bf2(o[h][x][u][2], o[h][x][u][3]);
                        }
                    }
                }
            } else {
                read_first();
            }
            __builtin_amdgcn_s_setprio(0);
            if (j + kStages - 1 < chunks) load(j + kStages - 1);
            // the state behind the chunk
            float more;   // by which what is added here counts in the accumulators
            if (OUT) {
                age += rows;
                faded = __builtin_amdgcn_exp2f(rate * age);
                more = 1.f;
                if (faded < 0x1p-8f) {
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int x = 0; x < TILES; ++x)
#pragma unroll
                            for (int r = 0; r < 4; ++r) s[t][x][r] *= faded;
                    age = 0;
                    faded = 1.f;
                } else {
                    more = __builtin_amdgcn_exp2f(-rate * age);
                }
            } else {
                more = exp2f(rate * (j * kChunk));
            }
            float weight[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) weight[e] = to_end[e] * more;
            if (OUT && rows < kChunk)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int left = rows - 1 - ((e & 4) * 4 + 4 * g + (e & 3));
                    weight[e] = left >= 0 ? exp2f(rate * left) * more : 0.f;
                }
            bf16x8_t w[TILES][3];
#pragma unroll
            for (int x = 0; x < TILES; ++x) {
                const u32x4_t raw = __builtin_bit_cast(u32x4_t, v[x]);
                f32x4_t lo, hi;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    lo[2 * e] = __uint_as_float(raw[e] << 16) * weight[2 * e];
                    lo[2 * e + 1] = __uint_as_float(raw[e] & 0xffff0000u) * weight[2 * e + 1];
                    hi[2 * e] = __uint_as_float(raw[2 + e] << 16) * weight[4 + 2 * e];
                    hi[2 * e + 1] = __uint_as_float(raw[2 + e] & 0xffff0000u) * weight[4 + 2 * e + 1];
                }
#pragma unroll
                for (int z = 0; z < 3; ++z) {
                    const u32x2_t l = take_bf16(lo), h = take_bf16(hi);
                    w[x][z] = pair(l, h);
                }
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                if (k + 1 < STEPS)
#pragma unroll
                    for (int y = 0; y < 2; ++y) keys[(k + 1) & 1][y] = read_keys(2 * k + 2 + y);
#pragma unroll
                for (int z = 2; z >= 0; --z)
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int x = 0; x < TILES; ++x) s[2 * k + y][x] = product(keys[k & 1][y], w[x][z], s[2 * k + y][x]);
            }
        }
        if (OUT && chunks > 0 && active) store(chunks - 1, count - (chunks - 1) * kChunk);
        float* end = nullptr;
        if (!OUT) end = a.states + (bk * (1 + segments) + segment + 1) * a.D * a.E;
        else if (a.state_out && segment == last_segment && member + HEADS == a.group) end = a.state_out + bk * a.D * a.E;
        if (end) {
            if (age > 0) {   // of no tokens as it is, infinities too
                const Fade fade(age * log_decay);
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int x = 0; x < TILES; ++x)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][x][r] = fade(s[t][x][r]);
            }
            int here = lane;   // computed anew: the offsets of the first state's values would stay in registers through the loop
            asm volatile("" : "+v"(here));
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int x = 0; x < TILES; ++x)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d = t / 2 * 32 + (here >> 4) * 8 + t % 2 * 4 + r, e = column_of(x, here & 15);
                        if (d < a.D && e < a.E) end[d * a.E + e] = s[t][x][r];
                    }
        }
        if (OUT) {   // the outputs behind the sequence
            // by rows: a count of 8-byte pieces passes 2^31 from 2^26 rows of 128 columns on
            const int behind = max(n - first, 0), rows = min(a.N - first, length);
            const int pieces = a.E / 4, each = WAVES * 64 / pieces, piece = threadIdx.x % pieces;
            if (static_cast<int>(threadIdx.x) < each * pieces)
                for (int i = behind + threadIdx.x / pieces; i < rows; i += each)
#pragma unroll
                    for (int h = 0; h < HEADS; ++h)
                        *reinterpret_cast<uint2*>(a.out + (row0 + i) * a.ld_o + static_cast<int64_t>(head + h) * a.E + piece * 4) = make_uint2(0, 0);
            if (turn_of + 1 < a.turns) {   // the next heads' loads reuse the stages
                asm volatile("" ::: "memory");
                s_waitcnt<0, 0>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
        }
    }
}

// From the pieces' own states to the state before each segment; the first is state_in or zeros.
__global__ void __launch_bounds__(kThreads) k_linear_carry(LinearArgs a) {
    constexpr int kAhead = 16;   // loads on their way: with 8, 255 pieces of one head of 128 took 13 us longer
    const int64_t size = static_cast<int64_t>(a.D) * a.E / 4, i = group_index() * kThreads + threadIdx.x;
    const int64_t bk = i / size;
    if (bk >= static_cast<int64_t>(a.B) * a.KH) return;
    const int64_t b = bk / a.KH;
    const int n = a.lens ? min(max(a.lens[b], 0), a.N) : a.N, last = n > 0 ? (n - 1) / (a.length * a.pieces) * a.pieces : 0;
    const Fade fade(static_cast<float>(a.length) * log_decay_of(a, static_cast<int>(bk % a.KH)));
    f32x4_t s = a.state_in ? reinterpret_cast<const f32x4_t*>(a.state_in)[i] : f32x4_t{0.f, 0.f, 0.f, 0.f};
    f32x4_t* at = reinterpret_cast<f32x4_t*>(a.states) + bk * (1 + (a.segments - 1) * a.pieces) * size + (i - bk * size);
    *at = s;
    for (int m = 1; m <= last; m += kAhead) {
        f32x4_t own[kAhead];
#pragma unroll
        for (int x = 0; x < kAhead; ++x) own[x] = at[min(m + x, last) * size];
#pragma unroll
        for (int x = 0; x < kAhead; ++x)
            if (m + x <= last) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[r] = fade(s[r]) + own[x][r];
                if ((m + x) % a.pieces == 0) at[(m + x) * size] = s;
            }
    }
}

int device_cus() {
    static std::atomic<int> cus[64] = {};
    int dev = 0;
    hip_check(hipGetDevice(&dev), "hipGetDevice");
    require(dev >= 0 && dev < 64, "attention_linear: device index out of range");
    int n = cus[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        hip_check(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev), "hipDeviceGetAttribute");
        require(n > 0, "attention_linear: device reports no compute units");
        cus[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// How a call runs: token after token for one or two (one token of 16 sequences, 32 heads of 128: 14.8 us against 19.0 for a chunk,
// two 18.3 against 18.8, four 24.8 against 18.7), else chunks, each sequence in `segments`, for one query head or two at once.
// The estimates, in us, were fitted to 70 shapes on one MI355X (1 to 200 heads of 32 to 128 columns, 64 to 65536 tokens), each
// with one and two heads at once in 1 to 256 segments: what they choose is within 5% of the fastest measured on 61, and
// 12% above it at worst (5 x 3000 tokens of 32 / 8 heads of 128). A chunk takes a workgroup `step` alone on a CU (two heads 1.45
// times that), and beside others the CU `share` of it for each; a call no less than its bytes at 4.6 TB/s; the first launch 0.4
// of a step a chunk; a state's load or store 34 us a MB for a workgroup, and the launch between its states at 4.6 TB/s and 0.09 a
// piece. 4 x 2048 tokens of 32 heads of 128 whole 137 us, in 4 segments 107, in 16 208; one head of 128 with 8192 tokens
// whole 523, in 64 segments 37, in 256 62. Two heads at once share the state's update and its splitting, and leave half the
// workgroups: 32 x 300 tokens of 32 / 8 heads of 128 64 us against 87, 65536 tokens 409 against 526, but 2 x 300 of 64 / 8 heads of
// 64 19.6 against 16.3.
struct Plan {
    bool tokens;                    // k_linear_tokens
    int segments, pieces, length;   // as in LinearArgs
    int heads = 1;                  // of a group, that a workgroup takes at once
};
Plan plan(const LinearShape& sh, bool may_split, int64_t cus) {
    if (sh.seq_len <= 2) return Plan{true, 1, 1, static_cast<int>(sh.seq_len)};
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const int64_t chunks = up(sh.seq_len, kChunk), rows = sh.batch * sh.kv_heads, group = sh.heads / sh.kv_heads;
    // columns as the kernels compute them
    const double width = static_cast<double>(up(sh.head_dim, 32) * 32 + (sh.value_dim > 64 ? 128 : 64));
    const double step = 0.1 + 0.0071 * width, shares[] = {width >= 192 ? 0.82 : 0.73, width >= 192 ? 0.86 : 0.84};
    const double state = 4e-6 * static_cast<double>(sh.head_dim * sh.value_dim);   // MB
    const double bytes = 2.0 * static_cast<double>(sh.seq_len * rows * (group + 1) * (sh.head_dim + sh.value_dim));
    Plan best{false, 1, 1, static_cast<int>(chunks * kChunk)};
    double least = 1e30;
    for (int heads = 1; heads <= (group % 2 == 0 ? 2 : 1); ++heads)
        for (int64_t want = 1; want == 1 || (may_split && want <= 512 && 2 * want <= chunks); want *= 2)
            for (int64_t pieces = 1; pieces <= (want > 1 ? 2 : 1); ++pieces) {
                const int64_t each = up(up(chunks, want), pieces) * pieces, segments = up(chunks, each);
                const double groups = static_cast<double>(rows * (group / heads) * segments), c = static_cast<double>(cus);
                const double per = step * (heads == 2 ? 1.45 : 1.0) * std::max(1.0, shares[heads - 1] * std::ceil(groups / c));
                double cost = 5 + std::max(each * per + std::max(1.0, groups / c) * state * 34, bytes / 4.6e6);
                if (segments > 1) {
                    const double first = static_cast<double>(rows * (segments - 1) * pieces), all = static_cast<double>(segments * pieces);
                    cost += 3 + each / pieces * 0.4 * step * std::max(1.0, shares[0] * std::ceil(first / c)) + std::max(1.0, first / c) * state * 34;
                    cost += 3 + 0.09 * all + static_cast<double>(rows) * (all + segments) * state / 4.6;
                }
                if (cost < least) {
                    least = cost;
                    best = Plan{false, static_cast<int>(segments), static_cast<int>(pieces), static_cast<int>(each / pieces * kChunk), heads};
                }
            }
    return best;
}

template <int STEPS, int TILES, int WAVES, int HEADS>
void launch(const LinearArgs& a, int64_t groups, hipStream_t s) {
    k_linear_chunks<STEPS, TILES, WAVES, HEADS><<<grid_of(groups, WAVES * 64), WAVES * 64, 0, s>>>(a);
    launch_check("attention_linear");
}
// More than 64 value columns to four waves of 32, or where a workgroup has its CU to itself to eight of 16, which take a chunk in
// 0.9 of the time (8 heads of 128 with 100 tokens 16.3 us against 18.0; two heads at once in 0.94 to 1.02) and two workgroups' chunks
// in 1.2 of it.
template <int STEPS, int HEADS>
void by_values(const LinearArgs& a, int64_t groups, int64_t cus, hipStream_t s) {
    if (a.E <= 64) return launch<STEPS, 1, 4, HEADS>(a, groups, s);
    if constexpr (HEADS > 0)
        if (groups <= cus) return launch<STEPS, 1, 8, HEADS>(a, groups, s);
    launch<STEPS, 2, 4, HEADS>(a, groups, s);
}
template <int HEADS>
void by_width(const LinearArgs& a, int64_t groups, int64_t cus, hipStream_t s) {
    switch ((a.D + 31) / 32) {
        case 1: return by_values<1, HEADS>(a, groups, cus, s);
        case 2: return by_values<2, HEADS>(a, groups, cus, s);
        case 3: return by_values<3, HEADS>(a, groups, cus, s);
        default: return by_values<4, HEADS>(a, groups, cus, s);
    }
}

}  // namespace

int64_t attention_linear_workspace_floats(const LinearShape& sh) {
    const Plan how = plan(sh, true, device_cus());
    const int64_t states = sh.batch * sh.kv_heads * sh.head_dim * sh.value_dim;
    // one state each where some of a group's workgroups would still read what one of them writes
    return how.segments > 1 ? (1 + (how.segments - 1) * how.pieces) * states : !how.tokens && sh.heads / sh.kv_heads > how.heads ? states : 0;
}

bh_attention_linear_plan attention_linear_plan(const LinearShape& sh, bool may_split, int cus) {
    const Plan how = plan(sh, may_split, cus > 0 ? cus : device_cus());
    if (how.tokens) return bh_attention_linear_plan{1, 1, sh.batch * sh.kv_heads * ((sh.value_dim + 31) / 32)};
    return bh_attention_linear_plan{kChunk, how.segments, sh.batch * sh.heads / how.heads * how.segments};
}

void launch_attention_linear(const bf16_t* q, const bf16_t* k, const bf16_t* v, bf16_t* out, const LinearShape& sh,
                             const float* log_decay, const int32_t* lens, const float* state_in, float* state_out, float* ws,
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
    const int64_t cus = device_cus();
    const Plan how = plan(sh, ws != nullptr, cus);
    a.states = ws;
    a.segments = how.segments;
    a.pieces = how.pieces;
    a.length = how.length;
    ProfileScope ps(K_ATTN_SELF, s, 2.0 * sh.batch * sh.seq_len * (sh.heads + sh.kv_heads) * sh.head_dim * sh.value_dim);
    const int64_t rows = sh.batch * sh.kv_heads;
    if (how.tokens) {
        k_linear_tokens<<<grid_of(rows * a.slices, kThreads), kThreads, 0, s>>>(a);
        launch_check("attention_linear");
        return;
    }
    // a group's workgroups, where it has several, read the first state while one of them may end and write it in place
    const bool in_place = state_in && state_in == state_out && a.group > how.heads;
    const bool copied = how.segments > 1 || (in_place && ws);
    a.first_state = copied ? 2 : state_in ? 1 : 0;
    a.turns = in_place && !copied ? a.group / how.heads : 1;
    const int64_t groups = rows * how.segments * (a.group / how.heads / a.turns);
    require(groups < (int64_t{1} << 31) && rows * how.segments * how.pieces < (int64_t{1} << 31), "attention_linear: too many heads");
    if (how.segments > 1) by_width<0>(a, rows * (how.segments - 1) * how.pieces, cus, s);
    if (copied) {
        k_linear_carry<<<grid_of((rows * a.D * a.E / 4 + kThreads - 1) / kThreads, kThreads), kThreads, 0, s>>>(a);
        launch_check("attention_linear");
    }
    if (how.heads == 2) by_width<2>(a, groups, cus, s);
    else by_width<1>(a, groups, cus, s);
}

}  // namespace bh
