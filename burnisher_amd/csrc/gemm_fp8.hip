// The matrix product of two e4m3 matrices with a scale per block of 128 along K:
//   out[m, n] = act(sum over blocks j of sa[j, m] * sb[n / 128, j] * sum over k in block j of A[m, k] B[n, k] + bias[n])
// Rows of A and B are fp8_row_bytes(k) apart, zero from k on.
//
// A block's scales are outside its sum, so its products add up in the matrix instruction and one fp32
// multiply-add an output takes the sum over: v_mfma_f32_16x16x128_f8f6f4 covers the 128 of a block at once.
// Two kernels. Few rows are bound by the bytes of B: k_gemm_fp8_rows reads both operands from memory straight
// into the matrix instruction, its waves side by side along K. Many rows are bound by the matrix cores and by how
// fast their operands get to them: k_gemm_fp8_tile keeps rings of blocks in LDS; K goes to several workgroups
// where there are fewer tiles than CUs.
#include "common.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace bh {
namespace {

#include "gemm_tile.inc"

typedef int i32x8_t __attribute__((ext_vector_type(8)));

struct Fp8Args {
    const uint8_t* a;
    const float* sa;     // [blocks, m]
    const uint8_t* b;
    const float* sb;     // [n / 128, blocks]
    const void* bias;    // [n] in the output's type, or null
    void* out;           // [m, n]
    int64_t m, n, ld;    // ld: row bytes of a and b
    int blocks;          // of K
    int act;
    float* part = nullptr;   // K split over gridDim.y slices: slice s's sums go to part[s][m][n] instead
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

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Sixteen codes as two bf16 operands: every e4m3 value is a bf16 value.
__device__ __forceinline__ void widen16(u32x4_t c, bf16x8_t (&f)[2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.0f, false);
        const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.0f, true);
        bf16x8_t& d = f[i >> 1];
        const int o = (i & 1) * 4;
        d[o] = lo[0]; d[o + 1] = lo[1]; d[o + 2] = hi[0]; d[o + 3] = hi[1];
    }
}

// The product of one block of 128: lane (l, h) = (lane % 16, lane / 16) holds the same 32 of the block's
// columns of row l of either operand (`x0`, `x1`), so their order within the block does not matter.
// EXACT: through bf16 operands, whose products and sums are fp32; otherwise through the 8-bit matrix
// instruction, at twice the rate, which adds the products of eight neighbouring columns at a time and drops of each what
// lies below 2^-13 of the largest of the eight (measured with both shapes of it). That is for bf16 outputs, whose 2^-8
// is coarser wherever the products do not cancel.
template <bool EXACT>
__device__ __forceinline__ f32x4_t block_product(u32x4_t x0, u32x4_t x1, u32x4_t y0, u32x4_t y1) {
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
        const i32x8_t x = __builtin_bit_cast(i32x8_t, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
        const i32x8_t y = __builtin_bit_cast(i32x8_t, __builtin_shufflevector(y0, y1, 0, 1, 2, 3, 4, 5, 6, 7));
        d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, d, 0, 0, 0, 0, 0, 0);
    }
    return d;
}

// 16 bytes of a row at `off`, zeros past the row's end.
__device__ __forceinline__ u32x4_t chunk(const uint8_t* row, int64_t off, int64_t ld) {
    return off < ld ? *reinterpret_cast<const u32x4_t*>(row + off) : u32x4_t{0, 0, 0, 0};
}

// Workgroup: 16 columns x 16 MT rows; its waves take every kWaves-th block of K and their sums meet in LDS. Bound by
// B's bytes and, where those are few, by the launch: 1 x 20480 x 4096 20 us (4.2 TB/s), 16 x 12288 x 4096 14.8 us
// (3.4), 1 x 4096 x 4096 5.7 us. Loading two or four blocks before the first product was no faster: the waves beside
// it (24 a CU at 12288 columns) keep memory as busy.
constexpr int kWaves = 8;

template <int MT, bool EXACT, typename OUT>
__global__ void __launch_bounds__(kWaves * 64) k_gemm_fp8_rows(Fp8Args a) {
    __shared__ float part[kWaves][MT][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, h = lane >> 4;
    const int64_t tiles_n = (a.n + 15) / 16;
    const int64_t id = group_index(), n0 = id % tiles_n * 16, m0 = id / tiles_n * 16 * MT;
    if (m0 >= a.m) return;
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
        const u32x4_t b0 = chunk(brow, off, a.ld), b1 = chunk(brow, off + 16, a.ld);
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

// ---- many rows: MFMA tiles out of LDS -------------------------------------------------------------
//
// Workgroup: eight waves, four along M and two along N, a tile of 64 MT x 64 NP; a wave has 16 MT rows and
// 32 NP columns of it in registers. LDS rows are the 128 bytes of one block of K with the swizzle, the
// row permutations (a_row, b_col) and the direct-to-LDS loads of gemm_tile.inc, so a lane ends with 8
// consecutive columns of MT consecutive rows.
//
// A block's product starts from zero and its sum is added with the block's scales, one fp32 multiply-add
// an output: four beside every 32-cycle MFMA, which they hide under.
//
// Measured: 8192 x 8192 x 8192 1.95 us a 256 x 256 x 128 block, two waves a SIMD at 65% of the matrix instruction's own
// rate (what is left is LDS reads and issue; loads are not waited for); 8192 x 8192 x 1152 94 us (1650 TFLOP/s), 8192 x
// 4608 x 1152 57 to 62 us, where the nine blocks of K end in stores that all workgroups issue together; 600 x 4096 x 10240
// in three slices 41 to 43 us. fp32 outputs, through bf16 products: 8192 x 8192 x 2048 268 us (1026 TFLOP/s), of which
// widening the codes is 12%.
namespace tile {

constexpr int kThreads = 512;

// A and B have rings of their own in LDS, of kSA and kSB blocks of K: what is in flight behind the block that is
// multiplied sets the pace (a load takes about 1.5 us under this load), so A's is longer where B's has no room
// to follow. A block's scales travel in A's ring.
template <int MT, int NP>
struct Geom {
    static constexpr int BM = 64 * MT, BN = 64 * NP;
    static constexpr int kScaleBytes = 2048;         // eight runs of 64 floats: four of sa, one of sb, spares
    static constexpr int kA = BM * 128 + kScaleBytes, kB = BN * 128;
    static constexpr int kRoom = 160 * 1024;
    static constexpr int kSB = kRoom / (kA + kB) < 5 ? kRoom / (kA + kB) : 5;
    static constexpr int kSA = kSB < 5 && (kSB + 1) * kA + kSB * kB <= kRoom ? kSB + 1 : kSB;
    static constexpr int kOffB = kSA * kA, kBytes = kOffB + kSB * kB;
    static constexpr int kItems = MT + NP + 1;       // loads a wave issues per block: B's, A's, the scales
    // How many later loads may be in flight when a block is needed: those issued after its B, and after its A.
    // With `ahead` a block's first fragments are read while the one before it is multiplied, so it is needed one
    // step earlier.
    static constexpr int wait(bool ahead) {
        const int need = ahead ? 3 : 2, after_b = (kSB - need) * kItems + MT + 1, after_a = (kSA - need) * kItems;
        return after_b < after_a ? after_b : after_a;
    }
    static_assert(kSB >= 2 && wait(false) < 63 && kItems <= 2 * MT * NP, "LDS, vmcnt, multiply()");
};

template <int MT, int NP>
__device__ __forceinline__ void tile_at(int v, int tiles_m, int tiles_n, int group_m, int64_t& m0, int64_t& n0) {
    const int T = tiles_m * tiles_n;
    if ((T & 7) == 0) v = (v & 7) * (T >> 3) + (v >> 3);   // an XCD's tiles are neighbours
    const int group_size = group_m * tiles_n, g = v / group_size, first = g * group_m;
    const int gm = min(tiles_m - first, group_m), in_group = v - g * group_size;
    m0 = static_cast<int64_t>(first + in_group % gm) * (64 * MT);
    n0 = static_cast<int64_t>(in_group / gm) * (64 * NP);
}

// The next block of K to load of one operand: its tile, its slot, the tile's uniform base at K = 0 and this lane's
// offsets from it, R row blocks of eight LDS rows.
template <int R>
struct Stream {
    const uint8_t* base;
    uint32_t off[R];
    int tile, kb, slot = 0;
};
template <int R, typename Row>
__device__ __forceinline__ void set_rows(Stream<R>& s, const uint8_t* base, int64_t first, int64_t rows, int64_t ld, int wave,
                                         int lane, Row row_of) {
    s.base = base + first * ld;
#pragma unroll
    for (int r = 0; r < R; ++r) {   // LDS row blocks 8 r + wave; rows past the end repeat the last
        const int row = (r * 8 + wave) * 8 + (lane >> 3);
        const int64_t in = min(static_cast<int64_t>(row_of(row)), rows - 1 - first);
        s.off[r] = static_cast<uint32_t>(in * ld) + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    }
}
struct Scales {
    const float* base;       // sa at the tile's rows (waves 0-3) or sb at its first column (waves 4-7)
    int64_t step;            // floats per block of K
    uint32_t off;
};
template <int MT>
__device__ __forceinline__ void set_scales(Scales& s, const Fp8Args& p, int64_t m0, int64_t n0, int wave, int lane) {
    if (wave < 4) {
        s.base = p.sa + m0;
        s.step = p.m;
        s.off = static_cast<uint32_t>(min(static_cast<int64_t>((wave % MT) * 64 + lane), p.m - 1 - m0)) * 4;
    } else {                         // lane l: the scale of columns 32 l .. + 31
        const int64_t first = n0 / 128, l = min(static_cast<int64_t>(lane & 15) * 32, p.n - 1 - n0);
        s.base = p.sb + first * p.blocks;
        s.step = 1;
        s.off = static_cast<uint32_t>(((n0 + l) / 128 - first) * p.blocks) * 4;
    }
}

// A wave's operands of one block of K that its products start from: the activation fragments, the first weight
// fragment and the scales.
template <int MT, int NP>
struct Start {
    u32x4_t a0[MT], a1[MT], b0, b1;
    float s[MT], sn[NP];
};
// Where a wave reads them: its rows of A's and B's slots.
template <int MT, int NP>
struct Block {
    const char *a_rows, *b_rows;
    const float *sa, *sb;
    int off0, off1;
    __device__ __forceinline__ Block(const char* a, const char* b, int wm, int wn, int lr, int off0_, int off1_)
        : a_rows(a + wm * (16 * MT * 128)), b_rows(b + wn * (32 * NP * 128)),
          sa(reinterpret_cast<const float*>(a + Geom<MT, NP>::BM * 128) + wm * 16 * MT + lr * MT),
          sb(reinterpret_cast<const float*>(a + Geom<MT, NP>::BM * 128 + 4 * 256) + wn * NP), off0(off0_), off1(off1_) {}
    __device__ __forceinline__ void a(int i, u32x4_t& x0, u32x4_t& x1) const {
        x0 = *reinterpret_cast<const u32x4_t*>(a_rows + i * 2048 + off0);
        x1 = *reinterpret_cast<const u32x4_t*>(a_rows + i * 2048 + off1);
    }
    __device__ __forceinline__ void b(int j, u32x4_t& x0, u32x4_t& x1) const {
        x0 = *reinterpret_cast<const u32x4_t*>(b_rows + j * 2048 + off0);
        x1 = *reinterpret_cast<const u32x4_t*>(b_rows + j * 2048 + off1);
    }
    __device__ __forceinline__ void scales(float (&s)[MT], float (&sn)[NP]) const {
#pragma unroll
        for (int i = 0; i < MT; ++i) s[i] = sa[i];
#pragma unroll
        for (int q = 0; q < NP; ++q) sn[q] = sb[q];
    }
    __device__ __forceinline__ void start(Start<MT, NP>& t) const {
        b(0, t.b0, t.b1);
#pragma unroll
        for (int i = 0; i < MT; ++i) a(i, t.a0[i], t.a1[i]);
        scales(t.s, t.sn);
    }
};

// One block of K for a wave: 2 NP weight fragments against MT activation fragments, and the loads
// of later blocks beside the first products (`load(r)`, r < MT + NP + 1). `live` is 8, or in the last block of
// rows that end inside it the chunks of 16 that are left. The order is fixed by hand: a product's sum is added three
// products later, when the matrix instruction has written it (left to the scheduler each addition waits for its
// own), and a weight fragment is read one fragment ahead. With kAhead `f` comes in read, and leaves as `next`'s,
// each fragment read behind its last use, so the matrix cores do not wait for LDS at a block's start:
// 8192 x 8192 x 1152 on 128 x 128 tiles 131 -> 124 us.
template <int MT, int NP, bool EXACT>
constexpr bool kAhead = Geom<MT, NP>::kSB >= 4 && !EXACT;   // where the rings have the room (fp32: the registers spill)

template <int MT, int NP, bool EXACT, typename Load>
__device__ __forceinline__ void multiply(f32x4_t (&acc)[MT][2 * NP], Start<MT, NP>& f, const Block<MT, NP>& at,
                                         const Block<MT, NP>& next, int live, int hi, Load load) {
    using G = Geom<MT, NP>;
    constexpr int J = 2 * NP, kSteps = J * MT, kLag = 3;
    constexpr bool kEarly = kAhead<MT, NP, EXACT>;
    if (!kEarly) at.start(f);
    u32x4_t b0[2], b1[2];
    float sc[NP][MT];
    b0[0] = f.b0;
    b1[0] = f.b1;
    if (live < 8) {   // B's are finite where its row is
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            f.a0[i] &= hi < live ? ~0u : 0u;
            f.a1[i] &= 4 + hi < live ? ~0u : 0u;
        }
    }
    f32x4_t d[kLag + 1];
    auto add = [&](int n) {
        const int j = n / MT, i = n % MT;
        if ((j & 1) == 0) sc[j >> 1][i] = f.s[i] * f.sn[j >> 1];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][j][t] = __builtin_fmaf(d[n % (kLag + 1)][t], sc[j >> 1][i], acc[i][j][t]);
        asm volatile("" : "+v"(acc[i][j]));   // here, not sunk behind the loop
    };
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < kSteps; ++n) {
        const int j = n / MT, i = n % MT;
        if (i == 0) {
            if (j + 1 < J) at.b(j + 1, b0[(j + 1) & 1], b1[(j + 1) & 1]);
            else if (kEarly) next.b(0, b0[0], b1[0]);
        }
        d[n % (kLag + 1)] = block_product<EXACT>(b0[j & 1], b1[j & 1], f.a0[i], f.a1[i]);
        if (n >= kLag) add(n - kLag);
        if (kEarly && j == J - 1) next.a(i, f.a0[i], f.a1[i]);
        if (n < G::kItems) load(n);
        __builtin_amdgcn_sched_group_barrier(0x008, EXACT ? 4 : 1, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int n = kSteps - kLag; n < kSteps; ++n) add(n);
    if (kEarly) {
        f.b0 = b0[0];
        f.b1 = b1[0];
        next.scales(f.s, f.sn);
    }
}

template <typename OUT>
__device__ __forceinline__ float act_out(float v, int act) {
    if constexpr (sizeof(OUT) == 4) return activate(v, act);
    if (act == 1) return gk::gelu_tanh_fast(v);
    if (act == 2) return gk::silu_fast(v);
    return v;
}

// Eight values of the bias from column n, -0.0 (which adds nothing to any value) without one and past the end.
template <typename OUT>
__device__ __forceinline__ void load_bias(const OUT* bias, int64_t n, int64_t N, float (&b)[8]) {
    if (bias && n + 8 <= N) {
        if constexpr (sizeof(OUT) == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) b[e] = bias[n + e];
        } else {
            typedef u32x4_t Any __attribute__((aligned(2)));
            const u32x4_t w = *reinterpret_cast<const Any*>(bias + n);
            gk::unpack8(make_uint4(w[0], w[1], w[2], w[3]), b);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = bias && n + e < N ? ld_out(bias + n + e) : -0.0f;
}

// The value of the neighbouring lane, lane ^ 1.
__device__ __forceinline__ uint32_t swap_pair(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xb1, 0xf, 0xf, true));   // quad_perm 1 0 3 2
}

// 16 bytes of a row that starts anywhere: memory takes them at the alignment of an element (8192 x 8191 x 1152 135 us,
// element by element 209).
template <bool LINES, typename V, typename T>
__device__ __forceinline__ void store16(V v, T* p) {
    typedef V Any __attribute__((aligned(sizeof(T))));
    if constexpr (LINES) __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
    else *reinterpret_cast<Any*>(p) = v;
}

// A tile that lies inside the output. Lanes lr and lr ^ 1 exchange halves, so that eight lanes
// write 128 consecutive bytes of a row. LINES: those are whole lines, which go past the caches (8192 x 8192 x 1152:
// 107 -> 94 us). Parts of lines are left for L2 to put together (8192 x 4616 x 1152 68 us, past the caches 75).
template <int MT, int NP, typename OUT, bool LINES>
__device__ __forceinline__ void store_inside(const f32x4_t (&acc)[MT][2 * NP], const float (&b)[NP][8], OUT* out, int64_t N,
                                             int act, int64_t m0, int64_t n0, int wm, int wn, int lr, int hi) {
    const bool odd = lr & 1;
    const int64_t row0 = m0 + wm * 16 * MT + (lr & ~1) * MT;   // of the lane's pair: row0 + i and row0 + MT + i
    if constexpr (sizeof(OUT) == 4) {
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int64_t n = n0 + (wn * NP + q) * 32 + hi * 8 + odd * 4;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                f32x4_t even_row, odd_row;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = act_out<OUT>(acc[i][2 * q][e] + b[q][e], act);
                    const float up = act_out<OUT>(acc[i][2 * q + 1][e] + b[q][4 + e], act);
                    const float got = __uint_as_float(swap_pair(__float_as_uint(odd ? lo : up)));
                    even_row[e] = odd ? got : lo;
                    odd_row[e] = odd ? up : got;
                }
                OUT* dst = out + (row0 + i) * N + n;
                store16<LINES>(even_row, dst);
                store16<LINES>(odd_row, dst + MT * N);
            }
        }
    } else {
        auto pair = [&](int i, int q, int e) {
            const f32x4_t& f = acc[i][2 * q + (e >> 1)];
            return f2bf2(act_out<OUT>(f[2 * (e & 1)] + b[q][2 * e], act), act_out<OUT>(f[2 * (e & 1) + 1] + b[q][2 * e + 1], act));
        };
#pragma unroll
        for (int q = 0; q + 1 < NP; q += 2) {
            const int64_t n = n0 + (wn * NP + q + odd) * 32 + hi * 8;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                u32x4_t even_row, odd_row;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w0 = pair(i, q, e), w1 = pair(i, q + 1, e), got = swap_pair(odd ? w0 : w1);
                    even_row[e] = odd ? got : w0;
                    odd_row[e] = odd ? w1 : got;
                }
                OUT* dst = out + (row0 + i) * N + n;
                store16<LINES>(even_row, dst);
                store16<LINES>(odd_row, dst + MT * N);
            }
        }
        if constexpr (NP % 2 == 1) {   // half lines of its own rows
            constexpr int q = NP - 1;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                u32x4_t w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pair(i, q, e);
                store16<LINES>(w, out + (m0 + wm * 16 * MT + lr * MT + i) * N + n0 + (wn * NP + q) * 32 + hi * 8);
            }
        }
    }
}

// A lane's 8 consecutive columns of MT rows a column pair. The bias is read before the first store: vmcnt counts loads and
// stores in order, so a load behind a store waits until memory has taken that.
template <int MT, int NP, typename OUT>
__device__ __forceinline__ void store(const f32x4_t (&acc)[MT][2 * NP], const Fp8Args& p, int64_t m0, int64_t n0,
                                      int wm, int wn, int lr, int hi) {
    OUT* out = static_cast<OUT*>(p.out);
    const int64_t m = m0 + wm * 16 * MT + lr * MT;
    float b[NP][8];
#pragma unroll
    for (int q = 0; q < NP; ++q)
        load_bias(static_cast<const OUT*>(p.bias), n0 + (wn * NP + q) * 32 + hi * 8, p.n, b[q]);
    if (m0 + 64 * MT <= p.m && n0 + 64 * NP <= p.n) {   // uniform: the whole tile
        if (((reinterpret_cast<uintptr_t>(out) | p.n * sizeof(OUT)) & 127) == 0) {
            asm volatile("");   // here and behind, or the two calls become one of ordinary stores
            store_inside<MT, NP, OUT, true>(acc, b, out, p.n, p.act, m0, n0, wm, wn, lr, hi);
            asm volatile("");
        } else {
            store_inside<MT, NP, OUT, false>(acc, b, out, p.n, p.act, m0, n0, wm, wn, lr, hi);
        }
        return;
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        const int64_t n = n0 + (wn * NP + q) * 32 + hi * 8;
        if (n >= p.n) continue;
        const bool whole = n + 8 <= p.n;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if (m + i >= p.m) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = act_out<OUT>(acc[i][2 * q + (e >> 2)][e & 3] + b[q][e], p.act);
            OUT* dst = out + (m + i) * p.n + n;
            if (whole) {
                if constexpr (sizeof(OUT) == 4) {
                    store16<false>(f32x4_t{v[0], v[1], v[2], v[3]}, dst);
                    store16<false>(f32x4_t{v[4], v[5], v[6], v[7]}, dst + 4);
                } else {
                    const uint4 w = gk::pack8(v);
                    store16<false>(u32x4_t{w.x, w.y, w.z, w.w}, dst);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n + e < p.n) st_out(dst + e, v[e]);
            }
        }
    }
}

// The sums of one slice of K: no bias, no activation.
template <int MT, int NP>
__device__ __forceinline__ void store_partial(const f32x4_t (&acc)[MT][2 * NP], const Fp8Args& p, int slice, int64_t m0,
                                              int64_t n0, int wm, int wn, int lr, int hi) {
    float* part = p.part + slice * p.m * p.n;
    if (m0 + 64 * MT <= p.m && n0 + 64 * NP <= p.n) {
        float b[NP][8];
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) b[q][e] = -0.0f;
        store_inside<MT, NP, float, false>(acc, b, part, p.n, 0, m0, n0, wm, wn, lr, hi);
        return;
    }
    const int64_t m = m0 + wm * 16 * MT + lr * MT;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t n = n0 + (wn * NP + q) * 32 + hi * 8 + h * 4;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (m + i >= p.m || n >= p.n) continue;
                float* dst = part + (m + i) * p.n + n;
                if (n + 4 <= p.n) {
                    store16<false>(acc[i][2 * q + h], dst);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n + e < p.n) dst[e] = acc[i][2 * q + h][e];
                }
            }
        }
}

// Persistent: a workgroup walks tiles blockIdx.x, + gridDim.x, ..., and its blocks of K run on across them,
// kSA - 1 of A and kSB - 1 of B ahead of the products.
template <int MT, int NP, bool EXACT, typename OUT>
__global__ void __launch_bounds__(kThreads, 1) k_gemm_fp8_tile(Fp8Args p, int tiles_m, int tiles_n, int group_m) {
    using G = Geom<MT, NP>;
    constexpr bool kEarly = kAhead<MT, NP, EXACT>;
    __shared__ __attribute__((aligned(1024))) char smem[G::kBytes];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave >> 1, wn = wave & 1, lr = lane & 15, hi = lane >> 4, sw = (lane >> 1) & 7;
    const int off0 = lr * 128 + ((hi ^ sw) * 16), off1 = lr * 128 + (((4 + hi) ^ sw) * 16);
    const int slice = blockIdx.y, slices = gridDim.y;
    const int kb0 = static_cast<int>(static_cast<int64_t>(slice) * p.blocks / slices);
    const int kb1 = static_cast<int>(static_cast<int64_t>(slice + 1) * p.blocks / slices);   // this slice's blocks of K
    const int KT = kb1 - kb0, grid = static_cast<int>(gridDim.x), tiles = tiles_m * tiles_n;
    const int total = (tiles - static_cast<int>(blockIdx.x) + grid - 1) / grid * KT;
    // Rows that end inside a block of K: the chunks of 16 that the last block has, and for a lane whose chunk lies
    // past them the distance back to the block's first chunk, which it loads instead (multiply() takes it as zero).
    const int last = static_cast<int>((p.ld - 1) / 16 % 8) + 1;
    const int chunk = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4));
    const uint32_t past = chunk >= last ? chunk * 16 : 0;

    Stream<MT> a;
    Stream<NP> b;
    Scales s;
    auto set_a = [&]() {
        int64_t m0, n0;
        tile_at<MT, NP>(a.tile, tiles_m, tiles_n, group_m, m0, n0);
        set_rows(a, p.a, m0, p.m, p.ld, wave, lane, [](int r) { return gk::a_row<MT>(r); });
        set_scales<MT>(s, p, m0, n0, wave, lane);
    };
    auto set_b = [&]() {
        int64_t m0, n0;
        tile_at<MT, NP>(b.tile, tiles_m, tiles_n, group_m, m0, n0);
        set_rows(b, p.b, n0, p.n, p.ld, wave, lane, [](int r) { return gk::b_col<4 * NP>(r); });
    };
    // To the next block of K; past the last one it is loaded again, into slots that nobody reads.
    auto advance = [&](auto& t, int slots, auto set) {
        t.slot = t.slot == slots - 1 ? 0 : t.slot + 1;
        if (++t.kb < kb1) return;
        if (t.tile + grid >= tiles) {
            t.kb = kb1 - 1;
            return;
        }
        t.kb = kb0;
        t.tile += grid;
        set();
    };
    auto back = [&](int kb) { return kb == p.blocks - 1 ? past : 0u; };
    auto load_a = [&](int r, uint32_t bk) {
        dma16_at(a.base + static_cast<int64_t>(a.kb) * 128, a.off[r] - bk, smem + a.slot * G::kA + (r * 8 + wave) * 1024);
    };
    auto load_b = [&](int r, uint32_t bk) {
        dma16_at(b.base + static_cast<int64_t>(b.kb) * 128, b.off[r] - bk, smem + G::kOffB + b.slot * G::kB + (r * 8 + wave) * 1024);
    };
    auto load_scales = [&]() { dma4_at(s.base + a.kb * s.step, s.off, smem + a.slot * G::kA + G::BM * 128 + wave * 256); };

    a.tile = b.tile = blockIdx.x;
    a.kb = b.kb = kb0;
    set_a();
    set_b();
#pragma unroll
    for (int g = 0; g < G::kSA - 1; ++g) {
        if (g < G::kSB - 1) {
#pragma unroll
            for (int r = 0; r < NP; ++r) load_b(r, back(b.kb));
            advance(b, G::kSB, set_b);
        }
#pragma unroll
        for (int r = 0; r < MT; ++r) load_a(r, back(a.kb));
        load_scales();
        advance(a, G::kSA, set_a);
    }
    auto block = [&](int sa, int sb) {
        return Block<MT, NP>(smem + sa * G::kA, smem + G::kOffB + sb * G::kB, wm, wn, lr, off0, off1);
    };
    Start<MT, NP> start;
    if (kEarly) {   // everything of block 0
        gk::wait_and_join<(G::kSB - 2) * G::kItems>();
        block(0, 0).start(start);
    }
    f32x4_t acc[MT][2 * NP];
    int tile = blockIdx.x, kb = 0, sa = 0, sb = 0;
    for (int g = 0; g < total; ++g) {
        if (kb == 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 2 * NP; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        // Block g (with kAhead, block g + 1) has landed -- this wave's part, and behind the barrier everyone's -- and
        // everyone has read block g - 1, whose slots take the next blocks. With kAhead the reads that may still be under
        // way are of block g, whose slots stay.
        asm volatile("" ::: "memory");
        s_waitcnt<G::wait(kEarly), kEarly ? 15 : 0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const uint32_t back_a = back(a.kb), back_b = back(b.kb);
        const int sa1 = sa == G::kSA - 1 ? 0 : sa + 1, sb1 = sb == G::kSB - 1 ? 0 : sb + 1;
        multiply<MT, NP, EXACT>(acc, start, block(sa, sb), block(sa1, sb1), kb0 + kb == p.blocks - 1 ? last : 8, hi, [&](int r) {
            if (r < NP) load_b(r, back_b);
            else if (r < NP + MT) load_a(r - NP, back_a);
            else load_scales();
        });
        advance(b, G::kSB, set_b);
        advance(a, G::kSA, set_a);
        sa = sa1;
        sb = sb1;
        if (++kb == KT) {
            int64_t m0, n0;
            tile_at<MT, NP>(tile, tiles_m, tiles_n, group_m, m0, n0);
            if (slices > 1) store_partial<MT, NP>(acc, p, slice, m0, n0, wm, wn, lr, hi);
            else store<MT, NP, OUT>(acc, p, m0, n0, wm, wn, lr, hi);
            kb = 0;
            tile += grid;
        }
    }
    gk::wait_and_join<0>();   // the trailing copies have landed before the LDS is given back
}

// The slices' sums in slice order, the bias and the activation: four columns a thread. Bound by bytes: three slices of
// 600 x 4096 7.1 us, 34 MB at 4.8 TB/s.
template <typename OUT>
__global__ void __launch_bounds__(256) k_sum_slices(Fp8Args p, int slices) {
    const int64_t at = (group_index() * 256 + threadIdx.x) * 4, size = p.m * p.n;
    if (at >= size) return;
    OUT* out = static_cast<OUT*>(p.out);
    const OUT* bias = static_cast<const OUT*>(p.bias);
    if (at + 4 <= size && p.n >= 4) {
        typedef f32x4_t Any __attribute__((aligned(4)));
        f32x4_t v = *reinterpret_cast<const f32x4_t*>(p.part + at);
        for (int s = 1; s < slices; ++s) v += *reinterpret_cast<const Any*>(p.part + s * size + at);
        const int64_t col = at % p.n;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = act_out<OUT>(bias ? v[e] + ld_out(bias + (col + e < p.n ? col + e : col + e - p.n)) : v[e], p.act);
        if constexpr (sizeof(OUT) == 4) {
            store16<false>(v, out + at);
        } else {
            typedef uint32_t Pair __attribute__((ext_vector_type(2)));
            store16<false>(Pair{f2bf2(v[0], v[1]), f2bf2(v[2], v[3])}, out + at);
        }
        return;
    }
    for (int64_t i = at; i < min(at + 4, size); ++i) {
        float v = p.part[i];
        for (int s = 1; s < slices; ++s) v += p.part[s * size + i];
        if (bias) v += ld_out(bias + i % p.n);
        st_out(out + i, act_out<OUT>(v, p.act));
    }
}

template <int MT, int NP, bool EXACT, typename OUT>
void launch(const Fp8Args& p, int slices, int64_t workgroups, hipStream_t s) {
    const int tiles_m = static_cast<int>((p.m + 64 * MT - 1) / (64 * MT)), tiles_n = static_cast<int>((p.n + 64 * NP - 1) / (64 * NP));
    k_gemm_fp8_tile<MT, NP, EXACT, OUT>
        <<<dim3(static_cast<unsigned>(workgroups), slices), kThreads, 0, s>>>(p, tiles_m, tiles_n, std::max(1, 16 / MT));
    if (slices == 1) return;
    launch_check("gemm_fp8");
    const int64_t blocks = (p.m * p.n + 1023) / 1024;
    k_sum_slices<OUT><<<grid_of(blocks, 256), 256, 0, s>>>(p, slices);
}

}  // namespace tile

int device_cus() {
    static std::atomic<int> cus[64] = {};
    int dev = 0;
    hip_check(hipGetDevice(&dev), "hipGetDevice");
    require(dev >= 0 && dev < 64, "gemm_fp8: device index out of range");
    int n = cus[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        hip_check(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev), "hipDeviceGetAttribute");
        require(n > 0, "gemm_fp8: device reports no compute units");
        cus[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Workgroups that walk a slice's tiles, one a CU at once. A multiple of eight keeps the tiles that a workgroup goes on
// to on its XCD, but not where that many would take a round more.
int64_t workgroups(int64_t tiles, int slices, int64_t cus) {
    const int64_t most = std::max<int64_t>(1, cus / slices), even = most & ~int64_t{7};
    auto rounds = [&](int64_t n) { return (tiles + n - 1) / n; };
    return std::min(tiles, even > 0 && rounds(even) == rounds(most) ? even : most);
}

// How a product runs: `mt` 16-row tiles of the rows kernel, or 64 mt x 64 np tiles with K in `slices`. Estimated
// times in ns. Fitted to one MI355X, 8192 x 8192 x 4096 on each tile: a block of K costs a workgroup 1.56 an
// operand row and 0.0176 an output (twice that through bf16 operands), a tile's end 0.072 a bf16 output and
// 0.16 an fp32 one: 256 x 256 tiles 1.95 us a block, 256 x 192 1.56 (measured 1.45), 256 x 128 1.18,
// 128 x 192 0.93, 128 x 128 0.69. Slices add a launch, 2400, and their fp32 sums, written and read. The rows kernel
// takes 140 or 250 for a block of K of 16 columns and 16 or 32, or 64 rows. What that chooses is within 7% of the fastest
// tile and number of slices on 63 of 64 products of 24 to 8192 rows, both output types (the other 14%: 128 x 4096 x 4096,
// eight slices 20.0 us, three 17.5).
struct Plan {
    bool tiles;
    int mt, np, slices;
    int64_t groups;   // workgroups, of each slice
};
Plan plan(int64_t m, int64_t n, int64_t k, bool f32, bool may_split, int64_t cus) {
    const int64_t blocks = (k + 127) / 128;
    const int rows_mt = m > 32 ? 4 : m > 16 ? 2 : 1;
    const int64_t groups = (n + 15) / 16 * ((m + 16 * rows_mt - 1) / (16 * rows_mt));
    Plan best{false, rows_mt, 0, 1, groups};
    if (m <= 16 || blocks == 0 || k >= (int64_t{1} << 22)) return best;   // 32-bit offsets inside a tile
    double least = std::max(1.0, static_cast<double>(groups) / cus) * blocks * (rows_mt == 4 ? 250 : 140);
    static constexpr int kTiles[][2] = {{4, 4}, {4, 3}, {4, 2}, {2, 4}, {2, 3}, {2, 2}};
    for (const auto& tile : kTiles) {
        const int64_t bm = 64 * tile[0], bn = 64 * tile[1], tiles = ((m + bm - 1) / bm) * ((n + bn - 1) / bn);
        if (tiles >= (int64_t{1} << 31) || (f32 && tile[0] + tile[1] > 7)) continue;   // 256 x 256 in fp32 spills
        for (int s = 1; s <= (may_split ? 8 : 1) && s <= blocks; ++s) {
            const int64_t at_once = workgroups(tiles, s, cus);
            const double rounds = static_cast<double>((tiles + at_once - 1) / at_once);
            double cost = rounds * ((blocks + s - 1) / s * (1.56 * (bm + bn) + (f32 ? 0.0352 : 0.0176) * bm * bn) +
                                    (f32 || s > 1 ? 0.16 : 0.072) * bm * bn);
            if (s > 1) cost += 2400 + (s * 4 + (f32 ? 4 : 2)) * static_cast<double>(m) * n / 5300;
            if (cost < least) {
                least = cost;
                best = Plan{true, tile[0], tile[1], s, at_once};
            }
        }
    }
    return best;
}

}  // namespace

int64_t gemm_fp8_workspace_floats(int64_t m, int64_t n, int64_t k, bool f32) {
    const Plan p = plan(m, n, k, f32, true, device_cus());
    return p.slices > 1 ? p.slices * m * n : 0;
}

bh_gemm_fp8_plan gemm_fp8_plan(int64_t m, int64_t n, int64_t k, bool f32, bool may_split, int cus) {
    const Plan p = plan(m, n, k, f32, may_split, cus > 0 ? cus : device_cus());
    const int rows = p.tiles ? 64 * p.mt : 16 * p.mt, cols = p.tiles ? 64 * p.np : 16;
    return bh_gemm_fp8_plan{p.tiles ? 1 : 0, rows, cols, p.slices, (m + rows - 1) / rows * ((n + cols - 1) / cols), p.groups};
}

void launch_gemm_fp8(const uint8_t* a, const float* sa, const uint8_t* b, const float* sb, const void* bias, void* out,
                     int64_t m, int64_t n, int64_t k, int act, bool f32, float* ws, hipStream_t s) {
    Fp8Args p{a, sa, b, sb, bias, out, m, n, fp8_row_bytes(k), static_cast<int>((k + 127) / 128), act, ws};
    ProfileScope ps(K_GEMM, s, 2.0 * m * n * k);
    const Plan how = plan(m, n, k, f32, ws != nullptr, device_cus());
    if (how.tiles) {
        auto go = [&](auto mt, auto np) {
            constexpr int MT = decltype(mt)::value, NP = decltype(np)::value;
            if constexpr (MT + NP <= 7) {
                if (f32) return tile::launch<MT, NP, true, float>(p, how.slices, how.groups, s);
            }
            tile::launch<MT, NP, false, bf16_t>(p, how.slices, how.groups, s);
        };
        constexpr std::integral_constant<int, 2> two;
        constexpr std::integral_constant<int, 3> three;
        constexpr std::integral_constant<int, 4> four;
        if (how.mt == 4) how.np == 4 ? go(four, four) : how.np == 3 ? go(four, three) : go(four, two);
        else how.np == 4 ? go(two, four) : how.np == 3 ? go(two, three) : go(two, two);
        launch_check("gemm_fp8");
        return;
    }
    const int mt = how.mt;
    const int64_t grid = how.groups;
    require(grid < (int64_t{1} << 31), "gemm_fp8: the output is too large");
    auto launch = [&](void (*kernel)(Fp8Args)) { kernel<<<grid_of(grid, kWaves * 64), kWaves * 64, 0, s>>>(p); };
    if (mt == 1) launch(f32 ? &k_gemm_fp8_rows<1, true, float> : &k_gemm_fp8_rows<1, false, bf16_t>);
    else if (mt == 2) launch(f32 ? &k_gemm_fp8_rows<2, true, float> : &k_gemm_fp8_rows<2, false, bf16_t>);
    else launch(f32 ? &k_gemm_fp8_rows<4, true, float> : &k_gemm_fp8_rows<4, false, bf16_t>);
    launch_check("gemm_fp8");
}

}  // namespace bh
