// Rotary positions with several axes: pair i of columns (u, v) of a head becomes
//   (u cos t - v sin t, u sin t + v cos t),  t = position[axis of i] * scale[axis] * frequency_i.
// The heads of a row share its angles, so a workgroup takes a few rows, computes their angles once into LDS and
// then streams the heads past them, q's and k's in one launch.
//
// An angle is formed in turns: position * (frequency / 2 pi) in fp64, whole turns taken off, and only the rest
// (below half a turn) rounded to fp32 for its sine and cosine. In fp32 the product alone would be off by
// position * 2^-24 radians. Host code computes the frequencies in fp64.
//
// Bound by HBM: 32256 rows of 24 + 24 heads of 128, bf16, 145 us (5.5 TB/s), 2 x 4096 of 16 + 16 heads of 72 15.1 us, of which a
// launch is 3; the angles are below the noise there (the hardware's sine gained nothing). A few rows are a launch.
#include "common.h"
#include "vec8.h"

#include <algorithm>
#include <cmath>

namespace bh {
namespace {

constexpr int kThreads = 256;

struct RopeArgs {
    const int32_t* positions;
    int64_t position_rows, rows;
    RopeSide q, k;
    int axes, pairs, head_dim;
    int sign;                       // of the sine
    int per;                        // rows a workgroup
    int vectors, items;             // of eight columns (pairs, where a pair's columns lie apart) per head, per row
    uint32_t by_pairs, by_vectors, by_items;   // floor(2^32 / n) + 1: the quotient of m by n is the high half of m times it
    double turns[kRopePairs];       // a pair's turns per position
    uint8_t axis[kRopePairs];
};

// WHOLE: a head's turned columns and those behind them are whole vectors.
template <typename T, bool INTERLEAVED, bool WHOLE>
__global__ void __launch_bounds__(kThreads) k_rope(RopeArgs a) {
    __shared__ float2 turn[1024];   // cos, sin: [row][pair]
    const int64_t row0 = group_index() * a.per;
    if (row0 >= a.rows) return;
    const int per = static_cast<int>(min(static_cast<int64_t>(a.per), a.rows - row0)), items = per * a.items;
    const int P = a.pairs, turned = (INTERLEAVED ? 2 * P + 7 : P + 7) / 8;

    // Item i: vector `vec` of a head of row `row`; the first columns it reads and writes.
    struct Item {
        const T* in;
        T* out;
        int row, vec, column;
    };
    auto item = [&](int i) {
        const int row = per == 1 ? 0 : a.items == 1 ? i : __umulhi(i, a.by_items), of_row = i - row * a.items;
        const int head = a.vectors == 1 ? of_row : __umulhi(of_row, a.by_vectors), vec = of_row - head * a.vectors;
        const bool of_q = head < a.q.heads;
        const int column = vec < turned ? vec * 8 : 2 * P + (vec - turned) * 8;
        const int64_t from = static_cast<int64_t>(of_q ? head : head - a.q.heads) * a.head_dim + column;
        return Item{static_cast<const T*>(of_q ? a.q.in : a.k.in) + (row0 + row) * (of_q ? a.q.ld_in : a.k.ld_in) + from,
                    static_cast<T*>(of_q ? a.q.out : a.k.out) + (row0 + row) * (of_q ? a.q.ld_out : a.k.ld_out) + from, row, vec, column};
    };
    // Its values: u, and where a pair's columns lie apart w. Those of the first item are on their way while the angles are found.
    constexpr bool kApart = !INTERLEAVED;
    Packed8<T> u, w;
    auto fetch = [&](const Item& it) {
        u.load(it.in);
        if (kApart && it.vec < turned) w.load(it.in + P);
    };
    Item it = item(min(static_cast<int>(threadIdx.x), items - 1));
    if constexpr (WHOLE) fetch(it);

    const int64_t at0 = row0 % a.position_rows;
    for (int i = threadIdx.x; i < per * P; i += kThreads) {
        const int r = P == 1 ? i : __umulhi(i, a.by_pairs), p = i - r * P;
        int64_t at = at0 + r;
        while (at >= a.position_rows) at -= a.position_rows;
        double t = a.positions[at * a.axes + a.axis[p]] * a.turns[p];
        t -= rint(t);
        float s, c;
        sincospif(2.0f * static_cast<float>(t), &s, &c);
        turn[i] = make_float2(c, a.sign < 0 ? -s : s);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += kThreads) {
        if (!WHOLE && i != static_cast<int>(threadIdx.x)) it = item(i);
        const float2* cs = turn + it.row * P;
        float x[8], y[8];
        if constexpr (WHOLE) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = u[e];
            if constexpr (kApart)
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = w[e];
        } else {
            load8(it.in, it.column, it.vec < turned ? (INTERLEAVED ? 2 * P : P) : a.head_dim, x);
            if (kApart && it.vec < turned) load8(it.in + P, it.column, P, y);
        }
        const Item now = it;
        if (WHOLE && i + kThreads < items) {
            it = item(i + kThreads);
            fetch(it);
        }
        if (now.vec >= turned) {
            store8(now.out, now.column, a.head_dim, x);
        } else if constexpr (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 t = cs[WHOLE ? now.vec * 4 + e : min(now.vec * 4 + e, P - 1)];
                const float v = x[2 * e];
                x[2 * e] = v * t.x - x[2 * e + 1] * t.y;
                x[2 * e + 1] = v * t.y + x[2 * e + 1] * t.x;
            }
            store8(now.out, now.column, 2 * P, x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 t = cs[WHOLE ? now.column + e : min(now.column + e, P - 1)];
                const float v = x[e];
                x[e] = v * t.x - y[e] * t.y;
                y[e] = v * t.y + y[e] * t.x;
            }
            store8(now.out, now.column, P, x);
            store8(now.out + P, now.column, P, y);
        }
    }
}

uint32_t reciprocal(int n) { return static_cast<uint32_t>((uint64_t{1} << 32) / n + 1); }

}  // namespace

void launch_rope(const bh_rope_axes& axes, const int32_t* positions, int64_t position_rows, const RopeSide& q, const RopeSide& k,
                 int64_t rows, int64_t head_dim, bool inverse, bool f32, hipStream_t s) {
    RopeArgs a = {};
    a.positions = positions;
    a.position_rows = position_rows;
    a.rows = rows;
    a.q = q;
    a.k = k;
    a.axes = axes.axes;
    a.head_dim = static_cast<int>(head_dim);
    a.sign = inverse ? -1 : 1;
    for (int x = 0; x < axes.axes; ++x) a.pairs += axes.pairs[x];
    // theta^(-m / n) = theta^(-8 (m / 8) / n) theta^(-(m % 8) / n): 16 powers for 64 pairs, whose 64 would take longer than the launch
    auto power = [&](int m, int n) { return std::pow(axes.theta, -static_cast<double>(m) / n); };
    bool finite = true;
    for (int x = 0, i = 0; x < axes.axes; ++x) {
        const int n = axes.joint ? a.pairs : axes.pairs[x], first = axes.joint ? i : 0;
        double low[8], high = 0.0;
        for (int b = 0; b < 8 && b < n; ++b) low[b] = power(b, n);
        for (int j = 0; j < axes.pairs[x]; ++j, ++i) {
            const int m = first + j;
            if (j == 0 || m % 8 == 0) high = power(m / 8 * 8, n);
            a.turns[i] = axes.scale[x] * (high * low[m % 8]) / (2.0 * M_PI);
            finite = finite && std::isfinite(a.turns[i] * 0x1p31);   // else a position times it, 0 too, is a NaN
            a.axis[i] = static_cast<uint8_t>(x);
        }
    }
    require(finite, "rope: a position times scale and frequency leaves the range of fp64");
    const bool interleaved = axes.interleaved != 0;
    const int turned = (interleaved ? 2 * a.pairs + 7 : a.pairs + 7) / 8;
    a.vectors = turned + (a.head_dim - 2 * a.pairs + 7) / 8;
    a.items = a.vectors * (q.heads + k.heads);
    // Several rows a workgroup where they are short and enough workgroups remain. Long ones by themselves: 32256 rows of 48 heads
    // of 128 (384 items) took 145 us, two to a workgroup 150, five 163. 8192 rows of 32 heads of 72 (288) are given two and took 15.1;
    // four took 14.7, but a limit that allows four of 288 items allows two of 384.
    a.per = static_cast<int>(std::min<int64_t>({16, 1024 / a.pairs, std::max(1, 640 / a.items), std::max<int64_t>(1, rows / 2048)}));
    a.by_pairs = reciprocal(a.pairs);
    a.by_vectors = reciprocal(a.vectors);
    a.by_items = reciprocal(a.items);
    const int64_t groups = (rows + a.per - 1) / a.per;
    require(groups < (int64_t{1} << 40), "rope: too many rows");
    const bool whole = (interleaved ? 2 * a.pairs : a.pairs) % 8 == 0 && (a.head_dim - 2 * a.pairs) % 8 == 0;
    auto choose = [&](auto value) {
        using T = decltype(value);
        return interleaved ? (whole ? &k_rope<T, true, true> : &k_rope<T, true, false>) : (whole ? &k_rope<T, false, true> : &k_rope<T, false, false>);
    };
    auto* kernel = f32 ? choose(float{}) : choose(bf16_t{});
    kernel<<<grid_of(groups, kThreads), kThreads, 0, s>>>(a);
    launch_check("rope");
}

}  // namespace bh
