// Rotary positions with several axes: pair i of columns (u, v) of a head becomes
//   (u cos t - v sin t, u sin t + v cos t),  t = position[axis of i] * scale[axis] * frequency_i.
// The heads of a row share its angles, so a workgroup takes a few rows, computes their angles once into LDS and
// then streams the heads past them, q's and k's in one launch.
//
// An angle is formed in turns: position * (frequency / 2 pi) in fp64, whole turns taken off, and only the rest
// (below half a turn) rounded to fp32 for its sine and cosine. In fp32 the product alone would be off by
// position * 2^-24 radians. Host code computes the frequencies in fp64.
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

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) k_rope(RopeArgs a) {
    __shared__ float2 turn[1024 + 2 * kRopePairs];   // cos, sin: [row][pair]
    const int64_t row0 = group_index() * a.per;
    if (row0 >= a.rows) return;
    const int per = static_cast<int>(min(static_cast<int64_t>(a.per), a.rows - row0));
    const int64_t at0 = row0 % a.position_rows;
    for (int i = threadIdx.x; i < per * a.pairs; i += kThreads) {
        const int r = a.pairs == 1 ? i : __umulhi(i, a.by_pairs), p = i - r * a.pairs;
        int64_t at = at0 + r;
        while (at >= a.position_rows) at -= a.position_rows;
        double t = a.positions[at * a.axes + a.axis[p]] * a.turns[p];
        t -= rint(t);
        float s, c;
        sincospif(2.0f * static_cast<float>(t), &s, &c);
        turn[i] = make_float2(c, a.sign < 0 ? -s : s);
    }
    __syncthreads();
    const int P = a.pairs, turned = (INTERLEAVED ? 2 * P + 7 : P + 7) / 8;
    for (int i = threadIdx.x; i < per * a.items; i += kThreads) {
        const int r = per == 1 || a.items == 1 ? (a.items == 1 ? i : 0) : __umulhi(i, a.by_items), item = i - r * a.items;
        const int head = a.vectors == 1 ? item : __umulhi(item, a.by_vectors), vec = item - head * a.vectors;
        const bool of_q = head < a.q.heads;
        const int64_t row = row0 + r, column = static_cast<int64_t>(of_q ? head : head - a.q.heads) * a.head_dim;
        const T* in = static_cast<const T*>(of_q ? a.q.in : a.k.in) + row * (of_q ? a.q.ld_in : a.k.ld_in) + column;
        T* out = static_cast<T*>(of_q ? a.q.out : a.k.out) + row * (of_q ? a.q.ld_out : a.k.ld_out) + column;
        const float2* cs = turn + r * P;
        if (vec >= turned) {
            float v[8];
            const int c = 2 * P + (vec - turned) * 8;
            load8(in + c, c, a.head_dim, v);
            store8(out + c, c, a.head_dim, v);
        } else if constexpr (INTERLEAVED) {
            float v[8];
            const int c = vec * 8;
            load8(in + c, c, 2 * P, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 t = cs[min(vec * 4 + e, P - 1)];
                const float u = v[2 * e], w = v[2 * e + 1];
                v[2 * e] = u * t.x - w * t.y;
                v[2 * e + 1] = u * t.y + w * t.x;
            }
            store8(out + c, c, 2 * P, v);
        } else {
            float u[8], w[8];
            const int c = vec * 8;
            load8(in + c, c, P, u);
            load8(in + P + c, c, P, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 t = cs[min(c + e, P - 1)];
                const float x = u[e];
                u[e] = x * t.x - w[e] * t.y;
                w[e] = x * t.y + w[e] * t.x;
            }
            store8(out + c, c, P, u);
            store8(out + P + c, c, P, w);
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
    for (int x = 0, i = 0; x < axes.axes; ++x)
        for (int j = 0; j < axes.pairs[x]; ++j, ++i) {
            const double power = axes.joint ? static_cast<double>(i) / a.pairs : static_cast<double>(j) / axes.pairs[x];
            a.turns[i] = axes.scale[x] * std::pow(axes.theta, -power) / (2.0 * M_PI);
            a.axis[i] = static_cast<uint8_t>(x);
        }
    const bool interleaved = axes.interleaved != 0;
    const int turned = (interleaved ? 2 * a.pairs + 7 : a.pairs + 7) / 8;
    a.vectors = turned + (a.head_dim - 2 * a.pairs + 7) / 8;
    a.items = a.vectors * (q.heads + k.heads);
    // several rows a workgroup where they are short and enough workgroups remain
    a.per = static_cast<int>(std::min<int64_t>({16, 1024 / a.pairs, std::max(1, 4096 / a.items), std::max<int64_t>(1, rows / 2048)}));
    a.by_pairs = reciprocal(a.pairs);
    a.by_vectors = reciprocal(a.vectors);
    a.by_items = reciprocal(a.items);
    const int64_t groups = (rows + a.per - 1) / a.per;
    require(groups < (int64_t{1} << 40), "rope: too many rows");
    auto* kernel = f32 ? (interleaved ? &k_rope<float, true> : &k_rope<float, false>)
                       : (interleaved ? &k_rope<bf16_t, true> : &k_rope<bf16_t, false>);
    kernel<<<grid_of(groups, kThreads), kThreads, 0, s>>>(a);
    launch_check("rope");
}

}  // namespace bh
