"""bh_rope on the GPU against the rotation in 64 bits on the same inputs.

The tolerance counts what is rounded: the rest of an angle, below half a turn, to fp32 (2^-26 turns, 2^-23.3
radians), sine and cosine (at most 4 ulp, 2^-22), the product's two roundings (2^-24 of |u| + |v| each), all
below 2^-21 (|u| + |v|), then the output's rounding. The 64-bit angle itself is off by a few 2^-53 of its size.
"""
import ctypes
import math

import pytest

import burnisher_amd as bh

pytestmark = pytest.mark.gpu


def dtypes():
    import torch
    return {"bf16": (torch.bfloat16, bh.BF16), "f32": (torch.float32, bh.F32)}


def normal(shape, seed, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def plain(x, positions, axes, inverse=False):
    """(turned x, tolerance) in 64 bits; x [rows, heads, head_dim]."""
    import torch
    pairs = list(axes.pairs)[:axes.axes]
    total, v = sum(pairs), x.double()
    out, tol = v.clone(), torch.zeros_like(v)
    rows = torch.arange(x.shape[0], device="cuda") % positions.shape[0]
    i = 0
    for a, count in enumerate(pairs):
        for j in range(count):
            f = axes.theta ** -(i / total if axes.joint else j / count) * axes.scale[a]
            t = positions[rows, a].double() * f * (-1 if inverse else 1)
            slack = (t.abs() * 2.0 ** -50)[:, None]
            c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
            n, m = (2 * i, 2 * i + 1) if axes.interleaved else (i, total + i)
            u, w = v[..., n], v[..., m]
            out[..., n], out[..., m] = u * c - w * s, u * s + w * c
            tol[..., n] = tol[..., m] = (u.abs() + w.abs()) * (2.0 ** -21 + slack)
            i += 1
    return out, tol + out.abs() * (torch.finfo(x.dtype).eps / 2)


def run(axes, positions, q, k, q_out, k_out, inverse=0, stream=None):
    """Operands [rows, heads, head_dim], views of any row stride; k may be None."""
    ld = lambda t: 0 if t is None else t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1] * t.shape[2])  # noqa: E731
    code = {2: bh.BF16, 4: bh.F32}[q.element_size()]
    bh.call("bh_rope", ctypes.byref(axes), positions.data_ptr(), positions.shape[0], q.data_ptr(), ld(q), q_out.data_ptr(),
            ld(q_out), q.shape[1], bh.ptr(k), ld(k), bh.ptr(k_out), ld(k_out), 0 if k is None else k.shape[1], q.shape[0],
            q.shape[2], inverse, code, bh.stream_ptr(stream))


def compare(got, x, positions, axes, inverse=False):
    want, tol = plain(x, positions, axes, inverse)
    bad = ~((got.double() - want).abs() <= tol)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {at}: {got[at]} for {want[at]}")


def grid(rows, axes, seed, low=-50, high=5000):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(low, high, (rows, axes), generator=g, device="cuda", dtype=torch.int32)


PAIRS = [([32], 64), ([16, 24, 24], 128), ([18, 18], 72), ([1], 2), ([1], 8), ([5, 0, 6], 25), ([3, 4], 20), ([8, 20, 12], 96),
         ([2, 2, 2, 2], 16), ([128], 256), ([7], 1024), ([13], 27)]


@pytest.mark.parametrize("joint,interleaved", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("pairs,head_dim", PAIRS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_axes_and_layouts(hip, dtype, pairs, head_dim, joint, interleaved):
    import torch
    t = dtypes()[dtype][0]
    axes = bh.RopeAxes.of(pairs, joint=joint, interleaved=interleaved)
    for rows, heads, kv_heads, at in ((1, 1, 1, 1), (37, 3, 1, 37), (50, 4, 2, 10)):
        q, k = normal((rows, heads, head_dim), 1, t), normal((rows, kv_heads, head_dim), 2, t)
        positions = grid(at, len(pairs), rows)
        q_out, k_out = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
        run(axes, positions, q, k, q_out, k_out)
        compare(q_out, q, positions, axes)
        compare(k_out, k, positions, axes)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,heads", [(5000, 1), (3001, 2), (2500, 40), (16, 300), (70000, 1)])
def test_many_rows_and_heads(hip, dtype, rows, heads):
    import torch
    t = dtypes()[dtype][0]
    axes = bh.RopeAxes.of([8, 8])
    q, positions = normal((rows, heads, 32), 3, t), grid(rows, 2, 4)
    out = torch.full_like(q, 9.0)
    run(axes, positions, q, None, out, None)
    compare(out, q, positions, axes)


@pytest.mark.parametrize("positions", [[2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 10 ** 6, 0, 1, -1, 131071]])
@pytest.mark.parametrize("scale", [1.0, 0.125, -2.0, 0.0, 1e-3])
def test_far_positions_and_scales(hip, positions, scale):
    import torch
    p = torch.tensor(positions, dtype=torch.int32, device="cuda")[:, None].contiguous()
    for theta in (10000.0, 1e6, 0.5, 1.0):
        axes = bh.RopeAxes.of([32], theta=theta, scale=[scale])
        q = normal((len(positions), 2, 64), 5, torch.float32)
        out = torch.empty_like(q)
        run(axes, p, q, None, out, None)
        compare(out, q, p, axes)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_odd_alignment_and_untouched_gaps(hip, dtype, interleaved):
    import torch
    t = dtypes()[dtype][0]
    axes = bh.RopeAxes.of([5, 6], interleaved=interleaved)
    rows, heads, kv_heads, d = 41, 3, 2, 25
    # q, k and v in one projection that starts at an odd element, outputs inside wider odd buffers
    width = (heads + 2 * kv_heads) * d + 3
    fused = normal((rows * width + 1,), 6, t)[1:].view(rows, width)
    q, k = fused[:, :heads * d].unflatten(1, (heads, d)), fused[:, heads * d:(heads + kv_heads) * d].unflatten(1, (kv_heads, d))
    buffers = [torch.full((rows * (h * d + 5) + 3,), 5.0, dtype=t, device="cuda")[3:].view(rows, h * d + 5) for h in (heads, kv_heads)]
    outs = [b[:, :h * d].unflatten(1, (h, d)) for b, h in zip(buffers, (heads, kv_heads))]
    positions, before = grid(rows, 2, 7), fused.clone()
    run(axes, positions, q, k, *outs)
    compare(outs[0], q, positions, axes)
    compare(outs[1], k, positions, axes)
    assert (buffers[0][:, heads * d:] == 5.0).all() and (buffers[1][:, kv_heads * d:] == 5.0).all()
    assert torch.equal(fused, before)


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_back(hip, interleaved):
    import torch
    axes = bh.RopeAxes.of([6, 9], interleaved=interleaved)
    x, positions = normal((60, 5, 36), 8, torch.float32), grid(60, 2, 9)
    y, apart = x.clone(), torch.empty_like(x)
    run(axes, positions, x, None, apart, None)
    run(axes, positions, y, None, y, None)
    assert torch.equal(y, apart), "in place differs"
    back = torch.empty_like(x)
    run(axes, positions, apart, None, back, None, inverse=1)
    compare(back, apart, positions, axes, inverse=True)
    # turning back undoes turning up to both roundings
    assert ((back - x).abs() <= 2.0 ** -19 * x.abs().amax()).all()


def test_the_inverse_is_the_gradient(hip):
    import torch
    # the rotation is linear: sum(g * turn(x)) changes with x by turn_back(g), here against differences in 64 bits
    axes = bh.RopeAxes.of([4, 4])
    x, g, positions = normal((7, 2, 16), 1, torch.float32), normal((7, 2, 16), 2, torch.float32), grid(7, 2, 3)
    back = torch.empty_like(g)
    run(axes, positions, g, None, back, None, inverse=1)
    turned = lambda v: (plain(v, positions, axes)[0] * g.double()).sum()  # noqa: E731
    for at in ((0, 0, 0), (3, 1, 5), (6, 0, 15), (2, 1, 9)):
        step = torch.zeros_like(x, dtype=torch.float64)
        step[at] = 0.5
        difference = turned(x.double() + step) - turned(x.double() - step)
        size = g[at[0], at[1]].abs().sum().double()
        assert (difference - back[at]).abs() <= 2.0 ** -20 * size


def test_infinities_and_nans_stay_in_their_pairs(hip):
    import torch
    axes = bh.RopeAxes.of([16])
    x, positions = normal((9, 2, 32), 1, torch.float32), grid(9, 1, 2)
    want, x2 = torch.empty_like(x), x.clone()
    run(axes, positions, x, None, want, None)
    x2[4, 1, 3], x2[2, 0, 20] = math.nan, math.inf
    got = torch.empty_like(x)
    run(axes, positions, x2, None, got, None)
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[4, 1, 3] = touched[4, 1, 19] = touched[2, 0, 20] = touched[2, 0, 4] = True
    assert torch.equal(got[~touched], want[~touched]) and not torch.isfinite(got[touched]).any()


def test_offsets_beyond_32_bits(hip):
    import torch
    # rows 2^20 + 64 elements apart: the last one starts more than 2^32 bytes in
    rows, ld, axes = 2100, 2 ** 20 + 64, bh.RopeAxes.of([16])
    buffer = torch.empty(rows * ld, dtype=torch.bfloat16, device="cuda").view(rows, ld)
    x = buffer[:, 8:40].unflatten(1, (1, 32))
    x.copy_(normal((rows, 1, 32), 1, torch.bfloat16))
    positions, out = grid(rows, 1, 2), torch.empty(rows, 1, 32, dtype=torch.bfloat16, device="cuda")
    run(axes, positions, x, None, out, None)
    compare(out, x, positions, axes)
    run(axes, positions, out, None, x, None)
    compare(x, out, positions, axes)


def test_in_a_graph_and_on_two_streams(hip):
    import torch
    axes = bh.RopeAxes.of([16, 16], interleaved=True)
    sets = [(normal((300, 4, 64), s, torch.bfloat16), grid(300, 2, s)) for s in (1, 2)]
    outs = [torch.empty_like(x) for x, _ in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for (x, p), out, stream in zip(sets, outs, streams):
            run(axes, p, x, None, out, None, stream=stream)
    torch.cuda.synchronize()
    for (x, p), out in zip(sets, outs):
        compare(out, x, p, axes)
    x, p = sets[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(axes, p, x, None, outs[0], None, stream=torch.cuda.current_stream())
    axes.theta = 7.0   # the captured call keeps what it was given
    for seed in (5, 6, 7):
        x.copy_(normal(tuple(x.shape), seed, torch.bfloat16))
        p.copy_(grid(300, 2, seed))
        graph.replay()
        torch.cuda.synchronize()
        compare(outs[0], x, p, bh.RopeAxes.of([16, 16], interleaved=True))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_keys_alone(hip, dtype):
    """No query heads, as for the keys of another sequence: q and q_out may be NULL."""
    import torch
    t, code = dtypes()[dtype]
    axes = bh.RopeAxes.of([8, 12, 12], interleaved=True)
    positions = grid(77, 3, 1)
    k = normal((231, 5, 64), 2, t)
    out = torch.full_like(k, 7.0)
    bh.call("bh_rope", ctypes.byref(axes), positions.data_ptr(), 77, None, 0, None, 0, 0, k.data_ptr(), 320, out.data_ptr(), 320, 5, 231, 64,
            0, code, bh.stream_ptr(None))
    torch.cuda.synchronize()
    compare(out, k, positions, axes)
