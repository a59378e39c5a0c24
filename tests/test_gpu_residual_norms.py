"""bh_residual_norms_run on the GPU against its formula in 64 bits on the same inputs.

The tolerance counts roundings in units of 2^-24 (u). A norm's mean and mean square are sums of at most 512 + 10
terms a lane and level, so each is off by less than 530 u of the mean magnitude, and behind the square root half
that; a normalised value is then off by (265 + 6) u of itself and 530 u times mean(|x|) / deviation. The products
and sums behind it add 8 u of the magnitudes they sum. The second norm divides what the first left by its own
deviation and adds the same. Outputs are rounded once.
"""
import ctypes
import math

import pytest

import burnisher_amd as bh

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def torch_type(name):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


CODE = {"bf16": bh.BF16, "f32": bh.F32}
KIND = {"none": bh.NORM_NONE, "layer": bh.NORM_LAYER, "rms": bh.NORM_RMS}


def make(rows, cols, dtype, stream, post, pre, mod_rows=1, parts="wbgmr", seed=0, mean=0.1, std=1.0, eps=1e-6):
    """Operands; `parts`: w weights, b biases, g gate, m scale and shift."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s, m=0.0, d=1.0, t=torch_type(dtype): (torch.randn(s, generator=g, device="cuda") * d + m).to(t)  # noqa: E731
    o = {"x": normal(rows, cols, m=mean, d=std), "residual": normal(rows, cols, m=0.2, d=3.0, t=torch_type(stream)),
         "post": post, "pre": pre, "mod_rows": mod_rows, "eps": eps, "offset": 0.0, "branch": 0.7, "keep": 1.3}
    for side, kind in (("post", post), ("pre", pre)):
        o[side + "_w"] = normal(cols, m=1.0, d=0.2) if "w" in parts and kind != "none" else None
        o[side + "_b"] = normal(cols, d=0.1) if "b" in parts and kind != "none" else None
    mod = normal(-(-rows // mod_rows), 3 * cols, d=0.5)
    o["ld_mod"] = 3 * cols
    o["gate"] = mod[:, :cols] if "g" in parts else None
    o["scale"], o["shift"] = (mod[:, cols:2 * cols], mod[:, 2 * cols:]) if "m" in parts else (None, None)
    return o


def plan(o):
    return bh.ResidualNorms(
        post_norm=KIND[o["post"]], post_weight=bh.ptr(o["post_w"]), post_bias=bh.ptr(o["post_b"]), post_eps=o["eps"],
        gate=bh.ptr(o["gate"]), branch_scale=o["branch"], residual_scale=o["keep"], pre_norm=KIND[o["pre"]],
        pre_weight=bh.ptr(o["pre_w"]), pre_bias=bh.ptr(o["pre_b"]), pre_eps=o["eps"], scale=bh.ptr(o["scale"]),
        shift=bh.ptr(o["shift"]), mod_rows=o["mod_rows"], ld_mod=o["ld_mod"], weight_offset=o["offset"])


def run(o, residual_out, out, stream=None):
    x, r = o["x"], o["residual"]
    ld = lambda t: 0 if t is None else max(t.stride(0), t.shape[1])  # noqa: E731
    code = lambda t: CODE["bf16" if t.element_size() == 2 else "f32"]  # noqa: E731
    bh.call("bh_residual_norms_run", x.data_ptr(), ld(x), r.data_ptr(), ld(r), bh.ptr(residual_out), ld(residual_out), bh.ptr(out),
            ld(out), x.shape[0], x.shape[1], ctypes.byref(plan(o)), code(r), code(x), bh.stream_ptr(stream))


def plain(o):
    """(residual, its tolerance, out, its tolerance) in 64 bits."""
    import torch
    x, r, rows = o["x"].double(), o["residual"].double(), o["x"].shape[0]
    of = torch.arange(rows, device="cuda") // o["mod_rows"]
    f32 = lambda v: torch.tensor(v, dtype=torch.float32).item()  # noqa: E731
    eps = f32(o["eps"])

    def norm(v, err, kind, w, b):
        if kind == "none":
            return v, err
        c = v.shape[1]
        level = v.abs().mean(1, keepdim=True)
        d = v - v.mean(1, keepdim=True) if kind == "layer" else v
        inv = 1 / torch.sqrt(d.square().mean(1, keepdim=True) + eps)
        n = d * inv
        # what the input's own error does: through the value, and through the mean and deviation of its row
        worst = err + err.amax(1, keepdim=True) * (1 + n.abs())
        e = n.abs() * 271 * U + inv * (level * 530 * U * (1 + n.abs()) if kind == "layer" else 0) + worst * inv
        if w is not None:
            ww = w.double() + o["offset"]
            n, e = n * ww, e * ww.abs() + (n * ww).abs() * 2 * U + n.abs() * U
        if b is not None:
            n, e = n + b.double(), e + (n.abs() + b.double().abs()) * U
        return n, e

    n, e = norm(x, torch.zeros_like(x), o["post"], o["post_w"], o["post_b"])
    if o["gate"] is not None:
        n, e = n * o["gate"].double()[of], (e + n.abs() * U) * o["gate"].double()[of].abs()
    branch, keep = f32(o["branch"]), f32(o["keep"])
    res = keep * r + branch * n
    e = abs(branch) * e + 2 * U * ((keep * r).abs() + (branch * n).abs())
    out, eo = norm(res, e, o["pre"], o["pre_w"], o["pre_b"])
    if o["scale"] is not None:
        s = 1 + o["scale"].double()[of]
        out, eo = out * s, (eo + 2 * out.abs() * U) * s.abs() + out.abs() * (1 + o["scale"].double()[of].abs()) * U
    if o["shift"] is not None:
        t = o["shift"].double()[of]
        out, eo = out + t, eo + (out.abs() + t.abs()) * U
    half = lambda t: torch.finfo(t.dtype).eps / 2  # noqa: E731
    return res, e + (res.abs() + e) * half(o["residual"]), out, eo + (out.abs() + eo) * half(o["x"])


def compare(o, residual_out, out):
    res, res_tol, want, tol = plain(o)
    for name, got, w, t in (("residual", residual_out, res, res_tol), ("out", out, want, tol)):
        if got is None:
            continue
        bad = ~((got.double() - w).abs() <= t + 1e-37)
        if bad.any():
            at = tuple(bad.nonzero()[0].tolist())
            raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {got[at]} for {w[at]} +- {t[at]}")


def check(*args, **how):
    import torch
    o = make(*args, **how)
    residual_out, out = torch.full_like(o["residual"], 9.0), torch.full_like(o["x"], 9.0)
    run(o, residual_out, out)
    compare(o, residual_out, out)
    return o


TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")]


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 63, 511, 512, 513, 1152, 2047, 2048, 2049, 4096, 4100, 8191, 8192, 8193, 12288, 20001, 32768])
def test_widths(hip, cols, dtype, stream):
    check(5, cols, dtype, stream, "layer", "rms", mod_rows=2, seed=cols)
    check(5, cols, dtype, stream, "rms", "layer", mod_rows=5, seed=cols)


@pytest.mark.parametrize("post", list(KIND))
@pytest.mark.parametrize("pre", list(KIND))
@pytest.mark.parametrize("parts", ["wbgm", "", "w", "b", "g", "m", "wg", "wbm"])
@pytest.mark.parametrize("cols", [333, 2500])
def test_norms_and_parts(hip, post, pre, parts, cols):
    for dtype, stream in TYPES:
        check(7, cols, dtype, stream, post, pre, mod_rows=3, parts=parts, seed=1)


@pytest.mark.parametrize("rows,cols,mod_rows", [(1, 4096, 1), (4097, 64, 4097), (1155, 2001, 385), (3, 32768, 1), (20000, 8, 7)])
def test_rows(hip, rows, cols, mod_rows):
    for dtype, stream in TYPES:
        check(rows, cols, dtype, stream, "rms", "layer", mod_rows=mod_rows, seed=rows)


def test_stored_differences_to_one(hip):
    import torch
    o = make(9, 700, "bf16", "f32", "rms", "rms", parts="w")
    for side in ("post_w", "pre_w"):
        o[side] = o[side] - 1
    o["offset"] = 1.0
    res, out = torch.empty_like(o["residual"]), torch.empty_like(o["x"])
    run(o, res, out)
    compare(o, res, out)


@pytest.mark.parametrize("cols", [640, 5000, 9000])
def test_one_output_and_in_place(hip, cols):
    import torch
    for dtype, stream in TYPES:
        o = make(11, cols, dtype, stream, "rms", "layer", mod_rows=4)
        res, out = torch.full_like(o["residual"], 9.0), torch.full_like(o["x"], 9.0)
        run(o, res, out)
        only = torch.full_like(o["x"], 9.0)
        run(o, None, only)
        assert torch.equal(only, out)
        only = torch.full_like(o["residual"], 9.0)
        run(o, only, None)
        assert torch.equal(only, res)
        run(o, o["residual"], o["x"])
        assert torch.equal(o["residual"], res) and torch.equal(o["x"], out)


def test_large_means_keep_their_digits(hip):
    # a mean 1000 times the deviation, fp32
    check(9, 3000, "f32", "f32", "layer", "layer", mean=1000.0, parts="wb")


def test_zero_rows(hip):
    import torch
    o = make(4, 900, "bf16", "bf16", "rms", "layer", mod_rows=4)
    o["x"].zero_()
    o["residual"][2:] = 0
    res, out = torch.empty_like(o["residual"]), torch.empty_like(o["x"])
    run(o, res, out)
    compare(o, res, out)


@pytest.mark.parametrize("poison", [math.nan, math.inf])
@pytest.mark.parametrize("cols", [333, 2500])
def test_a_bad_row_stays_alone(hip, cols, poison):
    import torch
    o = make(9, cols, "bf16", "f32", "layer", "rms", mod_rows=9)
    want, w_out = torch.empty_like(o["residual"]), torch.empty_like(o["x"])
    run(o, want, w_out)
    o["x"][4, 100] = poison
    res, out = torch.empty_like(o["residual"]), torch.empty_like(o["x"])
    run(o, res, out)
    keep = torch.arange(9, device="cuda") != 4
    assert torch.equal(res[keep], want[keep]) and torch.equal(out[keep], w_out[keep])
    assert torch.isnan(out[4]).all()


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("cols", [100, 1001, 2600])
def test_strides_odd_alignment_and_untouched_gaps(hip, dtype, stream, cols):
    import torch
    o = make(21, cols, dtype, stream, "layer", "layer", mod_rows=6)
    odd = lambda t, pad: torch.full((t.shape[0] * (cols + pad) + 1,), 5.0, dtype=t.dtype, device="cuda")[1:].view(t.shape[0], cols + pad)  # noqa: E731
    bx, br, bo, bs = odd(o["x"], 3), odd(o["residual"], 5), odd(o["x"], 7), odd(o["residual"], 1)
    bx[:, :cols], br[:, :cols] = o["x"], o["residual"]
    o["x"], o["residual"] = bx[:, :cols], br[:, :cols]
    run(o, bs[:, :cols], bo[:, :cols])
    compare(o, bs[:, :cols], bo[:, :cols])
    assert (bo[:, cols:] == 5.0).all() and (bs[:, cols:] == 5.0).all() and (bx[:, cols:] == 5.0).all()


def test_offsets_beyond_32_bits(hip):
    import torch
    rows, cols, ld = 2100, 40, 2 ** 20 + 8
    o = make(rows, cols, "bf16", "bf16", "rms", "rms", mod_rows=rows)
    wide = torch.empty(rows * ld, dtype=torch.bfloat16, device="cuda").view(rows, ld)
    wide[:, :cols], wide[:, 64:64 + cols] = o["x"], o["residual"]
    o["x"], o["residual"] = wide[:, :cols], wide[:, 64:64 + cols]
    run(o, wide[:, 128:128 + cols], wide[:, 192:192 + cols])
    compare(o, wide[:, 128:128 + cols], wide[:, 192:192 + cols])


def test_in_a_graph_and_on_two_streams(hip):
    import torch
    sets = [make(300, 1500, "bf16", "f32", "rms", "layer", mod_rows=100, seed=s) for s in (1, 2)]
    outs = [(torch.empty_like(o["residual"]), torch.empty_like(o["x"])) for o in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for o, to, stream in zip(sets, outs, streams):
            run(o, *to, stream=stream)
    torch.cuda.synchronize()
    for o, to in zip(sets, outs):
        compare(o, *to)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(sets[0], *outs[0], stream=torch.cuda.current_stream())
    for seed in (5, 6, 7):
        new = make(300, 1500, "bf16", "f32", "rms", "layer", mod_rows=100, seed=seed)
        for name in ("x", "residual", "post_w", "gate", "shift"):
            sets[0][name].copy_(new[name])
        graph.replay()
        torch.cuda.synchronize()
        compare(sets[0], *outs[0])
