"""Operators of a linear-attention block for image, video and text tokens, as measurable cases.

Three operators: rotary positions with several axes, linear attention with a decay for each head (a prompt, or a
token against a state), and the norms after one block and before the next with the gate and residual between them.
`own` selects between the library's kernels and the plain form: the same mathematics in elementary torch
operations, in fp32 (the angles and powers of the decay in fp64), rounded once at the end.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 64   # tokens of the plain form's chunks


# ---- cases ---------------------------------------------------------------------------------------

def _rope(batch, grid, heads, kv_heads, head_dim, pairs, joint, interleaved, dtype, span=0):
    """`grid`: the tokens' extent along each axis ("4x64x64": positions count through it), or with `span` a number
    of tokens whose positions lie anywhere below it. `pairs`: pairs of columns an axis turns ("16,24,24")."""
    return {"op": "rope", "batch": batch, "grid": grid, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "pairs": pairs, "joint": joint, "interleaved": interleaved, "dtype": dtype, "span": span}


def _linear(batch, tokens, heads, kv_heads, head_dim, value_dim, lens, with_state):
    """`lens`: each sequence's tokens ("full", or "ragged" between a quarter and all). `with_state`: it continues."""
    return {"op": "linear", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "value_dim": value_dim, "lens": lens, "with_state": with_state}


def _norms(batch, tokens, cols, post, pre, gated, modulated, dtype, stream):
    """`post`, `pre`: "none", "layer" or "rms". `stream`: the residual stream's type."""
    return {"op": "norms", "batch": batch, "tokens": tokens, "cols": cols, "post": post, "pre": pre, "gated": gated,
            "modulated": modulated, "dtype": dtype, "stream": stream}


def listed():
    return [
        # 16 sequences decode a token each at positions of long contexts: a call's latency
        dict(_rope(16, "1", 32, 8, 128, "64", True, False, "bf16", span=131072), name="rope-token"),
        # a 1024px DiT step, both guidance rows, rows and columns of its token grid
        dict(_rope(2, "64x64", 16, 16, 72, "18,18", False, True, "bf16"), name="rope-image"),
        # a clip of 21 latent frames of 32 x 48 tokens: time, height and width
        dict(_rope(1, "21x32x48", 24, 24, 128, "16,24,24", False, True, "bf16"), name="rope-video"),
        # an odd number of mixed text and image tokens, part of a head turned, one schedule over three axes, fp32
        dict(_rope(3, "385", 12, 3, 96, "8,20,12", True, False, "f32", span=4096), name="rope-ragged"),
        # 16 sequences decode a token each against their states: the states' bytes
        dict(_linear(16, 1, 32, 32, 128, 128, "full", True), name="linear-token"),
        # two padded prompts of at most 300 tokens, 64 heads of 64
        dict(_linear(2, 300, 64, 64, 64, 64, "ragged", False), name="linear-prompts"),
        # a chunk of a long prompt with grouped heads that continues from a state
        dict(_linear(2, 4096, 32, 8, 128, 128, "full", True), name="linear-long-prompt"),
        # one long document, few sequences and heads: the sequence itself has to be split
        dict(_linear(1, 65536, 16, 16, 128, 128, "full", False), name="linear-document"),
        # one token between two blocks: a call's latency
        dict(_norms(1, 1, 4096, "rms", "rms", False, False, "bf16", "bf16"), name="norms-token"),
        # two 300-token prompts, the residual stream kept in fp32
        dict(_norms(2, 300, 4096, "rms", "rms", False, False, "bf16", "f32"), name="norms-prompts"),
        # a 1024px DiT step: gated residual and modulated norm, a row of each for a batch row
        dict(_norms(2, 4096, 1152, "rms", "layer", True, True, "bf16", "bf16"), name="norms-image"),
        # sizes that divide nothing, fp32
        dict(_norms(3, 385, 2001, "layer", "layer", True, True, "f32", "f32"), name="norms-ragged"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "linear", "linear", "norms"])
    if kind == "rope":
        head_dim = rng.choice([32, 64, 72, 80, 96, 128])
        kv_heads = rng.choice([1, 2, 3, 8, 16])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        axes = rng.choice([1, 2, 2, 3, 3])
        total = head_dim // 2 if rng.random() < 0.7 else rng.randint(axes, head_dim // 2)
        cuts = sorted(rng.sample(range(1, total), axes - 1))
        pairs = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))
        batch = rng.randint(1, 4)
        if rng.random() < 0.5:
            grid, span = str(_log_int(rng, 1, 4096)), _log_int(rng, 16, 1 << 20)
        else:
            sides = [_log_int(rng, 2, 1024) if axes == 1 else _log_int(rng, 2, 64) if axes == 2 else _log_int(rng, 2, 24)
                     for _ in range(axes)]
            grid, span = "x".join(map(str, sides)), 0
        dtype = rng.choice(["bf16", "bf16", "f32"])
        rows, most = math.prod(_ints(grid, "x")), 2 * 21 * 32 * 48 * 48 * 128
        while batch * rows * (heads + kv_heads) * head_dim * (4 if dtype == "f32" else 2) > most:
            batch, heads, kv_heads = (batch - 1, heads, kv_heads) if batch > 1 else (1, heads // kv_heads, 1)
        return _rope(batch, grid, heads, kv_heads, head_dim, pairs, rng.random() < 0.5, rng.random() < 0.5, dtype, span)
    if kind == "linear":
        head_dim, value_dim = rng.choice([(32, 32), (64, 64), (72, 72), (80, 80), (96, 96), (128, 128), (64, 128), (128, 64)])
        kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        if rng.random() < 0.35:   # a token or a few against the state
            tokens = 1 if rng.random() < 0.5 else _log_int(rng, 2, 64)
            return _linear(rng.randint(1, 32), tokens, heads, kv_heads, head_dim, value_dim, rng.choice(["full", "ragged"]), True)
        batch, tokens = rng.randint(1, 4), _log_int(rng, 32, 32768)
        while batch * heads * tokens > 16 * 65536:
            batch, tokens = (batch - 1, tokens) if batch > 1 else (batch, tokens // 2)
        return _linear(batch, tokens, heads, kv_heads, head_dim, value_dim, rng.choice(["full", "ragged"]), rng.random() < 0.5)
    batch, tokens, cols = rng.randint(1, 4), _log_int(rng, 1, 4096), _log_int(rng, 64, 12288)
    if rng.random() < 0.5:   # widths of real layers; the rest divide nothing
        cols = (cols + 63) // 64 * 64
    while batch * tokens * cols > 8192 * 4096:
        tokens = max(1, tokens // 2)
    dtype, stream = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
    post, pre = rng.choice([("rms", "rms"), ("layer", "layer"), ("rms", "layer"), ("none", "rms"), ("none", "layer"), ("rms", "none")])
    return _norms(batch, tokens, cols, post, pre, rng.random() < 0.5, rng.random() < 0.5, dtype, stream)


# ---- inputs --------------------------------------------------------------------------------------

EPS = 1e-6
THETA = 10000.0


def _ints(text, sep):
    return [int(t) for t in text.split(sep)]


def _tokens_of(case):
    return math.prod(_ints(case["grid"], "x"))


def _lens(case, seed):
    if case["lens"] == "full":
        return [case["tokens"]] * case["batch"]
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    lens = torch.randint(max(1, case["tokens"] // 4), case["tokens"] + 1, (case["batch"],), generator=g).tolist()
    lens[seed % case["batch"]] = case["tokens"]
    return lens


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)

    if case["op"] == "rope":
        n, axes, d = _tokens_of(case), len(_ints(case["pairs"], ",")), case["head_dim"]
        rows, dtype = case["batch"] * n, DTYPES[case["dtype"]]
        # q, k and v as one projection leaves them
        fused = normal(rows, (case["heads"] + 2 * case["kv_heads"]) * d, dtype=dtype)
        if case["span"]:
            # a position for each token of each sequence and axis
            pos = torch.randint(0, case["span"], (rows, axes), generator=g, device="cuda", dtype=torch.int32)
        else:
            # the grid's indexes, the same for every batch row, moved as a crop or a later clip has them
            sides = [torch.arange(s, device="cuda", dtype=torch.int32) for s in _ints(case["grid"], "x")]
            pos = torch.stack(torch.meshgrid(*sides, indexing="ij"), dim=-1).reshape(n, axes) + seed % 50
            pos = pos.to(torch.int32).contiguous()
        return {"fused": fused, "positions": pos}
    if case["op"] == "linear":
        b, n, h, hk, d, e = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim", "value_dim"))
        # decays from under a half to almost one over the heads, each moved a little
        slope = -torch.exp2(-8.0 * (torch.arange(hk, device="cuda") + 1) / hk)
        slope = slope * (0.9 + 0.2 * torch.rand(hk, generator=g, device="cuda"))
        return {"q": normal(b, n, h, d), "k": normal(b, n, hk, d), "v": normal(b, n, hk, e), "log_decay": slope,
                "state_in": normal(b, hk, d, e, std=3.0, dtype=torch.float32) if case["with_state"] else None,
                "lens": _lens(case, seed)}
    rows, c = case["batch"] * case["tokens"], case["cols"]
    dtype, stream = DTYPES[case["dtype"]], DTYPES[case["stream"]]
    residual = normal(rows, c, std=4.0, mean=0.1, dtype=torch.float32)
    residual[:, ::97] *= 8.0   # the few large channels of a deep stream
    x = {"x": normal(rows, c, std=0.5, mean=0.05, dtype=dtype), "residual": residual.to(stream)}
    for side in ("post", "pre"):
        x[side + "_weight"] = normal(c, std=0.2, mean=1.0, dtype=dtype) if case[side] != "none" else None
        x[side + "_bias"] = normal(c, std=0.1, dtype=dtype) if case[side] == "layer" else None
    # the rows of one modulation projection: gate, scale, shift
    mod = normal(case["batch"], 3 * c, std=0.5, dtype=dtype)
    x["gate"] = mod[:, :c] if case["gated"] else None
    x["scale"], x["shift"] = (mod[:, c:2 * c], mod[:, 2 * c:]) if case["modulated"] else (None, None)
    return x


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    # the caller's buffers and plan: outputs, the workspace, the lengths on the device
    if case["op"] == "rope":
        d, rows = case["head_dim"], s["fused"].shape[0]
        s["pair_list"] = _ints(case["pairs"], ",")
        s["q"], s["k"] = s["fused"][:, :case["heads"] * d], s["fused"][:, case["heads"] * d:(case["heads"] + case["kv_heads"]) * d]
        s["q_out"] = torch.empty((rows, case["heads"], d), dtype=s["fused"].dtype, device="cuda")
        s["k_out"] = torch.empty((rows, case["kv_heads"], d), dtype=s["fused"].dtype, device="cuda")
    elif case["op"] == "linear":
        s["lens_dev"] = torch.tensor(s["lens"], dtype=torch.int32, device="cuda")
        s["out"] = torch.empty((case["batch"], case["tokens"], case["heads"], case["value_dim"]), dtype=torch.bfloat16, device="cuda")
        s["state_out"] = torch.empty((case["batch"], case["kv_heads"], case["head_dim"], case["value_dim"]), device="cuda")
    else:
        s["residual_out"], s["out"] = torch.empty_like(s["residual"]), torch.empty_like(s["x"])
    if own:
        import burnisher_amd as bh
        bh.call("bh_init", 0)
        if case["op"] == "rope":
            s["axes"] = bh.RopeAxes.of(s["pair_list"], theta=THETA, joint=case["joint"], interleaved=case["interleaved"])
        elif case["op"] == "linear":
            need = bh.lib().bh_attention_linear_workspace_bytes(case["batch"], case["heads"], case["kv_heads"], case["tokens"],
                                                                case["head_dim"], case["value_dim"])
            s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        else:
            kinds = {"none": bh.NORM_NONE, "layer": bh.NORM_LAYER, "rms": bh.NORM_RMS}
            s["plan"] = bh.ResidualNorms(
                post_norm=kinds[case["post"]], post_weight=bh.ptr(s["post_weight"]), post_bias=bh.ptr(s["post_bias"]),
                post_eps=EPS, gate=bh.ptr(s["gate"]), branch_scale=1.0, residual_scale=1.0, pre_norm=kinds[case["pre"]],
                pre_weight=bh.ptr(s["pre_weight"]), pre_bias=bh.ptr(s["pre_bias"]), pre_eps=EPS, scale=bh.ptr(s["scale"]),
                shift=bh.ptr(s["shift"]), mod_rows=case["tokens"], ld_mod=3 * case["cols"], weight_offset=0.0)
    return s


# ---- one pass: the plain forms -------------------------------------------------------------------

def _turn_plain(x, cos, sin, total, interleaved):
    """x [rows, heads, head_dim]; cos, sin [rows, 1, total]."""
    v = x.float()
    turned, rest = v[..., :2 * total], v[..., 2 * total:]
    u, w = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :total], turned[..., total:])
    a, b = u * cos - w * sin, u * sin + w * cos
    turned = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([turned, rest], dim=-1).to(x.dtype)


def _rope_plain(s):
    pairs, d = s["pair_list"], s["head_dim"]
    total = sum(pairs)
    axis = torch.repeat_interleave(torch.arange(len(pairs), device="cuda"), torch.tensor(pairs, device="cuda"), output_size=total)
    i = torch.arange(total, device="cuda", dtype=torch.float64)
    if s["joint"]:
        power = i / total
    else:
        size = torch.tensor(pairs, device="cuda", dtype=torch.float64)
        power = (i - (size.cumsum(0) - size)[axis]) / size[axis]
    angle = s["positions"].double()[:, axis] * torch.exp(-math.log(THETA) * power)
    rows = s["fused"].shape[0]
    cos, sin = (t.float()[:, None, :].repeat(rows // angle.shape[0], 1, 1) for t in (torch.cos(angle), torch.sin(angle)))
    return {"q": _turn_plain(s["q"].unflatten(1, (s["heads"], d)), cos, sin, total, s["interleaved"]),
            "k": _turn_plain(s["k"].unflatten(1, (s["kv_heads"], d)), cos, sin, total, s["interleaved"])}


def _linear_plain(s):
    b, n, h, hk, d, e = (s[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim", "value_dim"))
    size = min(CHUNK, n)
    g, nc, dev = h // hk, -(-n // size), "cuda"
    pad = nc * size - n
    log_decay = s["log_decay"].double()
    valid = (torch.arange(n, device=dev)[None, :] < s["lens_dev"][:, None])
    keep = valid[:, :, None, None].float()

    def chunked(x):   # [b, n, heads, width] -> [b, hk, nc, (group x) size, width]
        x = torch.nn.functional.pad(x.float() * keep, (0, 0, 0, 0, 0, pad))
        x = x.view(b, nc, size, hk, -1, x.shape[-1]).permute(0, 3, 1, 4, 2, 5)
        return x.reshape(b, hk, nc, -1, x.shape[-1])

    def powers(exponent):   # [hk, ...]: decay ** exponent, 0 where the exponent is negative
        p = torch.exp(exponent.double() * log_decay.view(-1, *([1] * exponent.dim())))
        return torch.where(exponent >= 0, p, torch.zeros_like(p)).float()

    q, k, v = chunked(s["q"]), chunked(s["k"]), chunked(s["v"])
    i = torch.arange(size, device=dev)
    within = powers(i[:, None] - i[None, :]).repeat(1, g, 1)[:, None]                # [hk, 1, g * size, size]
    out = ((q @ k.transpose(-1, -2).contiguous()) * within) @ v
    # what each chunk adds to the state, and the states before each chunk as sums of those and the first
    added = (k * powers(size - 1 - i)[:, None, :, None]).transpose(-1, -2).contiguous() @ v
    start = s["state_in"] if s["state_in"] is not None else torch.zeros((b, hk, d, e), device=dev)
    c = torch.arange(nc, device=dev)
    carry = torch.cat([powers(c[:, None] * size), powers((c[:, None] - 1 - c[None, :]) * size)], dim=2)
    before = carry @ torch.cat([start[:, :, None], added], dim=2).flatten(-2)
    out = out + (q * powers(i + 1).repeat(1, g)[:, None, :, None]) @ before.unflatten(-1, (d, e))
    out = out.view(b, hk, nc, g, size, e).permute(0, 2, 4, 1, 3, 5).reshape(b, nc * size, h, e)[:, :n] / math.sqrt(d)
    # the state after each sequence's own last token
    lens = s["lens_dev"].long()
    last = powers(lens[:, None] - 1 - torch.arange(n, device=dev)[None, :]).permute(1, 0, 2)[..., None]   # [b, hk, n, 1]
    kk = (s["k"].float().permute(0, 2, 1, 3) * last).transpose(-1, -2).contiguous()
    vv = (s["v"].float() * keep).permute(0, 2, 1, 3).contiguous()
    state = kk @ vv + powers(lens).t()[:, :, None, None] * start
    return {"out": (out * keep).to(torch.bfloat16), "state": state}


def _norm_plain(v, kind, weight, bias):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS) * weight.float()
    return v if bias is None else v + bias.float()


def _norms_plain(s):
    def rows(m):   # a batch row's modulation for each of its tokens
        return m.float().repeat_interleave(s["tokens"], dim=0)

    branch = _norm_plain(s["x"].float(), s["post"], s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        branch = branch * rows(s["gate"])
    stream = s["residual"].float() + branch
    out = _norm_plain(stream, s["pre"], s["pre_weight"], s["pre_bias"])
    if s["scale"] is not None:
        out = out * (1.0 + rows(s["scale"])) + rows(s["shift"])
    return {"residual": stream.to(s["residual"].dtype), "out": out.to(s["x"].dtype)}


# ---- one pass ------------------------------------------------------------------------------------

def run(s):
    if s["op"] == "rope":
        if not own:
            return _rope_plain(s)
        import burnisher_amd as bh
        d, hq, hk = s["head_dim"], s["heads"], s["kv_heads"]
        bh.call("bh_rope", ctypes.byref(s["axes"]), bh.ptr(s["positions"]), s["positions"].shape[0], bh.ptr(s["q"]),
                s["fused"].stride(0), bh.ptr(s["q_out"]), hq * d, hq, bh.ptr(s["k"]), s["fused"].stride(0), bh.ptr(s["k_out"]),
                hk * d, hk, s["fused"].shape[0], d, 0, bh.BF16 if s["dtype"] == "bf16" else bh.F32, bh.stream_ptr())
        return {"q": s["q_out"], "k": s["k_out"]}
    if s["op"] == "linear":
        if not own:
            return _linear_plain(s)
        import burnisher_amd as bh
        h, hk, d, e = s["heads"], s["kv_heads"], s["head_dim"], s["value_dim"]
        bh.call("bh_attention_linear", bh.ptr(s["q"]), h * d, bh.ptr(s["k"]), hk * d, bh.ptr(s["v"]), hk * e, bh.ptr(s["out"]),
                h * e, s["batch"], h, hk, s["tokens"], d, e, 0.0, bh.ptr(s["log_decay"]), bh.ptr(s["lens_dev"]),
                bh.ptr(s["state_in"]), bh.ptr(s["state_out"]), bh.BF16, bh.ptr(s["workspace"]), s["workspace"].numel(),
                bh.stream_ptr())
        return {"out": s["out"], "state": s["state_out"]}
    if not own:
        return _norms_plain(s)
    import burnisher_amd as bh
    c = s["cols"]
    kind = {"bf16": bh.BF16, "f32": bh.F32}
    bh.call("bh_residual_norms_run", bh.ptr(s["x"]), c, bh.ptr(s["residual"]), c, bh.ptr(s["residual_out"]), c, bh.ptr(s["out"]),
            c, s["x"].shape[0], c, ctypes.byref(s["plan"]), kind[s["stream"]], kind[s["dtype"]], bh.stream_ptr())
    return {"residual": s["residual_out"], "out": s["out"]}


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    size = {"bf16": 2, "f32": 4}
    if case["op"] == "rope":
        n, total, axes = _tokens_of(case), sum(_ints(case["pairs"], ",")), len(_ints(case["pairs"], ","))
        rows, heads = case["batch"] * n, case["heads"] + case["kv_heads"]
        positions = 4 * axes * (rows if case["span"] else n)
        return {"bytes": 2 * rows * heads * case["head_dim"] * size[case["dtype"]] + positions, "flops": 6 * rows * heads * total}
    if case["op"] == "linear":
        b, n, h, hk, d, e = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim", "value_dim"))
        # with every sequence as long as the case allows on average; an output row is written whether it holds a token or not
        tokens = b * n if case["lens"] == "full" else n + (b - 1) * max(1, n * 5 // 8)
        states = 4 * b * hk * d * e * (2 if case["with_state"] else 1)
        return {"bytes": 2 * (tokens * (h * d + hk * (d + e)) + b * n * h * e) + states, "flops": 2 * d * e * (h + hk) * tokens}
    rows, c = case["batch"] * case["tokens"], case["cols"]
    small = (case["post"] != "none") + (case["pre"] != "none") + case["batch"] * (case["gated"] + 2 * case["modulated"])
    return {"bytes": 2 * rows * c * (size[case["dtype"]] + size[case["stream"]]) + small * c * size[case["dtype"]], "flops": 16 * rows * c}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _rope_exact(case, x):
    pairs, d = _ints(case["pairs"], ","), case["head_dim"]
    total, rows = sum(pairs), x["fused"].shape[0]
    where = torch.arange(rows, device="cuda") % x["positions"].shape[0]

    def turned(v):
        out, at = v.double(), 0
        for a, count in enumerate(pairs):
            for j in range(count):
                f = THETA ** -((at / total) if case["joint"] else (j / count))
                t = x["positions"][where, a].double() * f
                z = torch.polar(torch.ones_like(t), t)[:, None]
                first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, total + at)
                z = z * torch.complex(v[..., first].double(), v[..., second].double())
                out[..., first], out[..., second] = z.real, z.imag
                at += 1
        return out

    q, k, _ = x["fused"].split([case["heads"] * d, case["kv_heads"] * d, case["kv_heads"] * d], dim=1)
    return {"q": turned(q.unflatten(1, (-1, d))), "k": turned(k.unflatten(1, (-1, d)))}


def _linear_exact(case, x):
    # every pair of tokens: weight decay^(i - j) for j <= i, and decay^(i + 1) for the state before the first
    b, n, h, hk, d, e = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "head_dim", "value_dim"))
    out = torch.zeros((b, n, h, e), dtype=torch.float64, device="cuda")
    state = torch.zeros((b, hk, d, e), dtype=torch.float64, device="cuda")
    rate = x["log_decay"].double().tolist()
    for bb in range(b):
        m = x["lens"][bb]
        at = torch.arange(m, device="cuda", dtype=torch.float64)
        for kh in range(hk):
            k, v = x["k"][bb, :m, kh].double(), x["v"][bb, :m, kh].double()
            first = x["state_in"][bb, kh].double() if case["with_state"] else None
            state[bb, kh] = (k * torch.exp(rate[kh] * (m - 1 - at))[:, None]).t().contiguous() @ v
            if first is not None:
                state[bb, kh] += math.exp(rate[kh] * m) * first
            # tokens whose weight is below e^-80 of a near one's are left out of the pairs
            reach = min(m, int(80.0 / -rate[kh]) + 2)
            for g in range(h // hk):
                q = x["q"][bb, :m, kh * (h // hk) + g].double() / math.sqrt(d)
                for i0 in range(0, m, 1024):
                    i1 = min(i0 + 1024, m)
                    j0 = max(0, i0 - reach)
                    gap = at[i0:i1, None] - at[None, j0:i1]
                    weight = torch.exp(rate[kh] * gap.clamp(min=0)) * (gap >= 0)
                    rows = (torch.mm(q[i0:i1], k[j0:i1].t().contiguous()) * weight) @ v[j0:i1]
                    if first is not None:
                        rows = rows + torch.exp(rate[kh] * (at[i0:i1] + 1))[:, None] * (q[i0:i1] @ first)
                    out[bb, i0:i1, kh * (h // hk) + g] = rows
    return {"out": out, "state": state}


def _norms_exact(case, x):
    def norm(v, side):
        if case[side] == "none":
            return v
        if case[side] == "layer":
            v = (v - v.mean(1, keepdim=True)) / torch.sqrt(v.var(1, unbiased=False, keepdim=True) + EPS)
            return v * x[side + "_weight"].double() + x[side + "_bias"].double()
        return v / torch.sqrt(v.square().mean(1, keepdim=True) + EPS) * x[side + "_weight"].double()

    of = torch.arange(case["batch"] * case["tokens"], device="cuda") // case["tokens"]
    branch = norm(x["x"].double(), "post")
    if case["gated"]:
        branch = x["gate"].double()[of] * branch
    stream = x["residual"].double() + branch
    out = norm(stream, "pre")
    if case["modulated"]:
        out = out + out * x["scale"].double()[of] + x["shift"].double()[of]
    return {"residual": stream, "out": out}


def exact(case, seed):
    x = _inputs(case, seed)
    return {"rope": _rope_exact, "linear": _linear_exact, "norms": _norms_exact}[case["op"]](case, x)
