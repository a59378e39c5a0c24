"""Operators of a text model held in 8 bits and of long-range attention, as measurable cases.

Three operators: quantising a matrix to e4m3 with one scale per 128 values (a token's activations) or
per 128 x 128 block (weights), the matrix product of two such matrices, and attention through a sliding
window with first tokens that stay visible. `own` selects between the library's kernels and the plain
form: the same mathematics in elementary torch operations, in fp32, rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128            # values a scale covers, along K (and along N for weights)
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -96   # a block's largest magnitude counts as at least this
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------

def _quant(rows, cols, block_rows, dtype):
    return {"op": "quantize", "rows": rows, "cols": cols, "block_rows": block_rows, "dtype": dtype}


def _gemm(m, n, k, act, bias, dtype):
    return {"op": "gemm", "m": m, "n": n, "k": k, "act": act, "bias": bias, "dtype": dtype}


def _attn(batch, heads, kv_heads, q_len, kv_len, head_dim, left, right, sinks, lens, at_end):
    """`lens`: each sequence's valid keys ("full", or "ragged" between a quarter and all of kv_len).
    `at_end`: the queries are the last q_len tokens of their sequence; otherwise the first."""
    return {"op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "q_len": q_len,
            "kv_len": kv_len, "head_dim": head_dim, "left": left, "right": right, "sinks": sinks,
            "lens": lens, "at_end": at_end}


def listed():
    return [
        # one token's activations before a projection of width 4096: a call's latency
        dict(_quant(1, 4096, 1, "bf16"), name="quantize-token"),
        # the T5 MLP's activations of two 300-token prompts
        dict(_quant(600, 10240, 1, "bf16"), name="quantize-prompts"),
        # an MLP weight of the T5 XXL encoder, once per load, from an fp32 checkpoint
        dict(_quant(10240, 4096, 128, "f32"), name="quantize-weights"),
        # one token through a 4096 x 4096 projection: the weights' bytes
        dict(_gemm(1, 4096, 4096, 0, False, "bf16"), name="gemm-token"),
        # the packed q/k/v projection of 16 sequences, a token each
        dict(_gemm(16, 12288, 4096, 0, False, "bf16"), name="gemm-tokens-16"),
        # the T5 MLP's output projection of two 300-token prompts: few tiles, a long K
        dict(_gemm(600, 4096, 10240, 0, False, "bf16"), name="gemm-prompts"),
        # sizes that divide nothing, fp32 out
        dict(_gemm(1155, 4100, 2001, 2, True, "f32"), name="gemm-ragged"),
        # the DiT's first MLP projection at 1024px, both guidance rows, with its GELU
        dict(_gemm(8192, 4608, 1152, 1, True, "bf16"), name="gemm-image"),
        # 16 sequences decode a token each from a cache of up to 8192 keys, window 4096, 4 sinks
        dict(_attn(16, 32, 8, 1, 8192, 128, 4095, 0, 4, "ragged", True), name="window-token"),
        # two padded prompts of at most 300 tokens, T5 XXL's heads, 128 keys to either side
        dict(_attn(2, 64, 64, 300, 300, 64, 128, 128, 0, "ragged", False), name="window-prompts"),
        # a long causal prompt with grouped heads, window 1024, 4 sinks
        dict(_attn(2, 32, 8, 4096, 4096, 128, 1023, 0, 4, "full", False), name="window-long-prompt"),
        # the image tokens of a 2048px step, 8 rows of 128 tokens to either side
        dict(_attn(2, 16, 16, 16384, 16384, 72, 1024, 1024, 0, "full", False), name="window-image"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "gemm", "gemm", "attention", "attention"])
    if kind == "quantize":
        if rng.random() < 0.5:
            rows, cols = _log_int(rng, 1, 8192), _log_int(rng, 16, 10240)
            return _quant(rows, cols, 1, rng.choice(["bf16", "f32"]))
        return _quant(_log_int(rng, 128, 12288), _log_int(rng, 128, 4608), 128, rng.choice(["bf16", "f32"]))
    if kind == "gemm":
        m = _log_int(rng, 1, 64) if rng.random() < 0.5 else _log_int(rng, 64, 8192)
        n, k = _log_int(rng, 64, 12288), _log_int(rng, 64, 10240)
        if rng.random() < 0.5:   # widths of real layers; the rest divide nothing
            n, k = (n + 127) // 128 * 128, (k + 127) // 128 * 128
        while m * n * k > 8192 * 4608 * 1152:
            m = max(1, m // 2)
        return _gemm(m, n, k, rng.choice([0, 0, 1, 2]), rng.random() < 0.5, rng.choice(["bf16", "bf16", "f32"]))
    head_dim = rng.choice([32, 64, 72, 80, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
    left = rng.choice([0, 63, _log_int(rng, 8, 4096), _log_int(rng, 8, 4096)])
    right = rng.choice([0, 0, left])
    sinks = rng.choice([0, 0, 4, rng.randint(1, 100)])
    if rng.random() < 0.5:   # single tokens or a short chunk against a cache
        batch, kv_len = rng.randint(1, 16), _log_int(rng, 16, 8192)
        q_len = 1 if rng.random() < 0.5 else min(kv_len // 4, _log_int(rng, 2, 300))
        return _attn(batch, heads, kv_heads, max(1, q_len), kv_len, head_dim, left, right, sinks, "ragged", True)
    batch, tokens = rng.randint(1, 4), _log_int(rng, 16, 8192)
    while batch * heads * tokens > 2 * 32 * 4096:
        batch, heads, kv_heads = (batch - 1, heads, kv_heads) if batch > 1 else (batch, heads // kv_heads, 1) \
            if kv_heads > 1 else (batch, 1, 1)
        if batch * heads == 1:
            break
    return _attn(batch, heads, kv_heads, tokens, tokens, head_dim, left, right, sinks,
                 rng.choice(["full", "ragged"]), False)


# ---- inputs --------------------------------------------------------------------------------------

def _pad16(k):
    return (k + 15) // 16 * 16


def _quantize_plain(x, block_rows):
    """(codes [rows, round_up(cols, 16)] in e4m3 with a zero tail, fp32 scales): [blocks of columns, rows]
    for block_rows 1, [blocks of rows, blocks of columns] for 128."""
    rows, cols = x.shape
    nc, nr = -(-cols // BLOCK), -(-rows // block_rows)
    padded = torch.zeros((nr * block_rows, nc * BLOCK), dtype=torch.float32, device=x.device)
    padded[:rows, :cols] = x
    blocks = padded.view(nr, block_rows, nc, BLOCK)
    amax = blocks.abs().amax(dim=(1, 3)).clamp(min=AMAX_FLOOR)
    top = torch.full_like(amax, E4M3_MAX)   # a tensor: torch replaces a division by a number by a product
    codes = (blocks * (top / amax)[:, None, :, None]).view(nr * block_rows, nc * BLOCK)
    codes = codes[:rows, :_pad16(cols)].to(torch.float8_e4m3fn)
    scales = amax / top
    return codes, (scales.t().contiguous() if block_rows == 1 else scales)


def _lens(case, seed):
    """Each sequence's valid keys, and the position of its first query."""
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    if case["lens"] == "full":
        lens = [case["kv_len"]] * case["batch"]
    else:
        low = max(case["q_len"] if case["at_end"] else 1, case["kv_len"] // 4)
        lens = torch.randint(low, case["kv_len"] + 1, (case["batch"],), generator=g).tolist()
        lens[seed % case["batch"]] = case["kv_len"]
    starts = [n - case["q_len"] for n in lens] if case["at_end"] else [0] * case["batch"]
    return lens, starts


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    if case["op"] == "quantize":
        # activations with a few channels much larger than the rest, as text models have; weights N(0, 0.02)
        x = normal(case["rows"], case["cols"], std=0.02 if case["block_rows"] > 1 else 1.0, dtype=torch.float32)
        if case["block_rows"] == 1:
            x[:, ::97] *= 20.0
        return {"x": x.to(DTYPES[case["dtype"]])}
    if case["op"] == "gemm":
        a, a_scales = _quantize_plain(normal(case["m"], case["k"], dtype=torch.float32), 1)
        b, b_scales = _quantize_plain(normal(case["n"], case["k"], std=0.02, dtype=torch.float32), BLOCK)
        bias = normal(case["n"], dtype=DTYPES[case["dtype"]]) if case["bias"] else None
        return {"a": a, "a_scales": a_scales, "b": b, "b_scales": b_scales, "bias": bias}
    d = case["head_dim"]
    lens, starts = _lens(case, seed)
    return {"q": normal(case["batch"], case["q_len"], case["heads"], d),
            "k": normal(case["batch"], case["kv_len"], case["kv_heads"], d),
            "v": normal(case["batch"], case["kv_len"], case["kv_heads"], d),
            "lens": lens, "starts": starts}


def prepare(case, seed):
    state = dict(case, **_inputs(case, seed))
    # the caller's buffers: outputs, and where the library asks for it the workspace
    if case["op"] == "quantize":
        rows, cols, br = case["rows"], case["cols"], case["block_rows"]
        nc, nr = -(-cols // BLOCK), -(-rows // br)
        state["out"] = torch.empty((rows, _pad16(cols)), dtype=torch.float8_e4m3fn, device="cuda")
        state["scales"] = torch.empty((nc, rows) if br == 1 else (nr, nc), device="cuda")
    elif case["op"] == "gemm":
        state["out"] = torch.empty((case["m"], case["n"]), dtype=DTYPES[case["dtype"]], device="cuda")
    else:
        state["out"] = torch.empty_like(state["q"])
        state["lens_dev"] = torch.tensor(state["lens"], dtype=torch.int32, device="cuda")
        state["starts_dev"] = torch.tensor(state["starts"], dtype=torch.int32, device="cuda")
    if own:
        import burnisher_amd as bh
        bh.call("bh_init", 0)
        need = 0
        if case["op"] == "gemm":
            need = bh.lib().bh_gemm_fp8_workspace_bytes(case["m"], case["n"], case["k"])
        elif case["op"] == "attention":
            need = bh.lib().bh_attention_window_workspace_bytes(
                case["batch"], case["heads"], case["kv_heads"], case["q_len"], case["kv_len"], case["head_dim"],
                case["left"], case["right"], case["sinks"])
        state["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return state


# ---- one pass ------------------------------------------------------------------------------------

def _act_plain(v, act):
    if act == 1:
        return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    if act == 2:
        return v / (1.0 + torch.exp(-v))
    return v


def _gemm_plain(s):
    k = s["k"]

    def dequant(codes, scales):   # scales [rows, blocks]
        full = scales.repeat_interleave(BLOCK, dim=1)[:, :k]
        return codes[:, :k].float() * full

    a = dequant(s["a"], s["a_scales"].t())
    b = dequant(s["b"], s["b_scales"].repeat_interleave(BLOCK, dim=0)[:s["n"]])
    out = a @ b.t()
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return _act_plain(out, s["act"]).to(DTYPES[s["dtype"]])


def _attention_plain(s):
    h, hk, d, n = s["heads"], s["kv_heads"], s["head_dim"], s["q_len"]
    group, scale = h // hk, 1.0 / math.sqrt(d)
    out = torch.empty_like(s["q"])
    step = 512
    for b in range(s["batch"]):
        for i0 in range(0, n, step):
            i1 = min(i0 + step, n)
            p0, p1, valid = s["starts"][b] + i0, s["starts"][b] + i1 - 1, s["lens"][b]
            lo, hi = max(0, p0 - s["left"]), max(0, min(valid, p1 + s["right"] + 1))
            lo = min(lo, hi)
            first = min(s["sinks"], lo)
            pos = torch.cat([torch.arange(first, device="cuda"), torch.arange(lo, hi, device="cuda")])
            k = torch.cat([s["k"][b, :first], s["k"][b, lo:hi]]).float().permute(1, 0, 2).contiguous()
            v = torch.cat([s["v"][b, :first], s["v"][b, lo:hi]]).float().permute(1, 0, 2).contiguous()
            q = s["q"][b, i0:i1].float().view(i1 - i0, hk, group, d).permute(1, 2, 0, 3)
            q = q.reshape(hk, group * (i1 - i0), d)
            at = torch.arange(p0, p1 + 1, device="cuda")[:, None]
            seen = (pos <= at + s["right"]) & ((pos >= at - s["left"]) | (pos < s["sinks"]))
            seen = seen.repeat(group, 1)
            score = (q @ k.transpose(1, 2).contiguous()) * scale
            score = torch.where(seen, score, torch.full_like(score, -math.inf))
            top = score.amax(dim=-1, keepdim=True)
            p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            total = p.sum(dim=-1, keepdim=True)
            o = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
            o = o.view(hk, group, i1 - i0, d).permute(2, 0, 1, 3).reshape(i1 - i0, h, d)
            out[b, i0:i1] = o.to(out.dtype)
    return out


def run(s):
    if s["op"] == "quantize":
        if own:
            import burnisher_amd as bh
            bh.call("bh_quantize_fp8", bh.ptr(s["x"]), s["cols"], bh.ptr(s["out"]), bh.ptr(s["scales"]), s["rows"],
                    s["cols"], s["block_rows"], bh.BF16 if s["dtype"] == "bf16" else bh.F32, bh.stream_ptr())
            codes, scales = s["out"], s["scales"]
        else:
            codes, scales = _quantize_plain(s["x"], s["block_rows"])
        return {"codes": codes[:, :s["cols"]], "scales": scales}
    if s["op"] == "gemm":
        if not own:
            return _gemm_plain(s)
        import burnisher_amd as bh
        bh.call("bh_gemm_fp8", bh.ptr(s["a"]), bh.ptr(s["a_scales"]), bh.ptr(s["b"]), bh.ptr(s["b_scales"]),
                bh.ptr(s["bias"]), bh.ptr(s["out"]), s["m"], s["n"], s["k"], s["act"],
                bh.BF16 if s["dtype"] == "bf16" else bh.F32, bh.ptr(s["workspace"]), s["workspace"].numel(),
                bh.stream_ptr())
        return s["out"]
    if not own:
        return _attention_plain(s)
    import burnisher_amd as bh
    d = s["head_dim"]
    bh.call("bh_attention_window", bh.ptr(s["q"]), s["heads"] * d, bh.ptr(s["k"]), bh.ptr(s["v"]),
            s["kv_heads"] * d, bh.ptr(s["out"]), s["heads"] * d, s["batch"], s["heads"], s["kv_heads"], s["q_len"],
            s["kv_len"], d, 0.0, s["left"], s["right"], s["sinks"], bh.ptr(s["lens_dev"]), bh.ptr(s["starts_dev"]),
            bh.BF16, bh.ptr(s["workspace"]), s["workspace"].numel(), bh.stream_ptr())
    return s["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    if case["op"] == "quantize":
        rows, cols, br = case["rows"], case["cols"], case["block_rows"]
        size = 2 if case["dtype"] == "bf16" else 4
        scales = -(-cols // BLOCK) * -(-rows // br)
        return {"bytes": rows * cols * size + rows * _pad16(cols) + 4 * scales, "flops": 3 * rows * cols}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        size, blocks = (2 if case["dtype"] == "bf16" else 4), -(-k // BLOCK)
        scales = 4 * blocks * (m + -(-n // BLOCK))
        return {"bytes": (m + n) * _pad16(k) + scales + (m + bool(case["bias"])) * n * size, "flops": 2 * m * n * k}
    # Keys seen, with every sequence as long as the case allows on average; a query row reads and writes once.
    lens = [case["kv_len"]] * case["batch"] if case["lens"] == "full" else \
        [case["kv_len"]] + [max(case["q_len"] if case["at_end"] else 1, case["kv_len"] * 5 // 8)] * (case["batch"] - 1)
    pairs = keys = 0
    for valid in lens:
        start = valid - case["q_len"] if case["at_end"] else 0
        lowest, top = valid, 0
        for i in range(case["q_len"]):
            hi = max(0, min(valid, start + i + case["right"] + 1))
            lo = min(max(0, start + i - case["left"]), hi)
            pairs += hi - lo + min(case["sinks"], lo)
            lowest, top = min(lowest, lo), max(top, hi)
        keys += max(0, top - lowest) + min(case["sinks"], lowest)
    d = case["head_dim"]
    return {"bytes": 2 * d * (2 * case["batch"] * case["q_len"] * case["heads"] + 2 * keys * case["kv_heads"]),
            "flops": 4 * d * pairs * case["heads"]}


# ---- the definition in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "quantize":
        # value / (largest magnitude / 448) and that scale, neither rounded
        v, br = x["x"].double(), case["block_rows"]
        codes = torch.empty_like(v)
        nr, nc = -(-case["rows"] // br), -(-case["cols"] // BLOCK)
        scales = torch.empty((nr, nc), dtype=torch.float64, device="cuda")
        for c in range(nc):
            cols = slice(c * BLOCK, min((c + 1) * BLOCK, case["cols"]))
            for r0 in ([0] if br == 1 else range(0, case["rows"], br)):
                part = v[:, cols] if br == 1 else v[r0:r0 + br, cols]
                top = part.abs().max(dim=1, keepdim=True).values if br == 1 else part.abs().max().view(1, 1)
                top = torch.maximum(top, torch.full_like(top, AMAX_FLOOR))
                if br == 1:
                    codes[:, cols] = part / top * E4M3_MAX
                    scales[:, c] = top[:, 0] / E4M3_MAX
                else:
                    codes[r0:r0 + br, cols] = part / top * E4M3_MAX
                    scales[r0 // br, c] = top[0, 0] / E4M3_MAX
        return {"codes": codes, "scales": scales.t().contiguous() if br == 1 else scales}
    if case["op"] == "gemm":
        # sum over blocks of 128: the codes' product, times both scales
        a, b = x["a"].double(), x["b"].double()
        total = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        of_column = torch.arange(case["n"], device="cuda") // BLOCK
        for j in range(-(-case["k"] // BLOCK)):
            cols = slice(j * BLOCK, min((j + 1) * BLOCK, case["k"]))
            part = torch.mm(a[:, cols].contiguous(), b[:, cols].t().contiguous())
            total += part * x["a_scales"][j].double()[:, None] * x["b_scales"][of_column, j].double()
        if x["bias"] is not None:
            total += x["bias"].double()
        if case["act"] == 1:
            total = total / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (total + 0.044715 * total ** 3)))
        elif case["act"] == 2:
            total = total * torch.sigmoid(total)
        return total
    lens, starts = x["lens"], x["starts"]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    rows = torch.arange(case["q_len"], device="cuda")
    for b in range(case["batch"]):
        keys = torch.arange(lens[b], device="cuda")
        for i in range(0, case["q_len"], 1024):
            at = starts[b] + rows[i:i + 1024]
            # the keys that some query of this piece sees
            near = (keys >= at[0] - case["left"]) & (keys <= at[-1] + case["right"])
            use = torch.nonzero(near | ((keys < case["sinks"]) & (keys <= at[-1] + case["right"])))[:, 0]
            if use.numel() == 0:
                continue
            gap = use[None, :] - at[:, None]
            hidden = ~((gap <= case["right"]) & ((gap >= -case["left"]) | (use < case["sinks"])[None, :]))
            for h in range(case["heads"]):
                kh, vh = x["k"][b, use, h // group].double(), x["v"][b, use, h // group].double()
                s = torch.mm(x["q"][b, i:i + 1024, h].double(), kh.t().contiguous()) / math.sqrt(case["head_dim"])
                s.masked_fill_(hidden, -math.inf)
                out[b, i:i + 1024, h] = torch.nan_to_num(torch.softmax(s, dim=1), nan=0.0) @ vh
    return out
