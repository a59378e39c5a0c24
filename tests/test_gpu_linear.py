"""bh_attention_linear on the GPU against its definition in 64 bits on the same bf16 inputs.

The tolerance counts what is rounded, in parts of A, the sum of the magnitudes that an output (or an element of a
state) adds up. A power of the decay, 2^x, is off by |x| 2^-24 of x's own rounding and 2 ulp, and |x| 2^-x is below
0.6, so by less than 2^-22 of 1; each token or chunk rounds the state twice at most, 2^-23 a token; a sum
of head_dim products adds head_dim 2^-24, and the tokens of a chunk and the terms of a split value 2^-18.
Scores and states that enter an output are sums of two bf16 values, off by 2^-16 each. The output is
rounded once. What a state is off by has no 2^-16 in it.
"""
import ctypes
import math

import pytest

import burnisher_amd as bh

pytestmark = pytest.mark.gpu


def normal(shape, seed, std=1.0, dtype=None):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype or torch.bfloat16)


def plain(q, k, v, log_decay, lens, state, scale=None):
    """(out, tolerance, state, tolerance) in 64 bits: every pair of tokens."""
    import torch
    batch, n, heads, d = q.shape
    kvh, e = k.shape[2], v.shape[3]
    group, scale = heads // kvh, scale or 1 / math.sqrt(d)
    out = torch.zeros(batch, n, heads, e, dtype=torch.float64, device="cuda")
    tol, new, new_tol = torch.zeros_like(out), torch.zeros(batch, kvh, d, e, dtype=torch.float64, device="cuda"), None
    new_tol = torch.zeros_like(new)
    rates = log_decay.double().nan_to_num(nan=0.0, neginf=-1e30).clamp(max=0.0).tolist()
    steps = n * 2.0 ** -23 + 2.0 ** -22 + d * 2.0 ** -24 + 2.0 ** -20
    for b in range(batch):
        m = n if lens is None else max(0, min(lens[b], n))
        at = torch.arange(m, device="cuda", dtype=torch.float64)
        for h in range(kvh):
            kk, vv = k[b, :m, h].double(), v[b, :m, h].double()
            s0 = torch.zeros(d, e, dtype=torch.float64, device="cuda") if state is None else state[b, h].double()
            w = torch.exp((rates[h] * (m - 1 - at)).nan_to_num())[:, None]
            keep = math.exp(rates[h] * m) if m else 1.0
            new[b, h] = (kk * w).t().contiguous() @ vv + keep * s0
            new_tol[b, h] = ((kk.abs() * w).t().contiguous() @ vv.abs() + keep * s0.abs()) * steps
            gap = at[:, None] - at[None, :]
            w = torch.exp((rates[h] * gap.clamp(min=0)).nan_to_num()) * (gap >= 0)
            first = torch.exp((rates[h] * (at + 1)))[:, None]
            for g in range(group):
                qq = q[b, :m, h * group + g].double() * scale
                out[b, :m, h * group + g] = ((qq @ kk.t().contiguous()) * w) @ vv + first * (qq @ s0)
                size = ((qq.abs() @ kk.abs().t().contiguous()) * w) @ vv.abs() + first * (qq.abs() @ s0.abs())
                tol[b, :m, h * group + g] = size * (steps + 2.0 ** -15)
    return out, tol + out.abs() * 2.0 ** -8 + 1e-37, new, new_tol + 1e-37


def ld_of(t):
    return t.stride(1) if t.shape[1] > 1 else max(t.stride(0), t.shape[2] * t.shape[3])


def call(q, k, v, out, log_decay, lens, state_in, state_out, scale, ws, ws_bytes, stream=None):
    batch, n, heads, d = q.shape
    bh.call("bh_attention_linear", q.data_ptr(), ld_of(q), k.data_ptr(), ld_of(k), v.data_ptr(), ld_of(v), out.data_ptr(), ld_of(out),
            batch, heads, k.shape[2], n, d, v.shape[3], scale, log_decay.data_ptr(), bh.ptr(lens), bh.ptr(state_in), bh.ptr(state_out),
            bh.BF16, bh.ptr(ws), ws_bytes, bh.stream_ptr(stream))


def workspace(q, k, v, fill=0xff):
    import torch
    need = bh.lib().bh_attention_linear_workspace_bytes(q.shape[0], q.shape[2], k.shape[2], q.shape[1], q.shape[3], v.shape[3])
    assert need >= 0
    return torch.full((max(need, 16),), fill, dtype=torch.uint8, device="cuda"), need


def run(q, k, v, log_decay, lens=None, state=None, scale=0.0, with_workspace=True, out=None, in_place=False, want_state=True):
    """(out, state behind the last token)."""
    import torch
    dl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    if out is None:
        out = torch.full((*q.shape[:3], v.shape[3]), 9.0, dtype=torch.bfloat16, device="cuda")
    new = torch.full((q.shape[0], k.shape[2], q.shape[3], v.shape[3]), 9.0, device="cuda")
    if in_place:
        new = state = state.clone()
    ws, need = workspace(q, k, v)
    call(q, k, v, out, log_decay, dl, state, new if want_state else None, scale, ws if with_workspace else None,
         need if with_workspace else 0)
    torch.cuda.synchronize()
    return out, new


def compare(got, want, tol, what="out"):
    bad = ~((got.double() - want).abs() <= tol)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {got[at]} for {want[at]} +- {tol[at]}")


def decays(kvh, seed=0, slow=8.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return -torch.exp2(-slow * torch.rand(kvh, generator=g, device="cuda"))


def inputs(batch, heads, kvh, n, d, e, seed=0):
    return normal((batch, n, heads, d), seed), normal((batch, n, kvh, d), seed + 1), normal((batch, n, kvh, e), seed + 2)


def check(batch, heads, kvh, n, d, e, lens=None, with_state=True, seed=0, log_decay=None, **how):
    import torch
    q, k, v = inputs(batch, heads, kvh, n, d, e, seed)
    state = normal((batch, kvh, d, e), seed + 3, 2.0, torch.float32) if with_state else None
    log_decay = decays(kvh, seed) if log_decay is None else log_decay
    out, new = run(q, k, v, log_decay, lens, state, **how)
    want, tol, new_want, new_tol = plain(q, k, v, log_decay, lens, state)
    compare(out, want, tol)
    if how.get("want_state", True):
        compare(new, new_want, new_tol, "state")
    return out, new


LENGTHS = [1, 2, 3, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 95, 127, 128, 130, 200, 257, 500]


@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("n", LENGTHS)
def test_lengths(hip, n, with_state):
    check(2, 4, 2, n, 64, 64, with_state=with_state, seed=n)
    check(3, 3, 3, n, 128, 128, lens=[n, n // 2, 1], with_state=with_state, seed=n)
    check(1, 6, 1, n, 72, 40, with_state=with_state, seed=n)


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 64, 72, 80, 88, 96, 104, 112, 120, 128])
@pytest.mark.parametrize("n", [1, 5, 150])
def test_head_dims(hip, n, d):
    check(2, 2, 2, n, d, d, lens=[n, max(1, n - 40)], seed=d)
    check(1, 4, 2, n, d, 136 - d if d < 128 else 8, seed=d)


@pytest.mark.parametrize("heads,kvh", [(1, 1), (8, 1), (32, 8), (6, 6), (40, 2)])
@pytest.mark.parametrize("n", [1, 4, 70])
def test_grouped_heads(hip, n, heads, kvh):
    check(2, heads, kvh, n, 64, 128, seed=heads)


# enough heads that no sequence is split, and few heads with long sequences
@pytest.mark.parametrize("batch,heads,kvh,n,d", [(16, 64, 64, 100, 64), (8, 64, 16, 77, 128), (1, 1, 1, 5000, 128), (1, 4, 2, 3001, 64),
                                                 (2, 8, 2, 2049, 72), (1, 2, 2, 4096, 96)])
@pytest.mark.parametrize("with_workspace", [True, False])
def test_few_and_many_heads(hip, batch, heads, kvh, n, d, with_workspace):
    lens = [n - 7 * b if b % 3 else n for b in range(batch)]
    check(batch, heads, kvh, n, d, d, lens=lens, seed=n, with_workspace=with_workspace)


@pytest.mark.parametrize("n", [1, 40, 300, 2500])
def test_lengths_of_nothing_and_beyond(hip, n):
    import torch
    lens = [0, 1, -5, 2 ** 31 - 1, n // 2]
    q, k, v = inputs(5, 4, 2, n, 64, 64, n)
    state, rate = normal((5, 2, 64, 64), 9, 1.0, torch.float32), decays(2)
    out, new = run(q, k, v, rate, lens, state)
    want, tol, new_want, new_tol = plain(q, k, v, rate, lens, state)
    compare(out, want, tol)
    compare(new, new_want, new_tol, "state")
    assert not out[0].any() and not out[2].any() and torch.equal(new[0], state[0]) and torch.equal(new[2], state[2])
    out, new = run(q, k, v, rate, lens, None)
    assert not out[0].any() and not new[0].any() and not new[2].any()


def test_no_tokens_copy_the_state(hip):
    import torch
    state = normal((2, 3, 64, 72), 1, 1.0, torch.float32)
    empty = torch.empty(2, 0, 3, 64, dtype=torch.bfloat16, device="cuda")
    new, rate = torch.full_like(state, 9.0), decays(3)
    for start, want in ((state, state), (None, torch.zeros_like(state))):
        bh.call("bh_attention_linear", None, 192, None, 192, None, 216, None, 216, 2, 3, 3, 0, 64, 72, 0.0, rate.data_ptr(), None,
                bh.ptr(start), new.data_ptr(), bh.BF16, None, 0, bh.stream_ptr())
        torch.cuda.synchronize()
        assert torch.equal(new, want)
    assert empty.numel() == 0


@pytest.mark.parametrize("n", [1, 20, 200, 3000])
def test_decays_at_their_ends(hip, n):
    import torch
    # none, almost none, the fastest, above 0 (none), not a number (none)
    rate = torch.tensor([0.0, -1e-6, -20.0, -math.inf, 3.0, math.nan, -1e-40, -3e38], device="cuda")
    out, new = check(1, 8, 8, n, 64, 64, log_decay=rate, seed=n)
    assert torch.isfinite(out.float()).all() and torch.isfinite(new).all()


def test_a_slow_decay_over_many_chunks_keeps_its_digits(hip):
    import torch
    # no keys: only the first state decays, by exp(-1e-5 * 60000). Its factor per chunk is applied as 1 - (1 - f), so each
    # of at most 60000 steps rounds once: 2^-24 sqrt(60000) = 2^-16 as a random walk, 4 times that at most
    n, rate = 60000, torch.tensor([-1e-5, -2e-5], device="cuda")
    q, k, v = inputs(1, 2, 2, n, 64, 64, 1)
    k.zero_()
    state = normal((1, 2, 64, 64), 9, 1.0, torch.float32)
    out, new = run(q, k, v, rate, None, state)
    want = state.double() * torch.exp(rate.double() * n)[None, :, None, None]
    assert ((new.double() - want).abs() <= want.abs() * 2.0 ** -14).all()


@pytest.mark.parametrize("n", [20, 32, 100, 150])
def test_states_keep_24_bits(hip, n):
    import torch
    # one token holds a key: its term of the state is decay^(n - 1 - t) k v, rounded a few times at 2^-24 and
    # no more than the chunks behind it
    q, k, v = inputs(1, 2, 2, n, 64, 64, n)
    rate = torch.tensor([-0.01, -0.003], device="cuda")
    for t in (0, n // 2, n - 1):
        one = torch.zeros_like(k)
        one[:, t] = k[:, t]
        _, new = run(q, one, v, rate)
        w = torch.exp(rate.double() * (n - 1 - t))[None, :, None, None]
        want = w * k[:, t].double()[..., :, None] * v[:, t].double()[..., None, :]
        # the decay's power: 2 ulp and its exponent's rounding, (n - t) * 0.01 * 1.5 * 2^-24
        slack = 2.0 ** -24 * (4 + 4 + (n if n < 32 else 2 * (n // 32 + 1)) + 0.02 * n)
        assert ((new.double() - want).abs() <= want.abs() * slack + 1e-37).all(), t


@pytest.mark.parametrize("n", [1, 10, 200, 3000])
@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_what_lies_behind_a_sequence_never_enters(hip, n, poison):
    import torch
    lens = [n, (n + 1) // 2, 1, 0]
    q, k, v = inputs(4, 4, 2, n, 64, 64, n)
    for b in range(4):
        q[b, lens[b]:], k[b, lens[b]:], v[b, lens[b]:] = poison, poison, poison
    rate = decays(2)
    out, new = run(q, k, v, rate, lens)
    want, tol, new_want, new_tol = plain(q, k, v, rate, lens, None)
    compare(out, want, tol)
    compare(new, new_want, new_tol, "state")


@pytest.mark.parametrize("poison", [math.nan, math.inf])
@pytest.mark.parametrize("n,at", [(200, 100), (3000, 1700)])
def test_a_bad_value_stays_behind_its_chunk(hip, n, at, poison):
    import torch
    q, k, v = inputs(1, 4, 2, n, 64, 64, n)
    rate = decays(2)
    want, _ = run(q, k, v, rate)
    v[0, at, 0, 5] = poison
    out, new = run(q, k, v, rate)
    before = at - 31
    assert torch.equal(out[:, :before], want[:, :before]), "reached back more than 31 tokens"
    assert torch.equal(out[:, :, 2:], want[:, :, 2:]), "reached another head"
    assert not torch.isfinite(out[0, at, :2, 5].float()).any() and not torch.isfinite(new[0, 0, :, 5]).any()


@pytest.mark.parametrize("n", [1, 90, 2100])
def test_strided_operands_and_untouched_gaps(hip, n):
    import torch
    batch, heads, kvh, d, e = 2, 6, 2, 72, 40
    fused = normal((batch, n, heads * d + kvh * (d + e) + 8), 4)
    q = fused[:, :, :heads * d].unflatten(2, (heads, d))
    k = fused[:, :, heads * d:(heads + kvh) * d].unflatten(2, (kvh, d))
    v = fused[:, :, (heads + kvh) * d:(heads + kvh) * d + kvh * e].unflatten(2, (kvh, e))
    buf = torch.full((batch, n, heads * e + 12), 5.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, :, :heads * e].unflatten(2, (heads, e))
    rate = decays(kvh)
    _, new = run(q, k, v, rate, out=out)
    want, tol, new_want, new_tol = plain(q, k, v, rate, None, None)
    compare(out, want, tol)
    compare(new, new_want, new_tol, "state")
    assert (buf[:, :, heads * e:] == 5.0).all()


@pytest.mark.parametrize("n,batch,heads,kvh", [(1, 3, 8, 2), (33, 3, 8, 2), (300, 2, 8, 2), (100, 16, 64, 16), (100, 16, 64, 64), (3000, 1, 4, 1)])
def test_state_in_place(hip, n, batch, heads, kvh):
    import torch
    q, k, v = inputs(batch, heads, kvh, n, 64, 64, n)
    state, rate = normal((batch, kvh, 64, 64), 9, 1.0, torch.float32), decays(kvh)
    for with_workspace in (True, False):
        out, new = run(q, k, v, rate, None, state, with_workspace=with_workspace)
        out2, new2 = run(q, k, v, rate, None, state, with_workspace=with_workspace, in_place=True)
        assert torch.equal(out, out2) and torch.equal(new, new2)
    alone, _ = run(q, k, v, rate, None, state, want_state=False)
    compare(alone, *plain(q, k, v, rate, None, state)[:2])


def test_scale(hip):
    q, k, v = inputs(1, 2, 2, 100, 64, 64, 1)
    rate = decays(2)
    compare(run(q, k, v, rate, scale=0.7)[0], *plain(q, k, v, rate, None, None, 0.7)[:2])


def test_prompt_in_pieces_is_the_prompt(hip):
    """Chunks of a prompt and then single tokens, the state handed on: as one call, within both tolerances."""
    import torch
    batch, heads, kvh, d, n = 2, 8, 2, 64, 700
    q, k, v = inputs(batch, heads, kvh, n, d, d, 5)
    rate, state, at, parts = decays(kvh), None, 0, []
    for m in (300, 1, 64, 2, 300, 31, 1, 1):
        piece = [t[:, at:at + m].contiguous() for t in (q, k, v)]
        out, state = run(*piece, rate, None, state)
        parts.append(out)
        at += m
    assert at == n
    want, tol, new_want, new_tol = plain(q, k, v, rate, None, None)
    compare(torch.cat(parts, 1), want, tol)
    compare(state, new_want, new_tol, "state")


def test_offsets_beyond_32_bits(hip):
    import torch
    # two sequences whose rows are 2^21 elements apart: the second starts more than 2^32 bytes in
    n, ld, heads, d = 1100, 2 ** 21, 2, 64
    buffer = torch.empty(2 * n * ld, dtype=torch.bfloat16, device="cuda").view(2, n, ld)
    views = [buffer[:, :, 8 * i * 64:8 * i * 64 + heads * d].unflatten(2, (heads, d)) for i in range(4)]
    q, k, v = inputs(2, heads, heads, n, d, d, 3)
    for view, t in zip(views, (q, k, v)):
        view.copy_(t)
    rate = decays(heads)
    _, new = run(*views[:3], rate, out=views[3])
    want, tol, new_want, new_tol = plain(q, k, v, rate, None, None)
    compare(views[3], want, tol)
    compare(new, new_want, new_tol, "state")
    one = [t[:, :1] for t in views[:3]]
    out = torch.empty(2, 1, heads, d, dtype=torch.bfloat16, device="cuda")
    ws, need = workspace(*one)
    new = torch.empty(2, heads, d, d, device="cuda")
    # a batch row here is a row of the buffer's stride: the first two tokens of the first sequence
    bh.call("bh_attention_linear", views[0].data_ptr(), ld, views[1].data_ptr(), ld, views[2].data_ptr(), ld, out.data_ptr(), heads * d,
            2, heads, heads, 1, d, d, 0.0, rate.data_ptr(), None, None, new.data_ptr(), bh.BF16, ws.data_ptr(), need, bh.stream_ptr())
    want, tol, _, _ = plain(q[0, :2, None], k[0, :2, None], v[0, :2, None], rate, None, None)
    compare(out, want, tol)


def test_stays_inside_its_workspace_and_refuses_a_small_one(hip):
    import torch
    q, k, v = inputs(1, 4, 2, 3000, 64, 64, 1)
    rate, out = decays(2), torch.zeros(1, 3000, 4, 64, dtype=torch.bfloat16, device="cuda")
    new = torch.zeros(1, 2, 64, 64, device="cuda")
    _, need = workspace(q, k, v)
    assert need > 0
    ws = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
    with pytest.raises(bh.BurnisherError, match="this call needs"):
        call(q, k, v, out, rate, None, None, new, 0.0, ws, need - 1)
    with pytest.raises(bh.BurnisherError, match="16-byte"):
        call(q, k, v, out, rate, None, None, new, 0.0, ws[4:], need)
    torch.cuda.synchronize()
    assert not out.any() and not new.any() and (ws == 0x5a).all(), "a refused call wrote"
    call(q, k, v, out, rate, None, None, new, 0.0, ws, need)
    torch.cuda.synchronize()
    assert (ws[need:] == 0x5a).all(), "written past the workspace"
    again, state = run(q, k, v, rate)
    assert torch.equal(out, again) and torch.equal(new, state)


@pytest.mark.parametrize("n", [1, 50, 2500])
def test_in_a_graph_and_on_two_streams(hip, n):
    import torch
    batch, heads, kvh, d = 2, 8, 2, 64
    sets = [inputs(batch, heads, kvh, n, d, d, s) for s in (1, 11)]
    states = [normal((batch, kvh, d, d), s, 1.0, torch.float32) for s in (4, 14)]
    lens, rate = torch.tensor([n, (n + 1) // 2], dtype=torch.int32, device="cuda"), decays(kvh)
    outs, news = [torch.zeros_like(s[0]) for s in sets], [torch.zeros_like(s) for s in states]
    ws = [workspace(*s) for s in sets]

    def one(i, stream):
        call(*sets[i], outs[i], rate, lens, states[i], news[i], 0.0, ws[i][0], ws[i][1], stream)

    want = [run(*s, rate, [n, (n + 1) // 2], x) for s, x in zip(sets, states)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for i in (0, 1):
            one(i, streams[i])
    torch.cuda.synchronize()
    for i in (0, 1):
        assert torch.equal(outs[i], want[i][0]) and torch.equal(news[i], want[i][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(0, torch.cuda.current_stream())
    for seed, new_lens in ((5, [n, n]), (6, [1, 0]), (7, [n // 2, n])):
        for t, s in zip(sets[0], range(3)):
            t.copy_(normal(tuple(t.shape), seed + s))
        lens.copy_(torch.tensor(new_lens, dtype=torch.int32))
        outs[0].fill_(3.0)
        news[0].fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        got = run(*sets[0], rate, new_lens, states[0])
        assert torch.equal(outs[0], got[0]) and torch.equal(news[0], got[1]), "a replay differs from the call"


def test_a_block_of_linear_attention(hip):
    """Norm, projection, rotary positions, linear attention, output projection and the norms around the residual as a
    model runs them: a prompt with its state, then a token. The token equals, within the roundings, the last row of
    one run over prompt and token together."""
    import torch
    batch, n, heads, kvh, d, width = 2, 75, 8, 2, 64, 512
    w_qkv, w_out = normal(((heads + 2 * kvh) * d, width), 1, 0.04), normal((width, heads * d), 2, 0.04)
    weight, rate = normal((width,), 3, 0.2) + 1, decays(kvh)
    axes = bh.RopeAxes.of([16, 16], interleaved=True)
    norms = bh.ResidualNorms(post_norm=bh.NORM_RMS, post_weight=weight.data_ptr(), post_eps=1e-6, branch_scale=1.0, residual_scale=1.0,
                             pre_norm=bh.NORM_RMS, pre_weight=weight.data_ptr(), pre_eps=1e-6, mod_rows=1, ld_mod=width)

    def project(x, w):
        out = torch.empty(x.shape[0], w.shape[0], dtype=torch.bfloat16, device="cuda")
        bh.call("bh_gemm", x.data_ptr(), w.data_ptr(), None, out.data_ptr(), x.shape[0], w.shape[0], x.shape[1], 1, 0, bh.BF16, bh.stream_ptr())
        return out

    def block(x, first, state):
        """x [batch, m, width] of the tokens from `first` on: the stream, its norm and the state behind them."""
        m = x.shape[1]
        rows = x.reshape(batch * m, width)
        normed = torch.empty_like(rows)
        bh.call("bh_norm", rows.data_ptr(), weight.data_ptr(), None, normed.data_ptr(), batch * m, width, 1e-6, 1, 0, 0, bh.BF16, bh.stream_ptr())
        fused = project(normed, w_qkv)
        t = torch.arange(first, first + m, device="cuda", dtype=torch.int32)
        positions = torch.stack([t // 10, t % 10], 1).contiguous()
        q, k = torch.empty(batch, m, heads, d, dtype=torch.bfloat16, device="cuda"), torch.empty(batch, m, kvh, d, dtype=torch.bfloat16, device="cuda")
        bh.call("bh_rope", ctypes.byref(axes), positions.data_ptr(), m, fused.data_ptr(), fused.stride(0), q.data_ptr(), heads * d, heads,
                fused[:, heads * d:].data_ptr(), fused.stride(0), k.data_ptr(), kvh * d, kvh, batch * m, d, 0, bh.BF16, bh.stream_ptr())
        v = fused.view(batch, m, -1)[:, :, (heads + kvh) * d:].unflatten(2, (kvh, d))
        out, state = run(q, k, v.contiguous(), rate, None, state)
        branch = project(out.view(batch * m, heads * d), w_out)
        stream, after = torch.empty_like(rows), torch.empty_like(rows)
        bh.call("bh_residual_norms_run", branch.data_ptr(), width, rows.data_ptr(), width, stream.data_ptr(), width, after.data_ptr(), width,
                batch * m, width, ctypes.byref(norms), bh.BF16, bh.BF16, bh.stream_ptr())
        torch.cuda.synchronize()
        return stream.view(batch, m, width), after.view(batch, m, width), state

    x = normal((batch, n, width), 4)
    stream, after, state = block(x, 0, None)
    _, _, handed = block(x[:, :n - 1].contiguous(), 0, None)
    one_stream, one_after, one_state = block(x[:, n - 1:].contiguous(), n - 1, handed)
    assert torch.isfinite(after.float()).all()
    # q, k, v and the attention's output are bf16 in both, and may differ by a step where sums were taken in
    # another order: four bf16 roundings, 4 * 2^-8 of the largest value, through a norm of unit size and its weight
    for got, want in ((one_stream, stream[:, n - 1:]), (one_after, after[:, n - 1:])):
        assert (got.float() - want.float()).abs().max() <= 4 * 2.0 ** -8 * want.float().abs().max()
    assert (one_state - state).abs().max() <= 2.0 ** -8 * state.abs().max()


def heads_at_once(batch, heads, kvh, n, d, e, with_workspace=True):
    plan = bh.AttentionLinearPlan()
    bh.call("bh_attention_linear_describe", batch, heads, kvh, n, d, e, int(with_workspace), 0, ctypes.byref(plan))
    return batch * heads * plan.segments / plan.workgroups


# enough workgroups that two heads of a group share one, with a CU to themselves or not; 65 tokens end in a chunk of one
@pytest.mark.parametrize("d", [8, 24, 32, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("batch,heads,kvh", [(8, 64, 16), (24, 48, 8)])
def test_two_heads_at_once(hip, batch, heads, kvh, d):
    for n, e in ((65, d), (20, 136 - d if d < 128 else 8)):
        assert heads_at_once(batch, heads, kvh, n, d, e) == 2
        check(batch, heads, kvh, n, d, e, lens=[max(0, n - 9 * (b % 9)) for b in range(batch)], seed=d)


@pytest.mark.parametrize("n,batch,heads,kvh,d", [(50, 12, 64, 16, 128), (50, 12, 32, 16, 128), (3000, 2, 16, 4, 128), (3000, 4, 12, 2, 64)])
def test_two_heads_at_once_in_place_and_captured(hip, n, batch, heads, kvh, d):
    """The state in place, with a workspace and without, where a workgroup takes a group's heads in turns of two; a replay."""
    import torch
    q, k, v = inputs(batch, heads, kvh, n, d, d, n)
    state, rate = normal((batch, kvh, d, d), 9, 1.0, torch.float32), decays(kvh)
    want, tol, new_want, new_tol = plain(q, k, v, rate, None, state)
    for with_workspace in (True, False):
        if with_workspace:
            assert heads_at_once(batch, heads, kvh, n, d, d) == 2
        out, new = run(q, k, v, rate, None, state, with_workspace=with_workspace, in_place=True)
        compare(out, want, tol)
        compare(new, new_want, new_tol, "state")
    (ws, need), out, new = workspace(q, k, v), torch.zeros_like(v.new_empty(batch, n, heads, d)), torch.zeros_like(state)
    eager = run(q, k, v, rate, None, state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q, k, v, out, rate, None, state, new, 0.0, ws, need, torch.cuda.current_stream())
    for _ in range(3):
        out.fill_(3.0)
        new.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(new, eager[1])


@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_a_head_of_two_at_once_stays_alone(hip, poison):
    """What is wrong with one query head's queries does not reach the head beside it, the other groups or the state."""
    import torch
    batch, heads, kvh, n, d = 12, 64, 16, 50, 64
    assert heads_at_once(batch, heads, kvh, n, d, d) == 2
    q, k, v = inputs(batch, heads, kvh, n, d, d, 3)
    rate = decays(kvh)
    clean, state = run(q, k, v, rate)
    q[:, 17, 6] = poison
    out, new = run(q, k, v, rate)
    others = [h for h in range(heads) if h != 6]
    assert torch.equal(out[:, :, others], clean[:, :, others]) and torch.equal(new, state)
    assert not out[:, 17, 6].isfinite().any()
    assert torch.equal(out[:, :17, 6], clean[:, :17, 6]) and torch.equal(out[:, 18:, 6], clean[:, 18:, 6])
