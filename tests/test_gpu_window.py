"""bh_attention_window on the GPU against its definition in 64 bits on the same bf16 inputs.

The tolerance counts what is rounded: a weight to bf16 for the matrix product (2^-8 of it), the output
to bf16 (2^-8 of the value) and the score's fp32 sum of head_dim products, whose error is a relative
error of its weight.
"""
import math

import pytest

from helpers import BF16

pytestmark = pytest.mark.gpu


def normal(shape, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def sees(positions, length, kv_len, left, right, sinks):
    """[queries, kv_len] truth values."""
    import torch
    j = torch.arange(kv_len, device="cuda")[None, :]
    p = positions[:, None]
    ok = (j < max(0, min(length, kv_len))).expand(p.shape[0], kv_len).clone()
    if right >= 0:
        ok &= j <= p + right
    if left >= 0:
        ok &= (j >= p - left) | (j < sinks)
    return ok


def plain(q, k, v, lens, starts, left, right, sinks, scale=None):
    """(64-bit result, tolerance), both [batch, q_len, heads, head_dim]."""
    import torch
    batch, n, heads, d = q.shape
    kv_len, group = k.shape[1], heads // k.shape[2]
    scale = scale or 1 / math.sqrt(d)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for b in range(batch):
        pos = torch.arange(n, device="cuda") + starts[b]
        ok = sees(pos, lens[b], kv_len, left, right, sinks)
        any_ok = ok.any(1)
        for h in range(heads):
            kk, vv = k[b, :, h // group].double(), v[b, :, h // group].double()
            used = ok.any(0)
            kk, vv = torch.where(used[:, None], kk, 0), torch.where(used[:, None], vv, 0)
            qq = q[b, :, h].double()
            s = (qq @ kk.t().contiguous()) * scale
            size = (qq.abs() @ kk.t().abs().contiguous()) * scale
            s = torch.where(ok, s, -math.inf)
            w = torch.where(any_ok[:, None], torch.softmax(s, 1).nan_to_num(0.0), 0)
            delta = ((d + 8) * 2.0 ** -23 * torch.where(ok, size, 0).amax(1) + 2.0 ** -20)[:, None] \
                if kv_len else torch.zeros(n, 1, dtype=torch.float64, device="cuda")
            out[b, :, h] = w @ vv
            # the weight's rounding, twice its score's error (numerator and denominator), the output's
            tol[b, :, h] = (w @ vv.abs()) * (2.0 ** -8 + 2 * delta) + out[b, :, h].abs() * (2.0 ** -8 + 2 * delta)
    return out, tol + 1e-30


def run(q, k, v, lens, starts, left, right, sinks, scale=0.0, workspace=True, out=None, stream=None):
    """q, k, v [batch, len, heads, head_dim], views with any row stride; lens and starts lists or None."""
    import torch
    import burnisher_amd as bh
    batch, n, heads, d = q.shape
    kv_len, kvh = k.shape[1], k.shape[2]
    dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    dl, ds = dev(lens), dev(starts)
    need = bh.lib().bh_attention_window_workspace_bytes(batch, heads, kvh, n, kv_len, d, left, right, sinks)
    assert need >= 0
    ws = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((batch, n, heads, d), 9.0, dtype=torch.bfloat16, device="cuda")
    # a view's stride over a length of one says nothing
    ld = lambda t: t.stride(1) if t.shape[1] != 1 else max(t.stride(0), t.shape[2] * d)  # noqa: E731
    bh.call("bh_attention_window", q.data_ptr(), ld(q), k.data_ptr(), v.data_ptr(), ld(k), out.data_ptr(), ld(out), batch,
            heads, kvh, n, kv_len, d, scale, left, right, sinks, bh.ptr(dl), bh.ptr(ds), BF16,
            ws.data_ptr() if workspace else None, need if workspace else 0, bh.stream_ptr(stream))
    torch.cuda.synchronize()
    return out


def check(batch, heads, kvh, n, kv_len, d, left, right, sinks, lens=None, starts=None, seed=0, **how):
    q, k, v = normal((batch, n, heads, d), seed), normal((batch, kv_len, kvh, d), seed + 1), \
        normal((batch, kv_len, kvh, d), seed + 2)
    got = run(q, k, v, lens, starts, left, right, sinks, **how)
    compare(got, q, k, v, lens, starts, left, right, sinks)
    return got


def compare(got, q, k, v, lens, starts, left, right, sinks, scale=None):
    batch, n, kv_len = q.shape[0], q.shape[1], k.shape[1]
    want, tol = plain(q, k, v, lens or [kv_len] * batch, starts or [kv_len - n] * batch, left, right, sinks, scale)
    bad = ~((got.double() - want).abs() <= tol)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {at}: {got[at]} for {want[at]}")


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (0, 0, 0), (5, 0, 2), (63, 0, 4), (64, 64, 0), (100, 3, 70), (7, -1, 3), (1000, 0, 1)]


@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("n,d,heads,kvh", [(1, 128, 8, 1), (3, 64, 4, 4), (65, 72, 2, 2), (200, 128, 8, 2), (333, 64, 3, 1)])
def test_self_attention_windows(hip, n, d, heads, kvh, left, right, sinks):
    check(2, heads, kvh, n, n, d, left, right, sinks, lens=[n, max(1, n // 3)], starts=[0, 0], seed=n)


# enough rows to fill the chip: tiles of 128 rows
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("batch,n,d,heads,kvh", [(4, 150, 64, 32, 32), (4, 200, 128, 32, 8), (3, 333, 72, 15, 15)])
def test_self_attention_windows_of_many_rows(hip, batch, n, d, heads, kvh, left, right, sinks):
    lens = [n, n // 3, 1, 0][:batch]
    check(batch, heads, kvh, n, n, d, left, right, sinks, lens=lens, starts=[0] * batch, seed=n)


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 64, 72, 80, 88, 96, 104, 112, 120, 128])
def test_head_dims_of_many_rows(hip, d):
    check(8, 16, 16, 70, 90, d, 20, 5, 3, lens=[90, 89, 70, 64, 33, 90, 90, 12], starts=[20, 0, 0, 10, 3, -5, 40, 0])


# few and many rows against few and many keys, at every width of the kernels' images
@pytest.mark.parametrize("d", [24, 64, 72, 88, 128])
@pytest.mark.parametrize("heads,kvh,n,kv_len,left,right,sinks", [
    (4, 4, 4, 1500, -1, 0, 0), (40, 8, 33, 300, 300, 300, 0), (40, 8, 70, 300, -1, 0, 0), (8, 8, 33, 1500, -1, 0, 0),
    (8, 8, 33, 5000, -1, -1, 0), (40, 8, 33, 3000, -1, 0, 0), (40, 8, 70, 300, 20, 0, 4), (40, 8, 150, 300, 200, 20, 0),
    (12, 4, 150, 300, 10, 0, 70)])
def test_row_tiles_and_splits(hip, d, heads, kvh, n, kv_len, left, right, sinks):
    lens = [kv_len, kv_len // 2, n]
    check(3, heads, kvh, n, kv_len, d, left, right, sinks, lens=lens, starts=[x - n for x in lens], seed=d)


@pytest.mark.parametrize("n,heads,kvh", [(130, 32, 32), (70, 64, 16)])
@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_unseen_keys_never_enter_many_rows(hip, n, heads, kvh, poison):
    check_poison(4, n, heads, kvh, poison)


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 64, 72, 80, 88, 96, 104, 112, 120, 128])
def test_head_dims(hip, d):
    check(1, 4, 2, 150, 150, d, 40, 0, 5)
    check(2, 4, 2, 1, 700, d, 300, 0, 5, lens=[700, 411], starts=[699, 410])


@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("heads,kvh", [(1, 1), (8, 1), (32, 8), (40, 2), (6, 6)])
def test_single_tokens_against_a_cache(hip, heads, kvh, left, right, sinks):
    lens = [1, 64, 65, 1000, 1500]
    check(5, heads, kvh, 1, 1500, 64, left, right, sinks, lens=lens, starts=[x - 1 for x in lens], seed=heads)


@pytest.mark.parametrize("n", [2, 7, 33, 130])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (50, 0, 3), (500, 0, 130), (20, 10, 0)])
def test_chunk_of_new_tokens(hip, n, left, right, sinks):
    lens = [n, 999, 1300]
    check(3, 8, 2, n, 1300, 128, left, right, sinks, lens=lens, starts=[x - n for x in lens], seed=n)


def test_long_keys_with_many_splits(hip):
    check(1, 8, 1, 1, 20000, 128, -1, 0, 0)
    check(2, 4, 2, 1, 20000, 64, 9000, 0, 100, lens=[20000, 12345], starts=[19999, 12344])
    check(1, 4, 4, 5, 9000, 72, -1, -1, 0)
    check(2, 8, 1, 1, 20000, 128, -1, 0, 0, lens=[20000, 3], starts=[19999, 2])


def test_the_default_positions_are_the_last_queries(hip):
    check(2, 4, 2, 40, 300, 64, 30, 0, 2)
    check(1, 4, 2, 300, 300, 64, 30, 0, 2)


def test_without_a_workspace(hip):
    check(2, 8, 1, 1, 5000, 128, -1, 0, 0, workspace=False)
    check(1, 4, 4, 100, 100, 64, 20, 0, 1, workspace=False)


@pytest.mark.parametrize("left,right,sinks", [(10, 0, 0), (10, 0, 4), (0, 0, 0), (-1, 0, 0), (3, 2, 0)])
def test_rows_that_see_nothing_are_zero(hip, left, right, sinks):
    import torch
    # no valid keys; queries far behind the last key; queries before the first one; a sequence of one
    lens, starts = [0, 5, 40, 1, -7], [0, 30, -60, 0, 0]
    got = check(5, 4, 2, 50, 50, 64, left, right, sinks, lens=lens, starts=starts)
    assert torch.equal(got[0], torch.zeros_like(got[0])) and torch.equal(got[4], torch.zeros_like(got[4]))
    check(5, 4, 2, 1, 5000, 64, left, right, sinks, lens=[0, 1, 4000, 5000, 3], starts=[0, 4999, 4500, -1, 2])


def test_no_keys_at_all(hip):
    import torch
    q = normal((2, 3, 4, 64), 1)
    k = torch.empty(2, 0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(run(q, k, k, None, None, -1, 0, 0), torch.zeros_like(q))


@pytest.mark.parametrize("n,heads", [(1, 8), (20, 2), (150, 2)])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_unseen_keys_never_enter(hip, n, heads, poison):
    check_poison(2, n, heads, 2, poison)


def check_poison(batch, n, heads, kvh, poison):
    import torch
    kv_len, left, sinks = 600, 90, 3
    q, k, v = normal((batch, n, heads, 64), 1), normal((batch, kv_len, kvh, 64), 2), normal((batch, kv_len, kvh, 64), 3)
    lens = [500, 211, 600, 333][:batch]
    starts = [x - n for x in lens]
    for b in range(batch):
        unseen = ~sees(torch.arange(n, device="cuda") + starts[b], lens[b], kv_len, left, 0, sinks).any(0)
        k[b, unseen], v[b, unseen] = poison, poison
    got = run(q, k, v, lens, starts, left, 0, sinks)
    compare(got, q, k, v, lens, starts, left, 0, sinks)


def test_strided_operands_and_untouched_gaps(hip):
    import torch
    # q, k and v in one projection of grouped heads, the output inside a wider buffer
    batch, n, heads, kvh, d = 2, 90, 6, 2, 72
    fused = normal((batch, n, (heads + 2 * kvh) * d + 8), 4)
    q = fused[:, :, :heads * d].unflatten(2, (heads, d))
    k = fused[:, :, heads * d:(heads + kvh) * d].unflatten(2, (kvh, d))
    v = fused[:, :, (heads + kvh) * d:(heads + 2 * kvh) * d].unflatten(2, (kvh, d))
    buf = torch.full((batch, n, heads * d + 12), 5.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, :, :heads * d].unflatten(2, (heads, d))
    run(q, k, v, None, None, 30, 0, 2, out=out)
    compare(out, q, k, v, None, None, 30, 0, 2)
    assert (buf[:, :, heads * d:] == 5.0).all()


def test_scale_and_large_scores(hip):
    q, k, v = normal((1, 70, 2, 64), 1), normal((1, 70, 2, 64), 2), normal((1, 70, 2, 64), 3)
    compare(run(q, k, v, None, None, 20, 20, 0, scale=0.3), q, k, v, None, None, 20, 20, 0, 0.3)
    big = (q.float() * 200).bfloat16()   # scores of thousands: the weights become one-hot
    compare(run(big, k, v, None, None, 20, 20, 0), big, k, v, None, None, 20, 20, 0)
    low = (q.float().abs() * -300).bfloat16()   # and all very negative
    kk = k.abs()
    compare(run(low, kk, v, None, None, 20, 0, 0), low, kk, v, None, None, 20, 0, 0)


def test_windows_beyond_any_length(hip):
    big = 2 ** 62
    check(1, 2, 2, 100, 100, 64, big, big, 0)
    check(1, 2, 2, 100, 100, 64, 10, 0, big)
    check(2, 2, 2, 10, 100, 64, 30, 0, 0, lens=[2 ** 31 - 1, 50], starts=[90, 2 ** 31 - 1])
    check(2, 2, 2, 10, 100, 64, 30, 50, 0, lens=[100, 50], starts=[-2 ** 31, 40])


def test_offsets_beyond_32_bits(hip):
    import torch
    # the second sequence's rows start 2^32 bytes in; k and v share the buffer
    kv_len, kvh, d = 2 ** 20, 16, 128
    cache = torch.empty(2, kv_len, kvh, d, dtype=torch.bfloat16, device="cuda")
    tail, left = 300, 200
    for b in range(2):
        cache[b, -tail:] = normal((tail, kvh, d), b)
        cache[b, :8] = normal((8, kvh, d), 5 + b)
    q = normal((2, 1, 32, d), 9)
    got = run(q, cache, cache, None, None, left, 0, 4)
    # the same keys in a short sequence: the four sinks before the window's tail
    short = torch.cat([cache[:, :4], cache[:, -left - 1:]], dim=1).contiguous()
    compare(got, q, short, short, None, None, -1, 0, 0)


def test_stays_inside_its_workspace_and_refuses_a_small_one(hip):
    import torch
    import burnisher_amd as bh
    batch, heads, kvh, kv_len, d = 1, 8, 2, 6000, 64
    q, k, v = normal((batch, 1, heads, d), 1), normal((batch, kv_len, kvh, d), 2), normal((batch, kv_len, kvh, d), 3)
    need = bh.lib().bh_attention_window_workspace_bytes(batch, heads, kvh, 1, kv_len, d, -1, 0, 0)
    assert need > 0
    out = torch.zeros_like(q)
    ws = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")

    def call(at, size):
        return bh.lib().bh_attention_window(q.data_ptr(), heads * d, k.data_ptr(), v.data_ptr(), kvh * d, out.data_ptr(),
                                            heads * d, batch, heads, kvh, 1, kv_len, d, 0.0, -1, 0, 0, None, None, BF16,
                                            at, size, bh.stream_ptr())

    assert call(ws.data_ptr(), need - 1) != 0 and b"this call needs" in bh.lib().bh_last_error()
    assert call(ws.data_ptr() + 4, need) != 0 and b"16-byte" in bh.lib().bh_last_error()
    torch.cuda.synchronize()
    assert not out.any() and (ws == 0x5a).all(), "a refused call wrote"
    assert call(ws.data_ptr(), need) == 0
    assert (ws[need:] == 0x5a).all(), "written past the workspace"
    assert torch.equal(out, run(q, k, v, None, None, -1, 0, 0))


def test_in_a_graph_and_on_two_streams(hip):
    import torch
    import burnisher_amd as bh
    batch, heads, kvh, n, kv_len, d = 2, 8, 1, 1, 6000, 128
    sets = [[normal((batch, n, heads, d), s), normal((batch, kv_len, kvh, d), s + 1), normal((batch, kv_len, kvh, d), s + 2)]
            for s in (1, 11)]
    lens = torch.tensor([6000, 4321], dtype=torch.int32, device="cuda")
    starts = lens - 1
    need = max(16, bh.lib().bh_attention_window_workspace_bytes(batch, heads, kvh, n, kv_len, d, -1, 0, 0))
    out = [torch.zeros_like(s[0]) for s in sets]
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in sets]

    def call(i, stream):
        q, k, v = sets[i]
        bh.call("bh_attention_window", q.data_ptr(), heads * d, k.data_ptr(), v.data_ptr(), kvh * d, out[i].data_ptr(),
                heads * d, batch, heads, kvh, n, kv_len, d, 0.0, -1, 0, 0, lens.data_ptr(), starts.data_ptr(), BF16,
                ws[i].data_ptr(), need, bh.stream_ptr(stream))

    want = [run(*s, [6000, 4321], [5999, 4320], -1, 0, 0) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for i in (0, 1):
            call(i, streams[i])
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0, torch.cuda.current_stream())
    for seed, new_lens in ((5, [6000, 1]), (6, [77, 0]), (7, [3000, 5999])):
        for t, s in zip(sets[0], range(3)):
            t.copy_(normal(tuple(t.shape), seed + s))
        lens.copy_(torch.tensor(new_lens, dtype=torch.int32))
        starts.copy_(lens - 1)
        out[0].fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        got = run(*sets[0], new_lens, [x - 1 for x in new_lens], -1, 0, 0)
        assert torch.equal(out[0], got), "a replay differs from the call"


def test_a_layer_in_8_bits_prompt_then_token(hip):
    """Projection, window attention and output projection as a text model runs them: a prompt into a cache,
    then one token. The token's output equals, within the roundings, the last row of one call over
    prompt and token together."""
    import torch
    import burnisher_amd as bh
    from test_gpu_fp8 import quantize, run_gemm
    batch, n, heads, kvh, d, width, left, sinks = 2, 70, 8, 2, 64, 512, 40, 4
    w_qkv, w_out = normal(((heads + 2 * kvh) * d, width), 1) * 0.04, normal((width, heads * d), 2) * 0.04
    qkv_w, out_w = quantize(w_qkv, 128), quantize(w_out, 128)

    def project(x, w, k):
        qx = quantize(x.reshape(-1, k), 1)
        return run_gemm(*qx, *w, None, k).view(*x.shape[:-1], -1)

    def split(fused):
        q, k, v = fused.split([heads * d, kvh * d, kvh * d], dim=2)
        return q.unflatten(2, (heads, d)), k.unflatten(2, (kvh, d)), v.unflatten(2, (kvh, d))

    x = normal((batch, n + 1, width), 3)
    q, k, v = split(project(x, qkv_w, width))
    whole = run(q, k, v, None, None, left, 0, sinks)
    full = project(whole.flatten(2), out_w, heads * d)
    compare(whole, q, k, v, None, None, left, 0, sinks)

    cache = torch.full((2, batch, 128, kvh, d), math.nan, dtype=torch.bfloat16, device="cuda")
    q, k, v = split(project(x[:, :n], qkv_w, width))
    cache[0, :, :n], cache[1, :, :n] = k, v
    prompt = run(q, cache[0], cache[1], [n] * batch, [0] * batch, left, 0, sinks)
    q, k, v = split(project(x[:, n:], qkv_w, width))
    cache[0, :, n:n + 1], cache[1, :, n:n + 1] = k, v
    token = run(q, cache[0], cache[1], [n + 1] * batch, [n] * batch, left, 0, sinks)
    compare(token, q, cache[0], cache[1], [n + 1] * batch, [n] * batch, left, 0, sinks)
    # two correct results of the same values: twice the weights' and the output's roundings, 4 * 2^-8 of the
    # largest value that is averaged
    top = cache[1, :, :n + 1].float().abs().max()
    assert (token[:, 0].float() - whole[:, n].float()).abs().max() <= 4 * 2.0 ** -8 * top
    assert (prompt.float() - whole[:, :n].float()).abs().max() <= 4 * 2.0 ** -8 * top
    last = project(token.flatten(2), out_w, heads * d)
    assert torch.isfinite(full).all() and torch.isfinite(last).all()
    bh.check(0)
