"""bh_rope, bh_attention_linear and bh_residual_norms_run in calls of more workgroups than one axis of a launch holds
(2^32 threads). The operands repeat a small piece, whose results a small call gives; that one is checked elsewhere."""
import ctypes

import pytest

import burnisher_amd as bh
from test_gpu_linear import call, decays, normal
from test_gpu_rope import grid, run as rope

pytestmark = pytest.mark.gpu


def test_rope_of_many_rows(hip):
    import torch
    piece, times = 1 << 14, (1 << 14) + 1
    rows = piece * times
    assert rows // 16 > 2 ** 24
    axes, positions = bh.RopeAxes.of([1]), grid(piece, 1, 1)
    x = normal((piece, 1, 2), 2)
    want = torch.empty_like(x)
    rope(axes, positions, x, None, want, None)
    out = torch.full((rows * 2 + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
    rope(axes, positions, x.repeat(times, 1, 1), None, out[:-64].view(rows, 1, 2), None)
    assert (out[-64:] == 9.0).all(), "written past the end"
    assert (out[:-64].view(times, piece * 2) == want.view(-1)).all()


@pytest.mark.parametrize("n", [1, 3])
def test_linear_attention_of_many_heads(hip, n):
    import torch
    batch, times, heads, d = 32, 2 ** 12 + 1, 128, 8
    assert batch * times * heads > 2 ** 24
    q, k, v = (normal((batch, n, heads, d), s) for s in (1, 2, 3))
    rate, want = decays(heads), torch.empty(batch, n, heads, d, dtype=torch.bfloat16, device="cuda")
    call(q, k, v, want, rate, None, None, None, 0.0, None, 0)
    out = torch.full((batch * times * n * heads * d + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
    call(*(t.repeat(times, 1, 1, 1) for t in (q, k, v)), out[:-64].view(batch * times, n, heads, d), rate, None, None, None, 0.0, None, 0)
    assert (out[-64:] == 9.0).all(), "written past the end"
    got = out[:-64].view(times, want.numel())
    for i in range(0, times, 1024):
        assert (got[i:i + 1024] == want.view(-1)).all()


def test_norms_of_many_rows(hip):
    import torch
    piece, times, cols = 4096, 2 ** 14 + 1, 3
    rows = piece * times
    assert rows // 4 > 2 ** 24
    x, r = normal((piece, cols), 1), normal((piece, cols), 2)
    plan = bh.ResidualNorms(post_norm=bh.NORM_RMS, post_eps=1e-6, branch_scale=1.0, residual_scale=1.0, pre_norm=bh.NORM_LAYER, pre_eps=1e-6)

    def run(x, r, res, out):
        bh.call("bh_residual_norms_run", x.data_ptr(), cols, r.data_ptr(), cols, res.data_ptr(), cols, out.data_ptr(), cols, x.shape[0], cols,
                ctypes.byref(plan), bh.BF16, bh.BF16, bh.stream_ptr())

    want = [torch.empty_like(x) for _ in range(2)]
    run(x, r, *want)
    got = [torch.full((rows * cols + 64,), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    run(x.repeat(times, 1), r.repeat(times, 1), *got)
    for g, w in zip(got, want):
        assert (g[-64:] == 9.0).all(), "written past the end"
        assert (g[:-64].view(times, piece * cols) == w.view(-1)).all()


# 2^26 tokens of 32 8-byte pieces: from there on a count of pieces behind the sequence passes 31 bits
@pytest.mark.parametrize("n", [2 ** 26, 2 ** 26 + 1, 2 ** 26 + 32])
def test_linear_attention_of_a_token_before_long_padding(hip, n):
    import torch
    d, e = 8, 128
    plan = bh.AttentionLinearPlan()
    bh.call("bh_attention_linear_describe", 1, 1, 1, n, d, e, 0, 0, ctypes.byref(plan))
    assert (plan.chunk, plan.segments) == (32, 1)
    rate, lens = decays(1), torch.tensor([1], dtype=torch.int32, device="cuda")
    first = [normal((1, 40, 1, w), s) for s, w in ((1, d), (2, d), (3, e))]
    want, new, new_want = torch.zeros(1, 40, 1, e, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, d, e, device="cuda"), torch.zeros(1, 1, d, e, device="cuda")
    call(*first, want, rate, lens, None, new_want, 0.0, None, 0)
    long = [torch.empty(1, n, 1, w, dtype=torch.bfloat16, device="cuda") for w in (d, d, e)]
    for t, x in zip(long, first):
        t[:, :1] = x[:, :1]
    # 4096 bytes before and behind the output stay as they are
    buffer = torch.full((n * e + 4096,), 9.0, dtype=torch.bfloat16, device="cuda")
    out = buffer[2048:-2048].view(1, n, 1, e)
    call(*long, out, rate, lens, None, new, 0.0, None, 0)
    torch.cuda.synchronize()
    assert want[0, 0].any() and torch.equal(out[0, 0], want[0, 0]) and torch.equal(new, new_want)
    for i in range(1, n, 2 ** 22):
        assert not out[0, i:i + 2 ** 22].any(), f"rows from {i} on are not zeros"
    assert (buffer[:2048] == 9.0).all() and (buffer[-2048:] == 9.0).all()
