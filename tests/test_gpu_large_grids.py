"""Calls of more workgroups than one axis of a launch holds: 2^32 threads, so 2^24 workgroups of 256 or 2^23 of 512.
The operands repeat a small piece, whose results a small call gives; that one is checked elsewhere."""
import pytest

from helpers import BF16
from test_gpu_fp8 import normal, quantize, quantize_plain, run_gemm, same_bits
from test_operator_plans import product, window

pytestmark = pytest.mark.gpu


def test_quantize_rows(hip):
    import torch
    rows, times = 4096, 2 ** 16 + 1
    assert rows * times // 16 > 2 ** 24
    piece = normal((rows, 16), 1, torch.bfloat16)
    codes, scales = quantize(piece.repeat(times, 1), 1, guard=64)
    want = quantize_plain(piece, 1)
    assert same_bits(codes[:rows], want[0])
    codes = codes.view(torch.uint8).view(times, rows * 16)
    assert (codes == codes[0]).all()
    assert (scales.view(times, rows) == want[1]).all()


def test_product_of_one_row(hip):
    import torch
    n, times, k = 16384, 2 ** 13 + 1, 16
    assert product(1, n * times, k).workgroups * 512 >= 2 ** 32
    a, sa = quantize_plain(normal((1, k), 1, torch.float32), 1)
    b, sb = quantize_plain(normal((n, k), 2, torch.float32, 0.02), 128)
    want = run_gemm(a, sa, b, sb, None, k)
    got = run_gemm(a, sa, b.view(torch.uint8).repeat(times, 1), sb.repeat(times, 1), None, k)
    assert (got.view(times, n) == want).all() and torch.equal(got[:, -n:], want)


@pytest.mark.parametrize("q_len,tile_rows", [(1, 16), (17, 32), (33, 128)])
def test_window_attention(hip, q_len, tile_rows):
    import torch
    import burnisher_amd as bh
    batch, times, heads, kv_len, d = 8, 2 ** 17 + 1, 16, 5, 8
    plan = window(batch * times, heads, heads, q_len, kv_len, d, -1, 0, 0)
    assert plan.tile_rows == tile_rows and plan.workgroups > 2 ** 24
    q, k, v = normal((batch, q_len, heads, d), 1, torch.bfloat16), *(normal((batch, kv_len, heads, d), s, torch.bfloat16) for s in (2, 3))

    def call(q, k, v):
        out = torch.full((q.numel() + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
        bh.call("bh_attention_window", q.data_ptr(), heads * d, k.data_ptr(), v.data_ptr(), heads * d, out.data_ptr(), heads * d,
                q.shape[0], heads, heads, q_len, kv_len, d, 0.0, -1, 0, 0, None, None, BF16, None, 0, bh.stream_ptr())
        assert (out[-64:] == 9.0).all(), "written past the end"
        return out[:-64]

    want = call(q, k, v)
    got = call(*(t.repeat(times, 1, 1, 1) for t in (q, k, v)))
    got = got.view(times, want.numel())
    for i in range(0, times, 8192):
        assert (got[i:i + 8192] == want).all()
