"""Every form of windowed attention at every head_dim: tiles of 16, 32 and 128 rows, a tile's keys whole and split over
workgroups. Which form a call takes is chosen by an estimate, so each case asserts the one that it is there for (on 256
compute units).

V marks its keys: column c of a value is 1 where its key is one of the groups of `step` keys numbered c modulo head_dim, so
an output is the weight of few keys, and a group that is left out, read twice or masked wrongly shows in its column."""
import ctypes

import pytest

from test_gpu_window import compare, normal, plain, run, sees

pytestmark = pytest.mark.gpu

HEAD_DIMS = list(range(8, 129, 8))


def marks(batch, kv_len, kvh, d, step):
    import torch
    at = torch.arange(kv_len, device="cuda") // step % d
    v = (at[:, None] == torch.arange(d, device="cuda")).to(torch.bfloat16)
    return v[None, :, None, :].expand(batch, kv_len, kvh, d).contiguous()


def check(form, batch, heads, kvh, n, kv_len, d, left, right, sinks, lens=None, starts=None, step=32):
    import burnisher_amd as bh
    plan = bh.AttentionWindowPlan()
    bh.call("bh_attention_window_describe", batch, heads, kvh, n, kv_len, d, left, right, sinks, 1, 0, ctypes.byref(plan))
    assert (plan.tile_rows, plan.splits > 1) == form, "this call has another form now: it needs another size"
    q, k, v = normal((batch, n, heads, d), d), normal((batch, kv_len, kvh, d), d + 1), normal((batch, kv_len, kvh, d), d + 2)
    compare(run(q, k, v, lens, starts, left, right, sinks), q, k, v, lens, starts, left, right, sinks)
    v = marks(batch, kv_len, kvh, d, step)
    compare(run(q, k, v, lens, starts, left, right, sinks), q, k, v, lens, starts, left, right, sinks)


@pytest.mark.parametrize("d", HEAD_DIMS)
@pytest.mark.parametrize("left,right,sinks,kvh", [(20, 5, 3, 16), (200, 90, 70, 16), (70, 0, 70, 4), (-1, -1, 0, 8), (64, 63, 0, 16)])
def test_tiles_of_128_rows(hip, d, left, right, sinks, kvh):
    check((128, False), 8, 16, kvh, 200, 240, d, left, right, sinks, lens=[240, 239, 200, 64, 33, 240, 0, 12],
          starts=[40, 0, 0, 10, 3, -5, 40, 0], step=4)


@pytest.mark.parametrize("d", HEAD_DIMS)
@pytest.mark.parametrize("left,right,sinks", [(300, 0, 5), (-1, 0, 0), (300, 30, 300)])
def test_tiles_of_16_rows(hip, d, left, right, sinks):
    check((16, False), 8, 16, 16, 8, 1000, d, left, right, sinks, lens=[1000, 999, 8, 500, 33, 1000, 0, 12],
          starts=[992, 991, 0, 10, 3, -5, 40, 900], step=8)


@pytest.mark.parametrize("d", HEAD_DIMS)
@pytest.mark.parametrize("left,right,sinks", [(2500, 0, 5), (2500, 30, 100)])
def test_tiles_of_32_rows(hip, d, left, right, sinks):
    if d <= 64:
        check((32, False), 2, 16, 16, 600, 3000, d, left, right, sinks, lens=[3000, 2222], starts=[2400, 1622])
    else:
        check((32, False), 4, 32, 8, 64, 4096, d, left, right, sinks, lens=[4096, 3001, 64, 1], starts=[4032, 2937, 0, 3])


@pytest.mark.parametrize("d", HEAD_DIMS)
@pytest.mark.parametrize("left,right,sinks", [(2000, 0, 5), (-1, 0, 0), (-1, -1, 0), (1800, 30, 130)])
def test_split_keys_of_16_rows(hip, d, left, right, sinks):
    check((16, True), 4, 8, 2, 1, 20000, d, left, right, sinks, lens=[20000, 12345, 3, 2001], starts=[19999, 12344, 2, 2500])


@pytest.mark.parametrize("d", HEAD_DIMS)
def test_split_keys_of_32_rows(hip, d):
    check((32, True), 3, 8, 2, 167, 7675, d, -1, 0, 70, lens=[7675, 5000, 40], starts=[7508, 4833, -100])


@pytest.mark.parametrize("kv_len,left,sinks", [(20000, -1, 0), (20000, 9000, 100), (8192, 4095, 4)])
def test_a_piece_of_keys_that_is_left_out_exceeds_the_tolerance(hip, kv_len, left, sinks):
    # the check itself: the 64-bit result without any one piece of 32 keys of the window is further from the whole one
    # than an output may be
    import torch
    d = 128
    q, k = normal((1, 1, 1, d), 1), normal((1, kv_len, 1, d), 2)
    v = marks(1, kv_len, 1, d, 32)
    want, tol = plain(q, k, v, [kv_len], [kv_len - 1], left, 0, sinks)
    seen = sees(torch.tensor([kv_len - 1], device="cuda"), kv_len, kv_len, left, 0, sinks)[0]
    w = torch.softmax(torch.where(seen, (k[0, :, 0].double() @ q[0, 0, 0].double()) / d ** 0.5, -float("inf")), 0)
    first = max(0, kv_len - 1 - left) if left >= 0 else 0
    for at in range(first, kv_len - 32, 32):
        rest = w.clone()
        rest[at:at + 32] = 0
        off = (rest / rest.sum()) @ v[0, :, 0].double() - want[0, 0, 0]
        assert (off.abs() > tol[0, 0, 0]).any(), at
