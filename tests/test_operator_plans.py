"""How the 8-bit products and windowed attention choose their kernels (no GPU here: the number of compute
units is an argument)."""
import ctypes
import random

import pytest

import burnisher_amd as bh


def product(m, n, k, dtype=bh.BF16, workspace=1, cus=256):
    plan = bh.GemmFp8Plan()
    bh.call("bh_gemm_fp8_describe", m, n, k, dtype, workspace, cus, ctypes.byref(plan))
    return plan


def window(batch, heads, kvh, n, kv_len, d, left, right, sinks, workspace=1, cus=256):
    plan = bh.AttentionWindowPlan()
    bh.call("bh_attention_window_describe", batch, heads, kvh, n, kv_len, d, left, right, sinks, workspace, cus,
            ctypes.byref(plan))
    return plan


@pytest.mark.parametrize("cus", [1, 5, 20, 60, 64, 104, 256, 304])
def test_a_slices_tiles_take_no_more_rounds_than_its_share_of_the_device_needs(cus):
    rng = random.Random(cus)
    sliced = walked = 0
    for _ in range(4000):
        m, n, k = (int(2 ** rng.uniform(*r)) for r in ((4.1, 13), (4, 14), (4, 13.5)))
        p = product(m, n, k, rng.choice([bh.BF16, bh.F32]), cus=cus)
        if not p.in_lds:
            continue
        share = max(1, cus // p.slices)   # workgroups of a slice that run at once
        assert 1 <= p.workgroups <= min(p.tiles, share), (m, n, k)
        assert -(-p.tiles // p.workgroups) == -(-p.tiles // share), (m, n, k, p.tiles, p.workgroups, share)
        sliced += p.slices > 1
        walked += p.tiles > p.workgroups
    assert sliced > 100 and walked > 100


@pytest.mark.parametrize("m,n,k", [(1104, 1120, 7736), (506, 1102, 4814), (829, 1791, 7442)])
def test_sliced_products_of_as_many_tiles_as_run_at_once(m, n, k):
    p = product(m, n, k)
    share = 256 // p.slices
    assert p.slices > 1 and share & ~7 < p.tiles <= share and p.workgroups == p.tiles


def test_whole_products_keep_a_workgroups_tiles_on_one_xcd():
    p = product(8192, 4608, 1152)
    assert (p.slices, p.workgroups) == (1, 256) and p.tiles > 256
    p = product(8192, 4608, 1152, cus=100)
    assert p.workgroups % 8 == 0 or -(-p.tiles // 96) > -(-p.tiles // 100)


def test_describe_answers_for_empty_calls_and_refuses():
    lib = bh.lib()
    p = product(0, 5, 5)
    assert (p.in_lds, p.tile_rows, p.slices, p.tiles, p.workgroups) == (0, 0, 0, 0, 0)
    w = window(0, 8, 2, 1, 64, 64, -1, 0, 0)
    assert (w.tile_rows, w.splits, w.workgroups) == (0, 0, 0)
    out = bh.GemmFp8Plan()
    assert lib.bh_gemm_fp8_describe(-1, 4, 4, bh.BF16, 1, 256, ctypes.byref(out)) != 0 and b"m is negative" in lib.bh_last_error()
    assert lib.bh_gemm_fp8_describe(4, 4, 1 << 30, bh.BF16, 1, 256, ctypes.byref(out)) != 0 and b"2^30" in lib.bh_last_error()
    assert lib.bh_gemm_fp8_describe(4, 4, 4, 7, 1, 256, ctypes.byref(out)) != 0 and b"dtype" in lib.bh_last_error()
    assert lib.bh_gemm_fp8_describe(4, 4, 4, bh.BF16, 1, -1, ctypes.byref(out)) != 0 and b"cus" in lib.bh_last_error()
    assert lib.bh_gemm_fp8_describe(4, 4, 4, bh.BF16, 1, 256, None) != 0 and b"null" in lib.bh_last_error()
    out = bh.AttentionWindowPlan()
    args = [1, 8, 2, 1, 64, 64, -1, 0, 0, 1]
    assert lib.bh_attention_window_describe(*args, -1, ctypes.byref(out)) != 0 and b"cus" in lib.bh_last_error()
    assert lib.bh_attention_window_describe(*args, 256, None) != 0 and b"null" in lib.bh_last_error()
    args[2] = 3
    assert lib.bh_attention_window_describe(*args, 256, ctypes.byref(out)) != 0 and b"kv_heads" in lib.bh_last_error()


def test_a_workspace_is_what_splitting_needs():
    for m, n, k in ((600, 4096, 10240), (17, 300, 5000), (8192, 4608, 1152)):
        assert product(m, n, k, workspace=0).slices == 1
    assert product(600, 4096, 10240).slices > 1
    assert window(16, 32, 8, 1, 8192, 128, 4095, 0, 4, workspace=0).splits == 1
    assert window(16, 32, 8, 1, 8192, 128, 4095, 0, 4).splits > 1
