"""What the 8-bit operators and windowed attention refuse, before any device work (no GPU here)."""
import pytest

import burnisher_amd as bh

D = 1 << 20   # an address that no check dereferences: every call below is refused before it is used


def refused(name, *args):
    status = getattr(bh.lib(), name)(*args)
    assert status != 0, f"{name}{args} was accepted"
    return bh.lib().bh_last_error().decode()


@pytest.fixture(autouse=True)
def no_pointer_lookups():
    """Operand addresses are not looked up, so the checks after that one are reached without a device."""
    bh.lib().bh_set_operand_checks(0)
    yield
    bh.lib().bh_set_operand_checks(1)


def quantize(**over):
    a = dict(x=D, ld=256, q=D, scales=D, rows=4, cols=256, block_rows=1, dtype=bh.BF16)
    a.update(over)
    return refused("bh_quantize_fp8", a["x"], a["ld"], a["q"], a["scales"], a["rows"], a["cols"], a["block_rows"],
                   a["dtype"], None)


@pytest.mark.parametrize("over,says", [
    (dict(x=None), "x is null"), (dict(q=None), "q is null"), (dict(scales=None), "scales is null"),
    (dict(rows=-1), "rows is negative"), (dict(cols=-1), "cols is negative"), (dict(block_rows=64), "1 or 128"),
    (dict(block_rows=0), "1 or 128"), (dict(ld=255), "below cols"), (dict(dtype=7), "dtype 7"),
    (dict(q=D + 4), "8-byte"), (dict(x=D + 1), "aligned to its type"), (dict(scales=D + 2), "aligned to its type"),
    (dict(rows=1 << 30), "2^30"), (dict(cols=1 << 30, ld=1 << 30), "2^30")])
def test_quantize_refuses(over, says):
    assert says in quantize(**over)


def gemm(**over):
    a = dict(a=D, sa=D, b=D, sb=D, bias=None, out=D, m=600, n=512, k=8192, epi=0, dtype=bh.BF16, ws=None, bytes=0)
    a.update(over)
    return refused("bh_gemm_fp8", a["a"], a["sa"], a["b"], a["sb"], a["bias"], a["out"], a["m"], a["n"], a["k"], a["epi"],
                   a["dtype"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("over,says", [
    (dict(a=None), "a is null"), (dict(sa=None), "a_scales is null"), (dict(b=None), "b is null"),
    (dict(sb=None), "b_scales is null"), (dict(out=None), "out is null"), (dict(m=-1), "m is negative"),
    (dict(n=-2), "n is negative"), (dict(k=-3), "k is negative"), (dict(epi=3), "GeluGated"), (dict(epi=4), "epilogue"),
    (dict(epi=-1), "epilogue"), (dict(dtype=2), "dtype 2"), (dict(a=D + 8), "16-byte"), (dict(b=D + 8), "16-byte"),
    (dict(out=D + 1), "aligned to its type"), (dict(bias=D + 1), "aligned to its type"), (dict(sa=D + 2), "aligned to"),
    (dict(k=1 << 30), "2^30"), (dict(m=1 << 30), "2^30")])
def test_gemm_refuses(over, says):
    assert says in gemm(**over)


def window(**over):
    a = dict(q=D, ld_q=512, k=D, v=D, ld_kv=128, out=D, ld_o=512, batch=1, heads=8, kvh=2, q_len=1, kv_len=20000, d=64,
             scale=0.0, left=-1, right=0, sinks=0, lens=None, starts=None, dtype=bh.BF16, ws=None, bytes=0)
    a.update(over)
    return refused("bh_attention_window", a["q"], a["ld_q"], a["k"], a["v"], a["ld_kv"], a["out"], a["ld_o"], a["batch"],
                   a["heads"], a["kvh"], a["q_len"], a["kv_len"], a["d"], a["scale"], a["left"], a["right"], a["sinks"],
                   a["lens"], a["starts"], a["dtype"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("over,says", [
    (dict(q=None), "q is null"), (dict(k=None), "k is null"), (dict(v=None), "v is null"), (dict(out=None), "out is null"),
    (dict(dtype=bh.F32), "bf16 only"), (dict(dtype=9), "dtype 9"), (dict(heads=9, ld_q=576, ld_o=576), "multiple of kv_heads"),
    (dict(kvh=0), "multiple of kv_heads"), (dict(kvh=-2), "multiple of kv_heads"), (dict(d=60), "multiple of 8"),
    (dict(d=136, ld_q=1088, ld_o=1088, ld_kv=272), "up to 128"), (dict(d=0), "multiple of 8"), (dict(ld_q=504), "row stride"),
    (dict(ld_kv=120), "row stride"), (dict(ld_o=508), "row stride"), (dict(ld_q=516), "multiples of 8"),
    (dict(ld_kv=132), "multiples of 8"), (dict(ld_o=514), "multiples of 8"), (dict(q=D + 8), "16-byte"),
    (dict(k=D + 8), "16-byte"), (dict(v=D + 2), "16-byte"), (dict(out=D + 4), "8-byte"), (dict(lens=D + 2), "aligned to"),
    (dict(starts=D + 1), "aligned to"), (dict(sinks=-1), "sinks is negative"), (dict(q_len=-1), "q_len is negative"),
    (dict(kv_len=-1), "kv_len is negative"), (dict(batch=-1), "batch is negative"), (dict(kv_len=1 << 30), "2^30"),
    (dict(q_len=1 << 29), "2^30"), (dict(ld_kv=1 << 24), "2^24")])
def test_window_refuses(over, says):
    assert says in window(**over)


def test_workspace_queries_refuse_and_answer():
    lib = bh.lib()
    assert lib.bh_gemm_fp8_workspace_bytes(-1, 4, 4) == -1 and b"negative" in lib.bh_last_error()
    assert lib.bh_attention_window_workspace_bytes(1, 8, 3, 1, 64, 64, -1, 0, 0) == -1
    assert lib.bh_attention_window_workspace_bytes(1 << 24, 1 << 24, 1 << 24, 1, 64, 64, -1, 0, 0) == -1
    assert b"batch * heads" in lib.bh_last_error()
    assert lib.bh_gemm_fp8_workspace_bytes(0, 4, 4) == 0 and lib.bh_last_error() == b""
    assert lib.bh_attention_window_workspace_bytes(0, 8, 2, 1, 64, 64, -1, 0, 0) == 0


def test_empty_calls_are_no_ops():
    lib = bh.lib()
    assert lib.bh_quantize_fp8(None, 0, None, None, 0, 0, 1, bh.BF16, None) == 0
    assert lib.bh_gemm_fp8(None, None, None, None, None, None, 0, 4, 4, 0, bh.BF16, None, 0, None) == 0
    assert lib.bh_attention_window(None, 512, None, None, 128, None, 512, 0, 8, 2, 1, 4, 64, 0.0, -1, 0, 0, None, None,
                                   bh.BF16, None, 0, None) == 0


def test_quantize_refuses_more_workgroups_than_it_numbers():
    assert "too large" in quantize(rows=(1 << 30) - 1, cols=1 << 20, ld=1 << 20)
