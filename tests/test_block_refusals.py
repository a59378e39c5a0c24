"""What bh_rope, bh_attention_linear and bh_residual_norms_run refuse, before any device work (no GPU here)."""
import ctypes
import math

import pytest

import burnisher_amd as bh
from test_operator_refusals import no_pointer_lookups, refused  # noqa: F401

D = 1 << 20   # an address that no check dereferences: every call below is refused before it is used


def rope(axes=None, **over):
    a = dict(positions=D, position_rows=4, q=D, ld_q=512, q_out=D, ld_q_out=512, q_heads=8, k=D, ld_k=128, k_out=D, ld_k_out=128,
             k_heads=2, rows=4, head_dim=64, inverse=0, dtype=bh.BF16)
    a.update(over)
    axes = bh.RopeAxes.of([32]) if axes is None else axes
    return refused("bh_rope", ctypes.byref(axes) if axes else None, *a.values(), None)


def axes_with(**over):
    a = bh.RopeAxes.of([8, 8])
    for name, v in over.items():
        if name == "pairs":
            a.pairs = (ctypes.c_int * 4)(*v)
        elif name == "scale":
            a.scale = (ctypes.c_double * 4)(*v)
        else:
            setattr(a, name, v)
    return a


@pytest.mark.parametrize("over,says", [
    (dict(positions=None), "positions is null"), (dict(q=None), "q is null"), (dict(q_out=None), "q_out is null"),
    (dict(k=None), "k is null"), (dict(k_out=None), "k_out is null"), (dict(rows=-1), "rows is negative"),
    (dict(q_heads=-1), "q_heads is negative"), (dict(k_heads=-1), "k_heads is negative"), (dict(head_dim=62), "head_dim"),
    (dict(head_dim=1025, ld_q=8200, ld_k=2050, ld_q_out=8200, ld_k_out=2050), "head_dim"), (dict(ld_q=511), "row stride"),
    (dict(ld_q_out=511), "row stride"), (dict(ld_k=127), "row stride"), (dict(ld_k_out=127), "row stride"), (dict(dtype=2), "dtype 2"),
    (dict(position_rows=0), "position_rows"), (dict(positions=D + 2), "aligned to its type"), (dict(q=D + 1), "aligned to its type"),
    (dict(k_out=D + 2, dtype=bh.F32), "aligned to its type"), (dict(rows=1 << 40), "2^40"), (dict(q_heads=65536, ld_q=1 << 22, ld_q_out=1 << 22), "2^16"),
    (dict(ld_q_out=520), "another stride"), (dict(ld_k=136), "another stride")])
def test_rope_refuses(over, says):
    assert says in rope(**over)


@pytest.mark.parametrize("over,says", [
    (dict(axes=0), "1 to 4 axes"), (dict(axes=5), "1 to 4 axes"), (dict(pairs=[0, 0, 5, 5]), "1 to 128 pairs"),
    (dict(pairs=[8, -1, 0, 0]), "negative number"), (dict(pairs=[100, 29, 0, 0]), "1 to 128 pairs"), (dict(theta=0.0), "theta"),
    (dict(theta=-3.0), "theta"), (dict(theta=math.nan), "theta"), (dict(theta=math.inf), "theta"),
    (dict(scale=[1.0, math.nan, 1.0, 1.0]), "scale"), (dict(scale=[math.inf, 1.0, 1.0, 1.0]), "scale")])
def test_rope_refuses_axes(over, says):
    assert says in rope(axes_with(**over))


# scale times frequency, or that times the farthest position, is no finite number in 64 bits
@pytest.mark.parametrize("over", [
    dict(theta=1e-300, scale=[1e100, 1.0, 1.0, 1.0]), dict(theta=1e-300, scale=[1.0, 1e100, 1.0, 1.0]), dict(scale=[1.0, 1.5e300, 1.0, 1.0]),
    dict(scale=[-1.7e308, 1.0, 1.0, 1.0]), dict(theta=5e-324, scale=[1.0, 1e60, 1.0, 1.0], joint=1)])
def test_rope_refuses_angles_without_a_value(over):
    assert "range of fp64" in rope(axes_with(**over))


def test_rope_refuses_no_axes():
    assert "axes is null" in rope(False)
    for pairs, scale in (([], ()), ([1] * 5, ()), ([1], (1.0, 1.0))):
        with pytest.raises(bh.BurnisherError, match="1 to 4 axes"):
            bh.RopeAxes.of(pairs, scale=scale)


def linear(**over):
    a = dict(q=D, ld_q=512, k=D, ld_k=128, v=D, ld_v=144, out=D, ld_o=576, batch=1, heads=8, kvh=2, n=5, d=64, e=72, scale=0.0, decay=D,
             lens=None, state_in=None, state_out=None, dtype=bh.BF16, ws=None, bytes=0)
    a.update(over)
    return refused("bh_attention_linear", *a.values(), None)


@pytest.mark.parametrize("over,says", [
    (dict(q=None), "q is null"), (dict(k=None), "k is null"), (dict(v=None), "v is null"), (dict(out=None), "out is null"),
    (dict(decay=None), "log_decay is null"), (dict(dtype=bh.F32), "bf16 only"), (dict(dtype=9), "dtype 9"),
    (dict(heads=9, ld_q=576, ld_o=648), "multiple of kv_heads"), (dict(kvh=0), "multiple of kv_heads"), (dict(kvh=-2), "multiple of kv_heads"),
    (dict(d=60), "multiples of 8"), (dict(d=136, ld_q=1088, ld_k=272), "up to 128"), (dict(d=0), "multiples of 8"), (dict(e=4), "multiples of 8"),
    (dict(e=136, ld_v=272, ld_o=1088), "up to 128"), (dict(ld_q=504), "row stride"), (dict(ld_k=120), "row stride"), (dict(ld_v=136), "row stride"),
    (dict(ld_o=572), "row stride"), (dict(ld_q=516), "multiples of 8"), (dict(ld_k=132), "multiples of 8"), (dict(ld_v=148), "multiples of 8"),
    (dict(ld_o=578), "multiples of 8"), (dict(q=D + 8), "16-byte"), (dict(k=D + 8), "16-byte"), (dict(v=D + 2), "16-byte"), (dict(out=D + 4), "8-byte"),
    (dict(state_in=D + 8), "state is not 16-byte"), (dict(state_out=D + 4), "state is not 16-byte"), (dict(lens=D + 2), "aligned to"),
    (dict(decay=D + 1), "aligned to"), (dict(n=-1), "seq_len is negative"), (dict(batch=-1), "batch is negative"), (dict(heads=-8), "heads is negative"),
    (dict(n=1 << 30), "2^30"), (dict(ld_q=1 << 24), "2^24"), (dict(ld_k=1 << 24), "2^24"), (dict(ld_v=1 << 24), "2^24"),
    (dict(batch=1 << 28), "2^31")])
def test_linear_refuses(over, says):
    assert says in linear(**over)


@pytest.mark.parametrize("same", ["q", "k", "v"])
def test_linear_refuses_an_output_on_an_input(same):
    apart = {name: D + (i << 20) for i, name in enumerate(("q", "k", "v"))}
    assert "out is " + same in linear(**apart, out=apart[same], ld_v=576, ld_q=576, ld_k=576)


def test_linear_refuses_a_state_without_query_heads():
    """Without query heads there is no call to make; one that is asked for a state may not leave it unwritten."""
    assert "query heads" in linear(heads=0, ld_q=0, ld_o=0, state_out=D)
    assert "kv_heads must be" in linear(heads=0, ld_q=0, ld_o=0, kvh=1 << 60)
    lib = bh.lib()
    assert lib.bh_attention_linear(None, 0, D, 64, D, 64, None, 0, 2, 0, 1, 5, 64, 64, 0.0, None, None, None, None, bh.BF16, None, 0, None) == 0
    assert lib.bh_attention_linear(None, 0, None, 64, None, 64, None, 0, 0, 0, 1, 5, 64, 64, 0.0, None, None, None, D, bh.BF16, None, 0, None) == 0


def norms(plan=None, **over):
    a = dict(x=D, ld_x=64, residual=D, ld_res=64, residual_out=D, ld_res_out=64, out=D, ld_out=64, rows=4, cols=64)
    kinds = dict(residual_dtype=bh.BF16, dtype=bh.BF16)
    for name, v in over.items():
        (kinds if name in kinds else a)[name] = v
    f = dict(post_norm=bh.NORM_RMS, pre_norm=bh.NORM_LAYER, post_eps=1e-6, pre_eps=1e-6, branch_scale=1.0, residual_scale=1.0)
    f.update(plan or {})
    f = None if plan is False else ctypes.byref(bh.ResidualNorms(**f))
    return refused("bh_residual_norms_run", *a.values(), f, *kinds.values(), None)


@pytest.mark.parametrize("over,says", [
    (dict(x=None), "x is null"), (dict(residual=None), "residual is null"), (dict(out=None, residual_out=None), "neither"),
    (dict(rows=-1), "rows is negative"), (dict(cols=0), "cols must be"), (dict(cols=32769, ld_x=1 << 16), "cols must be"),
    (dict(ld_x=63), "row stride"), (dict(ld_res=63), "row stride"), (dict(ld_res_out=63), "row stride"), (dict(ld_out=63), "row stride"),
    (dict(dtype=5), "dtype 5"), (dict(residual_dtype=5), "dtype 5"), (dict(dtype=bh.F32), "bf16 residual"),
    (dict(x=D + 1, out=D + 2), "aligned to its type"), (dict(residual=D + 2, residual_dtype=bh.F32), "aligned to its type"),
    (dict(ld_out=72), "another stride"), (dict(ld_res_out=72), "another stride")])
def test_norms_refuse(over, says):
    assert says in norms(**over)


@pytest.mark.parametrize("plan,says", [
    (False, "struct is null"), (dict(post_norm=3), "unknown norm"), (dict(pre_norm=-1), "unknown norm"), (dict(post_eps=-1.0), "eps is negative"),
    (dict(pre_eps=math.nan), "eps is negative"), (dict(post_norm=0, post_weight=D), "without a norm"), (dict(pre_norm=0, pre_bias=D), "without a norm"),
    (dict(gate=D), "mod_rows"), (dict(scale=D, mod_rows=1, ld_mod=63), "ld_mod"), (dict(shift=D + 1, mod_rows=4, ld_mod=64), "aligned to its type"),
    (dict(post_weight=D + 1), "aligned to its type")])
def test_norms_refuse_plans(plan, says):
    assert says in norms(plan)


def test_queries_refuse_and_answer():
    lib = bh.lib()
    assert lib.bh_attention_linear_workspace_bytes(-1, 8, 2, 5, 64, 64) == -1 and b"negative" in lib.bh_last_error()
    assert lib.bh_attention_linear_workspace_bytes(1, 8, 3, 5, 64, 64) == -1
    assert lib.bh_attention_linear_workspace_bytes(1, 8, 2, 5, 64, 60) == -1
    assert lib.bh_attention_linear_workspace_bytes(0, 8, 2, 5, 64, 64) == 0 and lib.bh_last_error() == b""
    assert lib.bh_attention_linear_workspace_bytes(1, 8, 2, 0, 64, 64) == 0
    out = bh.AttentionLinearPlan()
    assert lib.bh_attention_linear_describe(1, 8, 2, 5, 64, 64, 1, -1, ctypes.byref(out)) != 0 and b"cus" in lib.bh_last_error()
    assert lib.bh_attention_linear_describe(1, 8, 2, 5, 64, 64, 1, 256, None) != 0 and b"null" in lib.bh_last_error()
    bh.call("bh_attention_linear_describe", 0, 8, 2, 5, 64, 64, 1, 256, ctypes.byref(out))
    assert (out.chunk, out.segments, out.workgroups) == (0, 0, 0)


def test_empty_calls_are_no_ops():
    lib = bh.lib()
    axes, plan = bh.RopeAxes.of([4]), bh.ResidualNorms()
    assert lib.bh_rope(ctypes.byref(axes), None, 0, None, 64, None, 64, 1, None, 64, None, 64, 1, 0, 64, 0, bh.BF16, None) == 0
    assert lib.bh_rope(ctypes.byref(axes), None, 0, None, 0, None, 0, 0, None, 0, None, 0, 0, 7, 64, 0, bh.BF16, None) == 0
    assert lib.bh_attention_linear(None, 64, None, 64, None, 64, None, 64, 0, 1, 1, 5, 64, 64, 0.0, None, None, None, None, bh.BF16, None, 0, None) == 0
    assert lib.bh_attention_linear(None, 64, None, 64, None, 64, None, 64, 2, 1, 1, 0, 64, 64, 0.0, None, None, None, None, bh.BF16, None, 0, None) == 0
    assert lib.bh_residual_norms_run(None, 64, None, 64, D, 64, None, 64, 0, 64, ctypes.byref(plan), bh.F32, bh.BF16, None) == 0


def test_norms_struct_keeps_what_its_caller_does_not_name():
    """Factors that are not named are 1, those that are stay as given; a zeroed struct of C has 0."""
    plan = bh.ResidualNorms()
    assert (plan.branch_scale, plan.residual_scale) == (1.0, 1.0)
    assert (plan.post_norm, plan.pre_norm, plan.gate, plan.mod_rows, plan.weight_offset) == (bh.NORM_NONE, bh.NORM_NONE, None, 0, 0.0)
    plan = bh.ResidualNorms(post_norm=bh.NORM_RMS, branch_scale=0.0, residual_scale=0.5)
    assert (plan.post_norm, plan.branch_scale, plan.residual_scale) == (bh.NORM_RMS, 0.0, 0.5)
    plan = bh.ResidualNorms(bh.NORM_LAYER, None, None, 0.25, None, 3.0)
    assert (plan.post_norm, plan.post_eps, plan.branch_scale, plan.residual_scale) == (bh.NORM_LAYER, 0.25, 3.0, 1.0)
