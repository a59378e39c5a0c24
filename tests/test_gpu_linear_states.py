"""States of bh_attention_linear in the forms that a call takes: what an empty sequence hands on, in one launch or three,
with one query head at once or two, in place or not."""
import ctypes
import math

import pytest

import burnisher_amd as bh
from test_gpu_linear import decays, inputs, normal, run

pytestmark = pytest.mark.gpu

# batch, heads, kv_heads, tokens, columns, segments (0: one, 1: more), query heads at once; a workspace is passed
FORMS = {"chunks": (3, 4, 2, 40, 64, 0, 1), "two heads": (12, 64, 16, 50, 64, 0, 2), "split": (3, 2, 2, 3000, 64, 1, 1),
         "split, two heads": (2, 16, 4, 3000, 128, 1, 2)}


def form(name):
    """The sizes of a form, which the call takes here."""
    batch, heads, kvh, n, d, split, at_once = FORMS[name]
    plan = bh.AttentionLinearPlan()
    bh.call("bh_attention_linear_describe", batch, heads, kvh, n, d, d, 1, 0, ctypes.byref(plan))
    assert plan.chunk == 32 and (plan.segments > 1) == bool(split)
    assert batch * heads * plan.segments == at_once * plan.workgroups
    return batch, heads, kvh, n, d


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("with_workspace", [True, False])
@pytest.mark.parametrize("name", FORMS)
def test_an_empty_sequence_hands_its_state_on(hip, name, with_workspace, in_place):
    """Bit by bit, infinities and NaN among it, as one or two tokens' form does; the sequences beside it are not touched."""
    import torch
    batch, heads, kvh, n, d = form(name)
    for tokens in (n, 2, 1):
        q, k, v = inputs(batch, heads, kvh, tokens, d, d, 1)
        state, rate = normal((batch, kvh, d, d), 2, 1.0, torch.float32), decays(kvh)
        state[0, 0, 3, :4] = torch.tensor([math.inf, -math.inf, math.nan, -0.0])
        state[0, kvh - 1, d - 1, d - 1] = math.inf
        rate[0] = 0.0
        lens = [0] + [tokens] * (batch - 1)
        out, new = run(q, k, v, rate, lens, state, with_workspace=with_workspace, in_place=in_place)
        assert torch.equal(new[0].view(torch.int32), state[0].view(torch.int32)), tokens
        assert not out[0].any() and out[1:].isfinite().all() and new[1:].isfinite().all()


# unsplit chunks: a workgroup with all heads of a key head alone reads and writes its state; others need the first state kept apart
@pytest.mark.parametrize("batch,heads,kvh,n,d,apart", [(12, 32, 16, 50, 128, False), (16, 32, 32, 100, 64, False), (12, 64, 16, 50, 64, True),
                                                       (3, 4, 2, 40, 64, True)])
def test_a_state_is_kept_apart_only_where_heads_share_it(hip, batch, heads, kvh, n, d, apart):
    import torch
    plan = bh.AttentionLinearPlan()
    bh.call("bh_attention_linear_describe", batch, heads, kvh, n, d, d, 1, 0, ctypes.byref(plan))
    assert (plan.chunk, plan.segments) == (32, 1) and (batch * kvh < plan.workgroups) == apart
    q, k, v = inputs(batch, heads, kvh, n, d, d, 1)
    need = bh.lib().bh_attention_linear_workspace_bytes(batch, heads, kvh, n, d, d)
    assert need == (4 * batch * kvh * d * d if apart else 0)
    state, rate = normal((batch, kvh, d, d), 2, 1.0, torch.float32), decays(kvh)
    want = run(q, k, v, rate, None, state)
    for with_workspace in (True, False):
        got = run(q, k, v, rate, None, state, with_workspace=with_workspace, in_place=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
