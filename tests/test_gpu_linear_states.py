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


@pytest.mark.parametrize("name", FORMS)
def test_states_keep_24_bits_in_every_form(hip, name):
    """One token holds a key, so an element of the state is decay^(n - 1 - t) k v, and what it is off by is counted in units of 2^-24.

    The weight: two exponentials of 2, each with an exponent off by 2.5 of itself, and their product, 5; times the value 1, in three
    bf16 terms 1, added up one by one 3. In the sequence's last segment, or an unsplit one, the put-off decay 3 where it is applied
    on the way and 5 behind the last token. A piece of a split adds 1 for each piece behind it, whose decays are
    all near 1 here, and the other products are zeros. Together 24, the pieces behind, and 6 for each e-fold of the decay. A third
    term left out would be up to 256 (half a bf16 step of half a step)."""
    import torch
    batch, heads, kvh, n, d = form(name)
    plan = bh.AttentionLinearPlan()
    bh.call("bh_attention_linear_describe", batch, heads, kvh, n, d, d, 1, 0, ctypes.byref(plan))
    rate = torch.linspace(-1e-4, -3e-5, kvh, device="cuda")
    q, k, v = inputs(batch, heads, kvh, n, d, d, 7)
    for t in {0, n // 2, max(0, n - 3 * n // (2 * plan.segments)), max(0, n - 40), n - 1}:
        one = torch.zeros_like(k)
        one[:, t] = k[:, t]
        out, new = run(q, one, v, rate)
        fade = rate.double() * (n - 1 - t)
        want = torch.exp(fade)[None, :, None, None] * k[:, t].double()[..., :, None] * v[:, t].double()[..., None, :]
        pieces = 0 if plan.segments == 1 else 2 * ((n - t) * plan.segments // n + 1)
        slack = 2.0 ** -24 * (24 + pieces + 6 * fade.abs()[None, :, None, None])
        assert ((new.double() - want).abs() <= want.abs() * slack + 1e-37).all(), t
        assert not out[:, :t].any()
