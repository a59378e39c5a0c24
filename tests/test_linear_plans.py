"""How linear attention chooses its form (no GPU here: the number of compute units is an argument)."""
import ctypes
import random

import pytest

import burnisher_amd as bh


def plan(batch, heads, kvh, n, d, e, workspace=1, cus=256):
    out = bh.AttentionLinearPlan()
    bh.call("bh_attention_linear_describe", batch, heads, kvh, n, d, e, workspace, cus, ctypes.byref(out))
    return out


def test_a_token_goes_by_itself_and_a_prompt_in_chunks():
    for n in (1, 2):
        p = plan(16, 32, 8, n, 128, 128)
        assert (p.chunk, p.segments) == (1, 1)
    for n in (3, 64, 300, 4096):
        assert plan(2, 64, 64, n, 64, 64).chunk == 32


@pytest.mark.parametrize("cus", [1, 8, 64, 256, 304])
def test_segments_fill_the_device_and_no_more(cus):
    rng = random.Random(cus)
    split = 0
    for _ in range(3000):
        kvh = rng.choice([1, 2, 8, 32])
        batch, heads, n = rng.randint(1, 16), kvh * rng.choice([1, 2, 8]), int(2 ** rng.uniform(5, 20))
        d, e = rng.choice([64, 72, 128]), rng.choice([40, 64, 128])
        p, alone = plan(batch, heads, kvh, n, d, e, cus=cus), plan(batch, heads, kvh, n, d, e, 0, cus)
        assert alone.segments == 1
        if p.chunk == 1:
            continue
        chunks = -(-n // 32)
        assert 1 <= p.segments <= chunks
        split += p.segments > 1
    assert split > 100 or cus == 1


def test_few_long_sequences_are_split():
    assert plan(1, 16, 16, 65536, 128, 128).segments > 8
    assert plan(2, 32, 8, 4096, 128, 128).segments > 1
    assert plan(16, 64, 64, 100, 64, 64).segments == 1
    assert plan(2, 64, 64, 300, 64, 64).segments == 1


# What the estimate has to say, from its own terms (us): a chunk takes 0.78 to 1.9 alone on a CU, the launches of a split 6 in all,
# a state's load and store at most 2.2 a launch, the carry of at most 76 heads in four segments 8.7. Of c chunks four segments save
# 0.65 c chunks, so that 20 of them outweigh all that (15.9 / 1.25 < 14 at 128 columns, 7 / 0.5 = 14 at 32), rounding up included.
def sizes(rng, most):
    kvh = rng.choice([1, 2, 3, 8, 32])
    return rng.randint(1, most), kvh * rng.choice([1, 1, 2, 3, 4, 8]), kvh, int(2 ** rng.uniform(5, 20)), rng.choice([8, 32, 64, 72, 96, 128]), rng.choice(
        [8, 40, 64, 80, 128])


@pytest.mark.parametrize("cus", [64, 256, 304])
def test_no_long_segments_on_a_quarter_of_the_device(cus):
    rng, few = random.Random(cus), 0
    for _ in range(5000):
        batch, heads, kvh, n, d, e = sizes(rng, 4)
        p, alone = plan(batch, heads, kvh, n, d, e, cus=cus), plan(batch, heads, kvh, n, d, e, 0, cus)
        chunks = -(-n // 32)
        if 4 * alone.workgroups <= cus and chunks >= 20:
            few += 1
            assert p.segments > 1, (batch, heads, kvh, n, d, e)
            assert 4 * p.workgroups > cus or chunks < 20 * p.segments, (batch, heads, kvh, n, d, e, p.segments)
    assert few > 300


# A split reads k and v of half the sequence again at least, at 0.4 of a chunk's time: 0.2 of a call of one query head a key head.
# It can save what the last round of workgroups leaves idle, less than 0.2 from five rounds on. Of eight query heads a key head, two at
# once, the second reading is 0.2 * 0.73 / (4 * 1.45 * 0.84) = 0.03 of the call, and 34 rounds leave less.
@pytest.mark.parametrize("cus", [8, 64, 256, 304])
def test_a_full_device_splits_nothing(cus):
    rng, ungrouped, grouped = random.Random(cus), 0, 0
    for _ in range(5000):
        batch, heads, kvh, n, d, e = sizes(rng, rng.choice([64, 1024]))
        p = plan(batch, heads, kvh, n, d, e, cus=cus)
        if heads == kvh and batch * heads >= 5 * cus:
            ungrouped += 1
            assert p.segments == 1, (batch, heads, kvh, n, d, e)
        if batch * heads >= 2 * 34 * cus:
            grouped += 1
            assert p.segments == 1, (batch, heads, kvh, n, d, e)
    assert ungrouped > 100 and grouped > 100
