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
