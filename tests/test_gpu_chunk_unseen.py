"""Attention of packed chunks: what a row does not see does not reach it, whatever the cache's type."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

bf16, f16, f32, e4m3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn

TABLES = [0, 1 << 17]  # positions of the table: as many as needed, or so many that up to 16 rows of a sequence are few and more are many


def starts_of(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def widen(c, positions):
    if positions // c.size > c.P:
        c.table = torch.nn.functional.pad(c.table, (0, positions // c.size - c.P), value=-1)
    return c


@pytest.mark.parametrize("positions", TABLES)
@pytest.mark.parametrize("d", [64, 50, 128])
@pytest.mark.parametrize("counts", [[150, 40], [4, 3]])
@pytest.mark.parametrize("cache_dtype,dtype,what,bad", [(*types, what, bad) for types in [(bf16, bf16), (f16, f16), (f32, f32), (e4m3, bf16), (e4m3, f16)]
                                                        for what in ("key", "value", "both") for bad in (math.nan, math.inf, -math.inf, 240.0)
                                                        if (types[0] != e4m3 or not math.isinf(bad)) and (what == "key" or bad != 240.0)])  # (e4m3 has no infinities)
def test_what_a_position_holds_stays_with_the_rows_that_see_it(positions, cache_dtype, dtype, d, counts, what, bad):
    """At a position in the middle of the chunk: rows before it, the other head and the other sequence are what they are without, bit for bit; a NaN
    key makes NaN of the rows that see it, a value that is no number makes its column none.  (A large key: the maxima of rows beside it move.)"""
    lengths = [260, 45]
    c = widen(ref.Cache(lengths, 2, 16, d, cache_dtype, seed=8), positions)
    q = torch.randn(sum(counts), 4, d, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
    call = lambda: ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of(counts))  # noqa: E731
    clean = call()
    assert torch.isfinite(clean).all()
    at = lengths[0] - counts[0] // 2
    row = at - (lengths[0] - counts[0])
    page, slot = int(c.table[0, at // 16]), at % 16
    if what != "value":
        c.k_cache[page, 0, slot, 7] = bad
    if what != "key":
        c.v_cache[page, 0, slot, 5] = bad
    dirty = call()
    assert torch.equal(dirty[:row], clean[:row]) and torch.equal(dirty[counts[0]:], clean[counts[0]:])
    assert torch.equal(dirty[:, 2:], clean[:, 2:])
    seeing = dirty[row:counts[0], :2]
    if what == "value":
        others = [i for i in range(d) if i != 5]
        assert not torch.isfinite(seeing[..., 5]).any() and torch.equal(seeing[..., others], clean[row:counts[0], :2, others])
    elif math.isnan(bad):  # (of other keys the score may be of either sign)
        assert torch.isnan(seeing).all()
