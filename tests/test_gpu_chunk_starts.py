"""Attention of packed chunks whose starts are of any kind: nothing is written but the rows of the sequences."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

bf16, f32 = torch.bfloat16, torch.float32


def widen(c, positions):
    if positions // c.size > c.P:
        c.table = torch.nn.functional.pad(c.table, (0, positions // c.size - c.P), value=-1)
    return c


@pytest.mark.parametrize("positions", [0, 1 << 13, 1 << 17])
@pytest.mark.parametrize("dtype,d", [(bf16, 64), (f32, 64), (bf16, 50)])
@pytest.mark.parametrize("starts", [[5, 3, 2000, -7], [-5, 2**31 - 1, -(2**31), 90], [0, 0, 0, 0], [90, 90, 90, 90], [3, 40, 80, 85], [0, 2, 3, 4]])
def test_starts_of_any_kind_leave_the_rows_around_the_sequences_alone(positions, dtype, d, starts):
    """Between guards: rows before the first start (there are some where it is not 0) and behind the last, clamped to the rows, stay as they were."""
    c = widen(ref.Cache([100, 33, 50], 2, 16, d, dtype, seed=14), positions)
    N = 90
    q = torch.randn(N, 4, d, generator=torch.Generator().manual_seed(14)).to(dtype).cuda()
    store = torch.full((N + 64, 4, d), 7.0, dtype=dtype, device="cuda")
    out = store[32:32 + N]
    ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    assert (store[:32] == 7).all() and (store[32 + N:] == 7).all()
    at = [min(max(s, 0), N) for s in starts]
    covered = torch.zeros(N, dtype=torch.bool)
    for lo, hi in zip(at, at[1:]):
        covered[lo:max(lo, hi)] = True
    assert (out[~covered.cuda()] == 7).all()
    if at == sorted(at):  # (the rows of sequences are what they are by themselves)
        for b, (lo, hi) in enumerate(zip(at, at[1:])):
            n = c.lengths[b]
            for i in {lo, hi - 1} if hi > lo else ():
                seen = n - (hi - lo) + i - lo + 1
                k, v = (c.rows(cache, b, max(seen, 0)).double() for cache in (c.k_cache, c.v_cache))
                want, _, allowed, _ = ref.attention(q[i].cpu(), k, v, 1 / math.sqrt(d))
                assert ((out[i].cpu().double() - want).abs() <= allowed).all()
