"""How exact the weights of attention of packed chunks are, in the kernel for many rows of a sequence and in the one for few: those of 16-bit
queries are sums of 16-bit values that leave no more than f32 does, as in attention of single tokens, whichever kernel a call gets."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

bf16, f16, f32, e4m3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def starts_of(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def attend(c, q, counts, **options):
    scales = {"k_scale": c.k_scale, "v_scale": c.v_scale} if c.dtype == e4m3 else {}
    return ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of(counts), **scales, **options)


def flat_queries(N, H, d, dtype):
    """Small ones: scores of a few tenths, so that every position has its part and values of either sign cancel."""
    return (0.25 * torch.randn(N, H, d, generator=torch.Generator().manual_seed(N))).to(dtype).cuda()


@pytest.mark.parametrize("cache_dtype,dtype", [(bf16, bf16), (f16, f16), (e4m3, bf16), (e4m3, f16)])
@pytest.mark.parametrize("d", [64, 96, 100, 128, 192, 256])
@pytest.mark.parametrize("lengths,counts", [([3000, 700], [200, 130]), ([1300, 700], [600, 600]), ([700, 45], [3, 4])])
def test_weights_lose_no_more_than_in_attention_of_single_tokens(cache_dtype, dtype, d, lengths, counts):
    """Within the bound of paged_reference.attention, whose weights are two 16-bit values: half a step of the result, the sums' errors in f32 and
    the product of two half steps of the weights times values.  Weights rounded once would be off by half a step of weights times
    values, which is many times the results here."""
    c = ref.Cache(lengths, 2, 16, d, cache_dtype, seed=d, scales=(0.75, 1.5) if cache_dtype == e4m3 else (1.0, 1.0))
    q = flat_queries(sum(counts), 4, d, dtype)
    out, at = attend(c, q, counts).cpu().double(), 0
    for b, n in enumerate(lengths):
        k, v = (c.rows(cache, b, n).double() for cache in (c.k_cache, c.v_cache))
        for i in sorted({r % counts[b] for r in (0, 1, 15, 31, 32, 63, 64, 100, 127, 128, -2, -1)}):
            seen = n - counts[b] + i + 1
            want, _, allowed, _ = ref.attention(q[at + i].cpu(), k[:, :seen] * c.k_scale, v[:, :seen], 1 / math.sqrt(d), c.v_scale)
            assert ((out[at + i] - want).abs() <= allowed).all(), (b, i, float(((out[at + i] - want).abs() / allowed).max()))
        at += counts[b]


@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("count", [140, 3])
def test_weights_that_would_all_round_one_way(dtype, count):
    """Every second position has the weight 1 and the value 1, the others a weight far from any number of the type, and a value that takes the
    sum to about 0.  (A table of 2^17 positions: 140 rows are many.)"""
    n, d = 300, 64
    c = ref.Cache([n], 1, 16, d, dtype, seed=2)
    keys = -torch.rand(4000, generator=torch.Generator().manual_seed(4), dtype=torch.float64).to(dtype).double()
    weights = torch.exp(2.0 * keys)  # (a query of 16, a scale of 1 / 8)
    key = float(keys[((weights.to(dtype).double() - weights).abs() / weights).argmax()])
    odd = torch.arange(1, n, 2)
    page, slot = c.table_cpu[0, torch.arange(n) // 16].long().cuda(), (torch.arange(n) % 16).cuda()
    c.k_cache[page, 0, slot], c.v_cache[page, 0, slot] = 0.0, 1.0
    c.k_cache[page[odd], 0, slot[odd], 0], c.v_cache[page[odd], 0, slot[odd]] = key, -1.0 / math.exp(2.0 * key)
    q = torch.zeros(count, 2, d, dtype=dtype)
    q[..., 0] = 16.0
    c.table = torch.nn.functional.pad(c.table, (0, 2**17 // 16 - c.P), value=-1)
    out = attend(c, q.cuda(), [count]).cpu().double()
    k, v = (c.rows(cache, 0, n).double() for cache in (c.k_cache, c.v_cache))
    for i in range(count):
        seen = n - count + i + 1
        want, _, allowed, _ = ref.attention(q[i], k[:, :seen], v[:, :seen], 1 / 8)
        assert ((out[i] - want).abs() <= allowed).all(), (i, float(((out[i] - want).abs() / allowed).max()))


@pytest.mark.parametrize("dtype", [bf16, f16])
def test_a_request_has_the_same_weights_in_any_company(dtype):
    """Two tokens of a sequence alone (few rows), beside long prompts (many rows), and one at a time: all within twice the bound of each other."""
    lengths, counts = [600, 900, 900], [2, 900, 900]
    c = ref.Cache(lengths, 2, 16, 128, dtype, seed=3)
    q = flat_queries(sum(counts), 8, 128, dtype)
    among = attend(c, q, counts)[:2]
    alone = ops.paged_attention_chunk(q[:2], c.k_cache, c.v_cache, c.table[:1], c.device_lengths[:1], starts_of([2]))
    single = ops.paged_attention(q[1:2], c.k_cache, c.v_cache, c.table[:1], c.device_lengths[:1])
    k, v = (c.rows(cache, 0, 600).double() for cache in (c.k_cache, c.v_cache))
    for i in range(2):
        _, _, allowed, _ = ref.attention(q[i].cpu(), k[:, :599 + i], v[:, :599 + i], 1 / math.sqrt(128))
        results = [among[i], alone[i]] + ([single[0]] if i == 1 else [])
        for x in results:
            for y in results:
                assert ((x - y).cpu().double().abs() <= 2 * allowed).all()


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("count", [130, 2])
def test_many_weights_far_below_the_largest_have_their_part(first, count):
    """f16: one position 2^25 times as heavy as each of 32767 others, whose values alone are not 0.  The others' weights lie 2^-37 apart or less from
    what they are (half the smallest step of f16, where the largest is held as 2^12 or more): 2^-22 of the values in all, and the sums'
    errors as in paged_reference.attention; the result is 2^-10."""
    n, d = 32768, 64
    c = ref.Cache([n], 1, 64, d, f16, seed=1)
    heavy = 0 if first else n - count
    for t, k0, v0 in [(None, 0.0, 1.0), (heavy, 8.6640625, 0.0)]:
        for cache, x in ((c.k_cache, k0), (c.v_cache, v0)):
            at = torch.arange(n) if t is None else torch.tensor([t])
            rows = torch.zeros(len(at), d, dtype=f16)
            rows[:, 0] = x
            cache[c.table_cpu[0, at // 64].long().cuda(), 0, (at % 64).cuda()] = (torch.full_like(rows, x) if cache is c.v_cache else rows).cuda()
    q = torch.zeros(count, 2, d, dtype=f16)
    q[..., 0] = 16.0
    out = attend(c, q.cuda(), [count]).cpu().double()
    for i in (0, 1, count - 1):
        seen = n - count + i + 1
        weight = math.exp(-16.0 * 8.6640625 / 8.0)
        want = (seen - 1) * weight / (1 + (seen - 1) * weight)
        allowed = 2.0**-11 * want + (seen + 64 + 2 * (d + 8) * 18) * 2.0**-24 * want + seen * 2.0**-37
        assert ((out[i] - want).abs() <= allowed).all(), (i, want, float((out[i] - want).abs().max()), allowed)
