"""Attention of one new token over a paged cache against the 64-bit statement of it, at the sizes and masks where it can go wrong.
Every slot that no position uses holds NaN, every table entry behind a sequence a page that does not exist."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

bf16, f16, f32, e4m3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def check(q, c, out, *, scale=None, weights=None, before=None, lengths=None):
    scale = 1.0 / math.sqrt(c.d) if scale is None else scale
    out = out.cpu().double()
    for b, n in enumerate(c.lengths if lengths is None else lengths):
        k, v = (c.rows(cache, b, n).double() for cache in (c.k_cache, c.v_cache))
        want, w, allowed, w_allowed = ref.attention(q[b].cpu(), k * c.k_scale, v, scale, c.v_scale)
        bad = ~((out[b] - want).abs() <= allowed)
        assert not bad.any(), (b, n, float(((out[b] - want).abs() / allowed).max()))
        if weights is not None:
            got, old = weights[b].cpu().double(), before[b].cpu().double()
            assert (got[:, n:] == old[:, n:]).all()
            off = (got[:, :n] - old[:, :n] - w).abs()
            assert (off <= w_allowed + 2.0**-23 * got[:, :n].abs()).all(), (b, n)


RAGGED = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 400]


@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("d", [64, 128, 80, 256])
def test_lengths_around_every_border(dtype, d):
    c = ref.Cache(RAGGED, 2, 16, d, dtype, seed=d)
    q = torch.randn(len(RAGGED), 4, d, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths))


@pytest.mark.parametrize("heads,G", [(1, 1), (12, 1), (3, 5), (2, 16), (1, 17), (2, 40)])
def test_groups_of_heads(heads, G):
    c = ref.Cache([70, 333], heads, 32, 64, bf16, seed=G)
    q = torch.randn(2, heads * G, 64, generator=torch.Generator().manual_seed(2)).to(bf16).cuda()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths))


@pytest.mark.parametrize("size", [1, 7, 16, 24, 48, 100, 1024])
@pytest.mark.parametrize("layout", ["heads", "slots"])
def test_page_sizes_and_layouts(size, layout):
    c = ref.Cache([1, size, size + 1, 310], 3, size, 96, f16, seed=size, layout=layout, room=5)
    q = torch.randn(4, 6, 96, generator=torch.Generator().manual_seed(3)).to(f16).cuda()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths))


@pytest.mark.parametrize("dtype,d,pad", [(bf16, 1, 0), (bf16, 7, 0), (f16, 33, 2), (f32, 3, 0), (f32, 101, 1), (bf16, 255, 0), (f16, 72, 1),
                                         (bf16, 200, 8), (f32, 4, 0), (e4m3, 5, 0), (e4m3, 136, 0), (e4m3, 250, 3)])
def test_odd_head_dimensions_and_row_strides(dtype, d, pad):
    c = ref.Cache([5, 130, 0, 257], 2, 16, d, dtype, seed=d, pad=pad, scales=(0.5, 2.0) if dtype == e4m3 else (1.0, 1.0))
    q = torch.randn(4, 4, d, generator=torch.Generator().manual_seed(4)).to(bf16 if dtype == e4m3 else dtype).cuda()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, k_scale=c.k_scale, v_scale=c.v_scale))


@pytest.mark.parametrize("dtype,d,pad", [(bf16, 33, 0), (f16, 181, 2), (f32, 101, 0), (e4m3, 136, 0), (e4m3, 250, 1), (bf16, 9, 0), (f32, 5, 3), (e4m3, 17, 0)])
def test_odd_rows_of_long_caches(dtype, d, pad):
    """Rows that are no whole pieces, in several shares, with weights."""
    c = ref.Cache([3100, 17, 0, 1025], 2, 16, d, dtype, seed=d, pad=pad)
    q = torch.randn(4, 6, d, generator=torch.Generator().manual_seed(4)).to(bf16 if dtype == e4m3 else dtype).cuda()
    weights = torch.rand(4, 2, c.capacity, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    before = weights.clone()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, weights=weights), weights=weights, before=before)


@pytest.mark.parametrize("q_dtype", [bf16, f16])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
def test_cache_of_8_bits(q_dtype, d):
    c = ref.Cache(RAGGED, 2, 16, d, e4m3, seed=d, scales=(0.75, 1.5))
    q = torch.randn(len(RAGGED), 8, d, generator=torch.Generator().manual_seed(5)).to(q_dtype).cuda()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, k_scale=0.75, v_scale=1.5))


@pytest.mark.parametrize("dtype,G,size", [(bf16, 1, 16), (f16, 4, 16), (f32, 2, 24), (bf16, 20, 10), (e4m3, 3, 32)])
def test_weights_grow_by_the_probabilities(dtype, G, size):
    c = ref.Cache([0, 1, 100, 2000], 2, size, 64, dtype, seed=G)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(4, 2 * G, 64, generator=g).to(bf16 if dtype == e4m3 else dtype).cuda()
    store = torch.rand(4, 2, c.capacity + 9, generator=g).cuda()
    weights = store[:, :, : c.capacity + 3]
    before = weights.clone()
    out = ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, weights=weights)
    check(q, c, out, weights=weights, before=before)


@pytest.mark.parametrize("lengths,heads", [([3000], 1), ([5000, 1, 0, 2999], 2), ([700] * 3, 4)])
def test_long_caches_are_split_and_joined(lengths, heads):
    c = ref.Cache(lengths, heads, 64, 128, bf16, seed=7)
    q = (3.0 * torch.randn(len(lengths), 4 * heads, 128, generator=torch.Generator().manual_seed(7))).to(bf16).cuda()
    if max(lengths) > 1000:  # (partial results of several workgroups)
        assert ops.paged_attention_workspace_bytes(q, c.k_cache, c.v_cache, c.table) > 0
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths))


def test_a_table_much_wider_than_the_sequences():
    c = ref.Cache([5, 40, 129], 2, 16, 64, bf16, seed=8)
    wide = torch.full((3, 4000), -1, dtype=torch.int32, device="cuda")
    wide[:, : c.P] = c.table
    q = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(8)).to(bf16).cuda()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, wide, c.device_lengths))


def test_lengths_outside_the_table_are_clamped():
    c = ref.Cache([48, 48, 48], 2, 16, 64, bf16, seed=9)
    q = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(9)).to(bf16).cuda()
    lengths = torch.tensor([-5, 2**31 - 1, 49], dtype=torch.int32, device="cuda")
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, lengths), lengths=[0, 48, 48])


@pytest.mark.parametrize("size", [16, 10])
def test_pages_that_hold_nothing_are_left_out(size):
    """A position on a page outside the cache does not take part; a sequence of such pages alone gives 0."""
    c = ref.Cache([5 * size, 5 * size], 2, size, 64, bf16, seed=10)
    table = c.table.clone()
    table[0, 1], table[0, 3] = -7, c.pages
    table[1] = -1
    q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(10)).to(bf16).cuda()
    weights = torch.zeros(2, 2, 5 * size, device="cuda")
    out = ops.paged_attention(q, c.k_cache, c.v_cache, table, c.device_lengths, weights=weights).cpu()
    there = [t for t in range(5 * size) if t // size in (0, 2, 4)]
    k, v = (c.rows(cache, 0, 5 * size)[:, there].double() for cache in (c.k_cache, c.v_cache))
    want, w, allowed, _ = ref.attention(q[0].cpu(), k, v, 0.125)
    assert ((out[0].double() - want).abs() <= allowed).all()
    assert (out[1] == 0).all() and (weights[1] == 0).all()
    assert (weights[0, :, size:2 * size] == 0).all() and (weights[0, :, 3 * size:4 * size] == 0).all()
    assert (weights[0].cpu().double()[:, there] - w).abs().max() < 1e-5


def test_values_that_are_no_numbers_stay_where_they_are():
    """An infinite or NaN key or value of one position shows in its own sequence and head only."""
    c = ref.Cache([40, 40], 2, 16, 64, bf16, seed=11)
    q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(11)).to(bf16).cuda()
    clean = ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths)
    c.v_cache[c.table[0, 1].long(), 1, 3, 5] = math.inf
    out = ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths)
    assert not out[0, 1, 5].isfinite()
    out[0, 1, 5] = clean[0, 1, 5]
    assert torch.equal(out, clean)
    c.k_cache[c.table[0, 1].long(), 0, 3, 5] = math.nan
    out = ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths)
    assert out[0, 0].isnan().all() and torch.equal(out[1], clean[1])


@pytest.mark.parametrize("factor", [0.0, -1.0, 60.0])
def test_scales(factor):
    """No preference, a reversed one, and scores whose exponentials span the whole range of f32."""
    c = ref.Cache([3, 200], 2, 16, 64, f32, seed=12)
    q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(12)).cuda()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, scale=factor / 8), scale=factor / 8)


def test_many_small_probabilities_in_f16():
    """One position and, far below it, the 131071 others: each has a probability that f16 has no number for, together they are 0.4 %.
    All of them lie on one page, so that 512 long rows fit in little memory."""
    d, size, n, B, heads = 64, 16, 131072, 64, 8
    k, v = torch.zeros(2, heads, size, d, dtype=f16), torch.ones(2, heads, size, d, dtype=f16)
    k[0, :, 0, 0], v[0, :, 0] = 17.375, 0.0
    table = torch.ones(B, n // size, dtype=torch.int32)
    table[:, 0] = 0
    q = torch.zeros(B, heads, d, dtype=f16)
    q[:, :, 0] = 1.0
    out = ops.paged_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.full((B,), n, dtype=torch.int32).cuda(), scale=1.0).cpu().double()
    small = (n - 1) * math.exp(-17.375)
    want = small / (1.0 + small)
    # The result's rounding 2^-11.  The sum of a lane that starts with 1 does not see its 8 positions of at most 1024 steps: 8192 exp(-17.375)
    # = 2^-12.07.  The accumulators: at most 1024 steps of two products, 2^-24 each, 2^-13.  exp2 of a score of 25: 2^-19.
    assert ((out - want).abs() <= want * (2.0**-11 + 2.0**-12 + 2.0**-13 + 2.0**-16)).all(), float((out - want).abs().max() / want)


def test_strided_queries_and_outputs():
    c = ref.Cache([100, 30], 4, 16, 64, bf16, seed=13)
    store = torch.randn(2, 3 * 512 + 8, generator=torch.Generator().manual_seed(13)).to(bf16).cuda()
    q = store[:, 1:513].view(2, 8, 64)  # the first third of a fused projection, off by an element
    full = torch.full((2, 9, 70), 7.0, dtype=bf16, device="cuda")
    out = full[:, :8, 3:67]
    assert ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, out=out) is out
    check(q, c, out)
    assert (full[:, 8] == 7).all() and (full[:, :, :3] == 7).all() and (full[:, :, 67:] == 7).all()


def test_a_cache_behind_2_to_the_31_elements():
    pages = 2**31 // (16 * 128) + 9
    k_cache = torch.zeros(pages, 1, 16, 128, dtype=bf16, device="cuda")
    v_cache = torch.zeros(pages, 1, 16, 128, dtype=bf16, device="cuda")
    g = torch.Generator().manual_seed(14)
    k, v = (torch.randn(1, 1, 40, 128, generator=g).to(bf16).cuda() for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 5]], dtype=torch.int32, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv_append(k, v, k_cache, v_cache, table, zero)
    q = torch.randn(1, 2, 128, generator=g).to(bf16).cuda()
    out = ops.paged_attention(q, k_cache, v_cache, table, zero + 40)
    want, _, allowed, _ = ref.attention(q[0].cpu(), k[0].cpu(), v[0].cpu(), 128**-0.5)
    assert ((out[0].cpu().double() - want).abs() <= allowed).all()
    assert torch.equal(k_cache[pages - 1, 0], k[0, 0, :16]) and torch.equal(v_cache[pages - 5, 0, :8], v[0, 0, 32:])


def test_the_same_call_gives_the_same_bits_with_any_workspace():
    c = ref.Cache([2500, 7], 2, 16, 128, bf16, seed=15)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(15)).to(bf16).cuda()
    weights = torch.zeros(2, 2, c.capacity, device="cuda")
    first = ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, weights=weights)
    need = ops.paged_attention_workspace_bytes(q, c.k_cache, c.v_cache, c.table, weights=True)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # (NaN everywhere)
    again = torch.zeros_like(weights)
    assert torch.equal(first, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, weights=again, workspace=ws))
    assert torch.equal(weights, again)
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, weights=weights, workspace=ws[: need - 256])
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, weights=weights,
                            workspace=torch.empty(need + 256, dtype=torch.uint8, device="cuda")[16:])


@pytest.mark.parametrize("dtype", [bf16, f16, e4m3])
def test_probabilities_keep_the_places_of_f32(dtype):
    """Two values of +-256 whose probabilities differ by 2^-12 of themselves: what is left of their difference shows every place that a
    probability has lost on its way into the second product."""
    d, B, G = 64, 32, 16
    q_dtype = bf16 if dtype == e4m3 else dtype
    a = (1.0 + torch.arange(B * G) / 512.0).to(q_dtype).view(B, G)  # scores of -a and -a - 2^-12 beside one of 0
    q = torch.zeros(B, G, d, dtype=q_dtype)
    q[:, :, 0], q[:, :, 1] = a, 2.0**-12
    k, v = torch.zeros(1, 1, 16, d), torch.zeros(1, 1, 16, d)
    k[0, 0, 1:3, 0], k[0, 0, 2, 1] = -1.0, -1.0
    v[0, 0, 1], v[0, 0, 2] = 256.0, -256.0
    table = torch.zeros(B, 1, dtype=torch.int32).cuda()
    out = ops.paged_attention(q.cuda(), k.to(dtype).cuda(), v.to(dtype).cuda(), table, torch.full((B,), 3, dtype=torch.int32).cuda(), scale=1.0)
    s = a.double()
    p = torch.exp(-s)
    want = 256.0 * p * -math.expm1(-(2.0**-12)) / (1.0 + p + p * math.exp(-(2.0**-12)))
    # Scores are exact.  Times log2(e) in f32: 2^-25 of the factor and half a step of the product, both times ln 2 |x| <= 2: 2^-24 + 2^-24;
    # exp2 and the sum a step of 2^-23 each: 6 steps of 2^-24 for each probability.  The second product: six terms of at most 256 p
    # added in f32, 6 more; the quotient 2, relative to what is small.
    share = 256.0 * p / (1.0 + 2.0 * p)
    half = torch.finfo(q_dtype).eps / 2
    off = (out.cpu().double() - want[:, :, None]).abs()
    assert (off <= (half * want + share * (2 * 6 + 6) * 2.0**-24)[:, :, None]).all(), float(off.max())


def test_the_widest_table():
    """A table of nearly 2^31 positions, all on three pages; those of the last have nearly all the weight, and lie in the last share."""
    size, pages, d = 65536, 32766, 16
    k = torch.zeros(3, 1, size, d)
    k[2, :, :, 0] = 24.0
    v = (0.5 + torch.rand(3, 1, size, d, generator=torch.Generator().manual_seed(16))).to(e4m3)
    table = (torch.arange(pages, dtype=torch.int32) % 2).view(1, pages)
    table[0, -1] = 2
    q = torch.zeros(1, 1, d, dtype=bf16)
    q[0, 0, 0] = 1.0
    out = ops.paged_attention(q.cuda(), k.to(e4m3).cuda(), v.cuda(), table.cuda(), torch.full((1,), 2**31 - 1, dtype=torch.int32).cuda(), scale=1.0)
    mean = v.double().mean(2)[:, 0]
    rest = (pages - 1) // 2 * math.exp(-24.0)
    want = (mean[2] + rest * mean[0] + (rest + math.exp(-24.0)) * mean[1]) / (1.0 + 2 * rest + math.exp(-24.0))
    # Up to 2^18 positions of a lane and 2^16 steps of a wave are added one after the other in f32, and the result rounded to 2^-9.
    assert ((out[0, 0].cpu().double() - want).abs() <= want * (2.0**-6 + 2.0**-8 + 2.0**-9)).all()
    # Heads for every CU: a share is the whole table.
    B, heads = 129, 16
    k, v = (torch.randn(3, heads, size, d, generator=torch.Generator().manual_seed(17)).to(bf16) for _ in range(2))
    q = torch.randn(B, heads, d, generator=torch.Generator().manual_seed(18)).to(bf16)
    wide = torch.full((B, pages), -1, dtype=torch.int32)
    wide[:, 0] = torch.arange(B) % 3
    out = ops.paged_attention(q.cuda(), k.cuda(), v.cuda(), wide.cuda(), torch.arange(B, dtype=torch.int32).cuda())
    for b in range(B):
        want, _, allowed, _ = ref.attention(q[b], k[b % 3, :, :b], v[b % 3, :, :b], 0.25)
        assert ((out[b].cpu().double() - want).abs() <= allowed).all(), b


def test_a_workspace_sized_for_an_aligned_cache_serves_a_view():
    c = ref.Cache([4000, 17, 2100, 1], 8, 16, 128, f16, seed=19)
    q = torch.randn(4, 16, 128, generator=torch.Generator().manual_seed(19)).to(f16).cuda()
    need = ops.paged_attention_workspace_bytes(q, c.k_cache, c.v_cache, c.table)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, workspace=ws))
    store = torch.empty(2, c.k_cache.numel() + 4, dtype=f16, device="cuda")
    views = []
    for row, cache in zip(store, (c.k_cache, c.v_cache)):
        view = row[4:].view(cache.shape)  # 8 bytes further
        ref.as_bits(view).copy_(ref.as_bits(cache))
        views.append(view)
    check(q, c, ops.paged_attention(q, *views, c.table, c.device_lengths, workspace=ws))


@pytest.mark.parametrize("q_dtype", [bf16, f16])
@pytest.mark.parametrize("d,size,layout,pad", [(64, 24, "heads", 0), (128, 7, "slots", 0), (192, 24, "heads", 0), (256, 10, "slots", 16), (160, 8, "heads", 3), (32, 8, "heads", 0)])
def test_cache_of_8_bits_on_any_pages(q_dtype, d, size, layout, pad):
    c = ref.Cache([0, 1, size, 3 * size + 1, 1300], 2, size, d, e4m3, seed=d + size, layout=layout, pad=pad, scales=(0.75, 1.5))
    q = torch.randn(5, 8, d, generator=torch.Generator().manual_seed(20)).to(q_dtype).cuda()
    weights = torch.zeros(5, 2, c.capacity, device="cuda")
    before = weights.clone()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, weights=weights, k_scale=0.75, v_scale=1.5), weights=weights, before=before)


@pytest.mark.parametrize("d,size", [(64, 8), (128, 24), (256, 8), (32, 24), (24, 40)])
@pytest.mark.parametrize("dtype", [bf16, f32])
def test_pages_that_end_inside_a_tile(dtype, d, size):
    """Several shares of positions on pages that are a multiple of 8 but not of 16, tables with unused entries."""
    c = ref.Cache([2500, 8, 0, 777], 3, size, d, dtype, seed=d, room=3)
    q = torch.randn(4, 6, d, generator=torch.Generator().manual_seed(21)).to(dtype).cuda()
    check(q, c, ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths))
