"""Appending to a paged cache and evicting from it: every byte of the caches is compared."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

bf16, f16, f32, e4m3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def appended(cache, table, x, positions, counts, scale):
    """The cache's bits after the tokens, on the CPU."""
    bits = ref.as_bits(cache).cpu().clone()
    B, heads, T, d = x.shape
    size = cache.shape[2]
    for b in range(B):
        for t in range(T if counts is None else min(T, counts[b])):
            at = positions[b] + t
            if not 0 <= at < table.shape[1] * size:
                continue
            page = int(table[b, at // size])
            if not 0 <= page < cache.shape[0]:
                continue
            row = x[b, :, t].cpu()
            if cache.dtype == e4m3:
                row = torch.clamp(row.float() / scale, -448.0, 448.0)
            bits[page, :, at % size] = ref.as_bits(row.to(cache.dtype))
    return bits


@pytest.mark.parametrize("dtype,cache_dtype", [(bf16, bf16), (f16, f16), (f32, f32), (bf16, e4m3), (f16, e4m3), (f32, e4m3)])
@pytest.mark.parametrize("d,size,layout,pad", [(64, 16, "heads", 0), (7, 5, "slots", 0), (100, 16, "slots", 3), (1, 1, "heads", 0), (256, 32, "heads", 8)])
def test_append(dtype, cache_dtype, d, size, layout, pad):
    B, heads, T = 5, 3, 9
    c = ref.Cache([40] * B, heads, size, d, cache_dtype, layout=layout, pad=pad, seed=d)
    g = torch.Generator().manual_seed(d)
    k, v = ((200 * torch.randn(B, T, heads, d, generator=g)).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    positions, counts = [0, 13, 40 - T, -3, 38], [T, 4, T, T, 7]
    c.table[1, -1] = -1
    table = c.table.cpu()
    scales = (0.37, 1.7) if cache_dtype == e4m3 else (1.0, 1.0)
    device = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for many in (counts, None):
        want = [appended(cache, table, x, positions, many, s) for cache, x, s in ((c.k_cache, k, scales[0]), (c.v_cache, v, scales[1]))]
        got = ops.kv_append(k, v, c.k_cache, c.v_cache, c.table, device(positions), counts=None if many is None else device(many),
                            k_scale=scales[0], v_scale=scales[1])
        assert got[0] is c.k_cache and got[1] is c.v_cache
        for cache, bits in zip(got, want):
            assert torch.equal(ref.as_bits(cache).cpu(), bits)


@pytest.mark.parametrize("B,T,heads", [(64, 1, 12), (1, 1, 1), (2, 700, 2), (300, 1, 1)])
def test_append_of_one_token_and_of_many(B, T, heads):
    c = ref.Cache([T] * B, heads, 16, 64, bf16, seed=B)
    store = torch.randn(2, B, T, heads * 64, generator=torch.Generator().manual_seed(B)).to(bf16).cuda()
    k, v = (x.view(B, T, heads, 64).transpose(1, 2) for x in store)
    want = [appended(cache, c.table_cpu, x, [0] * B, None, 1.0) for cache, x in ((c.k_cache, k), (c.v_cache, v))]
    ops.kv_append(k, v, c.k_cache, c.v_cache, c.table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    assert torch.equal(ref.as_bits(c.k_cache).cpu(), want[0]) and torch.equal(ref.as_bits(c.v_cache).cpu(), want[1])


def test_codes_of_8_bits_saturate_round_to_even_and_keep_nan():
    x = torch.tensor([0.0, -0.0, 448.0, 464.0, 1e30, -1e30, math.inf, -math.inf, math.nan, 2**-9, 2**-10, 3 * 2**-10, 17.0, 19.0, 2**-12, -21.0])
    c = ref.Cache([1], 1, 1, 16, e4m3)
    ops.kv_append(x.view(1, 1, 1, 16).cuda(), -x.view(1, 1, 1, 16).cuda(), c.k_cache, c.v_cache, c.table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    for cache, y in ((c.k_cache, x), (c.v_cache, -x)):
        row = cache[c.table[0, 0].long(), 0, 0].float().cpu()
        assert torch.equal(row.nan_to_num(nan=7.0), y.clamp(-448, 448).to(e4m3).float().nan_to_num(nan=7.0))
        assert row[8].isnan()


def evicted(c, weights, budget, recent):
    """Bits of both caches and the weights after the eviction, on the CPU."""
    caches = [ref.as_bits(x).cpu().clone() for x in (c.k_cache, c.v_cache)]
    w = weights.cpu().clone()
    new = []
    for b, n in enumerate(c.lengths):
        m = min(n, budget)
        new.append(m)
        if n <= budget:
            continue
        at = lambda t: (int(c.table_cpu[b, t // c.size]), t % c.size)  # noqa: E731
        for h in range(c.heads):
            kept = ref.evict(w[b, h], n, budget, recent)
            for bits in caches:
                rows = [bits[at(t)[0], h, at(t)[1]].clone() for t in kept]
                for j, row in enumerate(rows):
                    bits[at(j)[0], h, at(j)[1]] = row
            w[b, h, :m] = w[b, h][kept].clone()
            w[b, h, m:n] = 0
    return new, caches, w


def weights_like(c, seed, kind="spread"):
    g = torch.Generator().manual_seed(seed)
    shape = (len(c.lengths), c.heads, c.capacity)
    w = torch.exp(3 * torch.randn(shape, generator=g))
    if kind == "ties":  # few values, many times each
        w = torch.randint(0, 4, shape, generator=g).float()
    elif kind == "odd":
        w = torch.randn(shape, generator=g)
        w.view(-1)[::5] = 0.0
        w.view(-1)[1::5] = -0.0
        w.view(-1)[2::7] = math.nan
        w.view(-1)[3::11] = -math.inf
        w.view(-1)[4::13] = math.inf
        w.view(-1)[6::17] = 1e-42
    elif kind == "same":
        w = torch.full(shape, 0.25)
    return w.cuda()


def check_evict(c, weights, budget, recent, **options):
    new, caches, w = evicted(c, weights, budget, recent)
    got = ops.kv_evict(c.k_cache, c.v_cache, weights, c.table, c.device_lengths, budget, recent=recent, **options)
    assert got.tolist() == new
    for cache, bits in zip((c.k_cache, c.v_cache), caches):
        assert torch.equal(ref.as_bits(cache).cpu(), bits)
    assert torch.equal(ref.as_bits(weights).cpu(), ref.as_bits(w))  # (bits: a NaN or -0 that stays is moved, not made)
    return got


@pytest.mark.parametrize("kind", ["spread", "ties", "odd", "same"])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (100, 0), (100, 100), (100, 17), (257, 1), (700, 64), (5000, 9)])
def test_evict(kind, budget, recent):
    c = ref.Cache([0, 1, 99, 100, 101, 700, 701, 1025], 2, 16, 64, bf16, seed=budget)
    check_evict(c, weights_like(c, recent, kind), budget, recent)


@pytest.mark.parametrize("dtype,d,size,layout,pad", [(f32, 80, 24, "slots", 0), (e4m3, 128, 16, "heads", 0), (e4m3, 5, 7, "heads", 2), (f16, 7, 1, "slots", 0),
                                                     (bf16, 256, 64, "heads", 0), (f32, 3, 5, "heads", 1), (f16, 100, 32, "slots", 5)])
def test_evict_moves_rows_of_any_type_and_layout(dtype, d, size, layout, pad):
    c = ref.Cache([3, 150, 290], 3, size, d, dtype, seed=d, layout=layout, pad=pad)
    check_evict(c, weights_like(c, d), 61, 20)


def test_evict_of_a_long_sequence():
    c = ref.Cache([20000, 4097], 1, 64, 64, bf16, seed=3)
    check_evict(c, weights_like(c, 3), 4000, 100)


def test_evict_writes_the_lengths_in_place_and_can_be_repeated():
    c = ref.Cache([30, 300], 2, 16, 64, bf16, seed=4)
    weights = weights_like(c, 4)
    got = check_evict(c, weights, 50, 10, out=c.device_lengths)
    assert got is c.device_lengths
    c.lengths = [30, 50]
    check_evict(c, weights, 50, 10, out=c.device_lengths)  # nothing is longer now
    check_evict(c, weights, 20, 20)


def test_evict_with_a_strided_weight_tensor_and_a_workspace():
    c = ref.Cache([130, 90], 2, 16, 64, bf16, seed=5)
    full = torch.full((2, 3, c.capacity + 11), 5.0, device="cuda")
    weights = full[:, :2, : c.capacity + 4]
    weights[:, :, : c.capacity] = weights_like(c, 5)
    need = ops.kv_evict_workspace_bytes(c.k_cache, c.table, 64)
    check_evict(c, weights, 64, 8, workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    assert (full[:, 2] == 5).all() and (full[:, :, c.capacity:] == 5).all()
    with pytest.raises(ValueError, match="workspace"):
        ops.kv_evict(c.k_cache, c.v_cache, weights, c.table, c.device_lengths, 64, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("d", [64, 128])
def test_evict_of_many_heads(d):
    """Workgroups enough for slices of whole lines, several blocks of rows each, the last of them cut anywhere."""
    c = ref.Cache([1500, 701, 2000, 5, 1024, 769], 8, 16, d, f16, seed=6)
    check_evict(c, weights_like(c, 6), 700, 30)
    c = ref.Cache([1500, 770, 2000, 5, 1024, 769], 8, 16, d, f16, seed=7)
    check_evict(c, weights_like(c, 7, "ties"), 769, 0)


@pytest.mark.parametrize("d", [64, 7])
@pytest.mark.parametrize("heads", [2, 40])
def test_rows_on_pages_that_hold_nothing_do_not_move(heads, d):
    """A row stays where it is if its page, or the one it would go to, is none; all others and the weights move."""
    c = ref.Cache([600, 333], heads, 16, d, bf16, seed=8)
    table = c.table_cpu.clone()
    table[0, 3], table[0, 30], table[1, 0], table[1, 20] = -1, c.pages, 2**31 - 1, -(2**31)
    weights = weights_like(c, 8)
    caches = [ref.as_bits(x).cpu().clone() for x in (c.k_cache, c.v_cache)]
    w = weights.cpu().clone()
    for b, n in enumerate(c.lengths):
        for h in range(heads):
            kept = ref.evict(w[b, h], n, 300, 40)
            for bits in caches:
                before = bits[:, h].clone()
                for j, t in enumerate(kept):
                    source, target = int(table[b, t // 16]), int(table[b, j // 16])
                    if 0 <= source < c.pages and 0 <= target < c.pages:
                        bits[target, h, j % 16] = before[source, t % 16]
            w[b, h, :300] = w[b, h][kept].clone()
            w[b, h, 300:n] = 0
    assert ops.kv_evict(c.k_cache, c.v_cache, weights, table.cuda(), c.device_lengths, 300, recent=40).tolist() == [300, 300]
    for cache, bits in zip((c.k_cache, c.v_cache), caches):
        assert torch.equal(ref.as_bits(cache).cpu(), bits)
    assert torch.equal(ref.as_bits(weights).cpu(), ref.as_bits(w))


@pytest.mark.parametrize("dtype,cache_dtype", [(bf16, bf16), (f32, f32), (bf16, e4m3), (f32, e4m3)])
@pytest.mark.parametrize("B,T,heads,d", [(2, 2101, 2, 64), (3, 5001, 1, 7), (5, 903, 16, 128), (1, 36003, 1, 16), (4, 4500, 3, 20)])
def test_append_of_prompts_whose_workgroups_take_several_tokens(dtype, cache_dtype, B, T, heads, d):
    """2 to 16 tokens a workgroup; counts that end anywhere in its share, positions that leave the table, a page that is none."""
    c = ref.Cache([0] * B, heads, 16, d, cache_dtype, room=T + 40, seed=T)
    g = torch.Generator().manual_seed(T)
    k, v = ((100 * torch.randn(B, T, heads, d, generator=g)).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    positions = [0, 39, 45, -6, 3][:B]
    counts = [T - 1, T - 18, T + 5, 1, T // 2][:B]
    c.table[0, 7] = -1
    table = c.table.cpu()
    scales = (0.37, 1.7) if cache_dtype == e4m3 else (1.0, 1.0)
    device = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for many in (counts, None):
        want = [written(cache, table, x, positions, many, s) for cache, x, s in ((c.k_cache, k, scales[0]), (c.v_cache, v, scales[1]))]
        ops.kv_append(k, v, c.k_cache, c.v_cache, c.table, device(positions), counts=None if many is None else device(many), k_scale=scales[0], v_scale=scales[1])
        for cache, bits in zip((c.k_cache, c.v_cache), want):
            assert torch.equal(ref.as_bits(cache).cpu(), bits)


def written(cache, table, x, positions, counts, scale):
    """`appended` for many tokens: a sequence at a time."""
    bits = ref.as_bits(cache).cpu().clone()
    B, _, T, _ = x.shape
    size = cache.shape[2]
    for b in range(B):
        t = torch.arange(T if counts is None else min(T, counts[b]))
        at = positions[b] + t
        t, at = (y[(at >= 0) & (at < table.shape[1] * size)] for y in (t, at))
        page = table[b].long()[at // size]
        there = (page >= 0) & (page < cache.shape[0])
        rows = x[b].cpu()[:, t[there]].transpose(0, 1)
        if cache.dtype == e4m3:
            rows = torch.clamp(rows.float() / scale, -448.0, 448.0)
        bits[page[there], :, (at % size)[there]] = ref.as_bits(rows.to(cache.dtype).contiguous())
    return bits


def test_evict_clamps_the_lengths_to_the_table():
    c = ref.Cache([48, 48, 48, 48], 2, 16, 64, bf16, seed=10)
    weights = weights_like(c, 10)
    given = torch.tensor([-5, 2**31 - 1, 49, 20], dtype=torch.int32, device="cuda")
    c.lengths = [0, 48, 48, 20]
    new, caches, w = evicted(c, weights, 30, 4)
    assert ops.kv_evict(c.k_cache, c.v_cache, weights, c.table, given, 30, recent=4).tolist() == new == [0, 30, 30, 20]
    for cache, bits in zip((c.k_cache, c.v_cache), caches):
        assert torch.equal(ref.as_bits(cache).cpu(), bits)
    assert torch.equal(weights.cpu(), w)
    assert ops.kv_evict(c.k_cache, c.v_cache, weights, c.table, given, 60).tolist() == [0, 48, 48, 20]
