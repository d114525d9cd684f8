"""Attention of packed chunks over a paged cache against the 64-bit statement of it, row by row.  Every slot that no position uses holds
NaN, every table entry behind a sequence a page that does not exist."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

bf16, f16, f32, e4m3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


WIDE = [False]


@pytest.fixture(autouse=True, params=[False, True], ids=["tight", "wide"])
def wide(request):
    """Every test with tables as wide as the sequences need, and with ones of 2^19 positions: which kernel a call is for goes by what it might have to do."""
    WIDE[0] = request.param


def widened(c, positions):
    columns = positions // c.size
    if columns > c.table.shape[1] and columns * c.table.shape[0] <= 1 << 24:
        c.table = torch.nn.functional.pad(c.table, (0, columns - c.table.shape[1]), value=-1)
    return c


def cache(*args, **options):
    c = ref.Cache(*args, **options)
    return widened(c, 1 << 19) if WIDE[0] else c


def starts_of(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def queries(counts, H, d, dtype, seed=0, spare=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (size * torch.randn(sum(counts) + spare, H, d, generator=g)).to(bf16 if dtype == e4m3 else dtype).cuda()


def statement(q, k, v, scale, v_scale=1.0):
    """(result, error allowed) of one row in 64 bits: that of paged attention, and, for 16-bit queries, of weights rounded to their type once: each is
    off by half a step, in the sum of values and in the sum that it is divided by."""
    want, _, allowed, _ = ref.attention(q, k, v, scale, v_scale)
    if q.dtype != f32:
        allowed = allowed + 2.02 * torch.finfo(q.dtype).eps / 2 * ref.attention(q, k, v.abs(), scale, v_scale)[0]
    return want, allowed


def check(q, c, counts, out, *, scale=None, rows=None, lengths=None):
    """`rows`: of each sequence, which of its rows are looked at (None: all)."""
    scale = 1.0 / math.sqrt(c.d) if scale is None else scale
    out, at = out.cpu().double(), 0
    for b, n in enumerate(c.lengths if lengths is None else lengths):
        k, v = (c.rows(cache, b, n).double() for cache in (c.k_cache, c.v_cache))
        for i in range(counts[b]) if rows is None else sorted({r % counts[b] for r in rows} if counts[b] else ()):
            seen = max(n - counts[b] + i + 1, 0)
            want, allowed = statement(q[at + i].cpu(), k[:, :seen] * c.k_scale, v[:, :seen], scale, c.v_scale)
            bad = ~((out[at + i] - want).abs() <= allowed)
            assert not bad.any(), (b, n, i, float(((out[at + i] - want).abs() / allowed).max()))
        at += counts[b]


def run(c, counts, H, seed=0, **options):
    q = queries(counts, H, c.d, c.dtype, seed)
    scales = {"k_scale": c.k_scale, "v_scale": c.v_scale} if c.dtype == e4m3 else {}
    return q, ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of(counts), **scales, **options)


RAGGED = [0, 1, 17, 64, 65, 130, 200, 33]
COUNTS = [0, 1, 17, 3, 65, 30, 129, 0]
SOME = (0, 1, 2, 15, 16, 31, 32, 63, 64, -1, -2)


@pytest.mark.parametrize("dtype", [bf16, f16, f32, e4m3])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("G", [1, 3])
def test_lengths_around_every_border(dtype, d, G):
    c = cache(RAGGED, 2, 16, d, dtype, seed=d, scales=(0.75, 1.5) if dtype == e4m3 else (1.0, 1.0))
    q, out = run(c, COUNTS, 2 * G)
    check(q, c, COUNTS, out, rows=SOME)


@pytest.mark.parametrize("dtype", [bf16, f16, f32, e4m3])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("counts", [[0, 1, 1, 1, 1, 1, 1, 1], [0, 1, 4, 4, 3, 2, 1, 4], [0, 0, 0, 0, 0, 1, 0, 0]])
def test_few_rows(dtype, d, counts):
    c = cache(RAGGED, 2, 16, d, dtype, seed=d, scales=(0.75, 1.5) if dtype == e4m3 else (1.0, 1.0))
    q, out = run(c, counts, 8)
    check(q, c, counts, out)


@pytest.mark.parametrize("heads,G", [(1, 1), (12, 1), (3, 5), (2, 16), (1, 17), (2, 40), (1, 200)])
def test_groups_of_heads(heads, G):
    for counts in ([9, 70], [1, 2]):
        c = cache([70, 90], heads, 32, 64, bf16, seed=G)
        q, out = run(c, counts, heads * G)
        check(q, c, counts, out, rows=SOME)


@pytest.mark.parametrize("size", [1, 7, 16, 24, 100, 1024])
@pytest.mark.parametrize("layout", ["heads", "slots"])
def test_page_sizes_and_layouts(size, layout):
    c = cache([1, size, size + 1, 310], 3, size, 96, f16, seed=size, layout=layout, room=5)
    for counts in ([1, 1, 2, 140], [1, 1, 1, 1]):
        q, out = run(c, counts, 6)
        check(q, c, counts, out, rows=SOME)


@pytest.mark.parametrize("dtype,d,pad", [(bf16, 1, 0), (bf16, 7, 0), (f16, 33, 2), (f32, 3, 0), (f32, 101, 1), (bf16, 255, 0), (f16, 72, 1), (bf16, 200, 8),
                                         (f32, 4, 0), (e4m3, 5, 0), (e4m3, 136, 0), (e4m3, 250, 3), (e4m3, 100, 0), (f32, 250, 0), (f32, 61, 0), (f16, 190, 0),
                                         (bf16, 8, 0), (bf16, 9, 0), (e4m3, 9, 1), (f32, 5, 0)])
@pytest.mark.parametrize("counts", [[5, 90, 0, 129], [1, 4, 0, 3]])
def test_odd_head_dimensions_and_row_strides(dtype, d, pad, counts):
    c = cache([5, 130, 0, 257], 2, 16, d, dtype, seed=d, pad=pad, scales=(0.5, 2.0) if dtype == e4m3 else (1.0, 1.0))
    q, out = run(c, counts, 4)
    check(q, c, counts, out, rows=SOME)


@pytest.mark.parametrize("dtype,d", [(bf16, 128), (f16, 64), (f32, 64), (e4m3, 128), (bf16, 256), (f16, 37)])
@pytest.mark.parametrize("counts", [[140, 1, 0, 7], [2, 1, 0, 4], [1500, 1, 0, 60]])
@pytest.mark.parametrize("positions", [3000, 20480])
def test_long_caches_are_split_and_joined(dtype, d, counts, positions):
    c = widened(cache([3000, 1, 0, 2222], 2, 64, d, dtype, seed=7), positions)
    q = queries(counts, 4, d, dtype, 7, size=3.0)
    assert positions == 3000 or ops.paged_attention_chunk_workspace_bytes(q, c.k_cache, c.v_cache, c.table) > 0
    out = ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of(counts))
    check(q, c, counts, out, rows=(0, 1, 63, 64, 65, 1000, -1))


@pytest.mark.parametrize("dtype,d", [(bf16, 128), (f32, 64), (e4m3, 128), (f16, 96)])
@pytest.mark.parametrize("B", [2, 20, 33, 70])
def test_pieces_among_single_tokens(dtype, d, B):
    """Sequences with few rows beside ones with many, around the number of rows (32: 8 tokens here) that parts them, up to 12 shares of positions."""
    counts = [(1, 8, 9, 0, 300, 2, 33)[b % 7] if b < 14 else b % 2 for b in range(B)]
    counts[-1] = 140
    lengths = [n + (0, 1, 64, 250, 2700, 500)[b % 6] if b < 14 else n + b for b, n in enumerate(counts)]
    c = cache(lengths, 2, 16, d, dtype, seed=B, scales=(0.75, 1.5) if dtype == e4m3 else (1.0, 1.0))
    q, out = run(c, counts, 8, seed=B)
    check(q, c, counts, out, rows=(0, 31, 32, -1))


@pytest.mark.parametrize("dtype", [bf16, f32, e4m3])
def test_only_sequences_with_few_rows_are_cut(dtype):
    counts = [300, 2, 8, 10]
    c = cache([300, 900, 1500, 700], 32, 16, 64, dtype, seed=18)
    q, out = run(c, counts, 128)
    check(q, c, counts, out, rows=(0, 3, 7, 255, -1))


@pytest.mark.parametrize("B", [30, 900, 4100])
@pytest.mark.parametrize("dtype,some", [(bf16, [1, 4, 1, 2]), (f32, [1, 4, 200, 2]), (e4m3, [1, 1, 1, 150])])
def test_most_sequences_idle(B, dtype, some):
    counts, lengths = [0] * B, [0] * B
    for b, n in zip((0, 1, B // 2, B - 1), some):
        counts[b], lengths[b] = n, n + 1100 + b % 5
    c = cache(lengths, 2, 16, 64, dtype, seed=20)
    q, out = run(c, counts, 8)
    check(q, c, counts, out, rows=(0, 1, -1))
    assert ops.paged_attention_chunk_workspace_bytes(q, c.k_cache, c.v_cache, c.table) < 16 << 20  # (256 rows, 8 shares: 1.1 MB)


@pytest.mark.parametrize("d", [128, 125])
def test_a_cache_behind_2_to_the_31_elements(d):
    """Stored there and read from there, as few rows and as many."""
    pages = 2**31 // (16 * 128) + 9
    k_cache, v_cache = (torch.zeros(pages, 1, 16, 128, dtype=bf16, device="cuda")[..., :d] for _ in range(2))
    g = torch.Generator().manual_seed(14)
    k, v = (torch.randn(40, 1, d, generator=g).to(bf16).cuda() for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 5]], dtype=torch.int32, device="cuda")
    at = torch.arange(40, device="cuda")
    ops.kv_store(k, v, k_cache, v_cache, table[0].long()[at // 16] * 16 + at % 16)
    assert torch.equal(k_cache[pages - 1, 0], k[:16, 0]) and torch.equal(v_cache[pages - 5, 0, :8], v[32:, 0])
    lengths = torch.tensor([40], dtype=torch.int32, device="cuda")
    for n in (3, 40):
        q = queries([n], 2, d, bf16, seed=n)
        out = ops.paged_attention_chunk(q, k_cache, v_cache, table, lengths, starts_of([n])).cpu().double()
        for i in range(n):
            seen = 40 - n + i + 1
            want, allowed = statement(q[i].cpu(), k[:seen, 0].cpu().double()[None], v[:seen, 0].cpu().double()[None], 1 / math.sqrt(d))
            assert ((out[i] - want).abs() <= allowed).all()


@pytest.mark.parametrize("heads,counts,lengths,d", [(20, [700, 600, 500, 300], [4200, 700, 3000, 2100], 128), (9, [800, 700], [1100, 900], 256), (36, [700, 600, 800], [4100, 900, 3500], 64)])
def test_tiles_that_nearly_fill_the_device(heads, counts, lengths, d):
    """More tiles of 128 rows than half, or a little more than all, of the workgroups that run at once: in one share or in three."""
    c = cache(lengths, heads, 64, d, bf16, seed=21)
    q, out = run(c, counts, 2 * heads)
    check(q, c, counts, out, rows=(0, 64, -1))


def test_a_whole_prompt_is_what_attention_gives():
    c = cache([700, 300], 4, 16, 64, f32, seed=3)
    counts = [700, 300]
    q, out = run(c, counts, 8)
    for b, n in enumerate(counts):
        k, v = (c.rows(cache, b, n)[:, None].expand(4, 2, n, 64).reshape(1, 8, n, 64).contiguous().cuda() for cache in (c.k_cache, c.v_cache))
        rows = slice(0, 700) if b == 0 else slice(700, 1000)
        want = ops.attention(q[rows].transpose(0, 1)[None].contiguous(), k, v, causal=True)[0].transpose(0, 1)
        assert (out[rows] - want).abs().max() < 2e-5
    # the last rows, one at a time
    last = ops.paged_attention(q[[699, 999]], c.k_cache, c.v_cache, c.table, c.device_lengths)
    assert (out[[699, 999]] - last).abs().max() < 1e-5


def test_chunks_give_what_the_whole_gives():
    c = cache([517], 2, 16, 128, bf16, seed=4)
    q, whole = run(c, [517], 8)
    at = 0
    for n in (1, 100, 3, 256, 157):
        part = ops.paged_attention_chunk(q[at:at + n], c.k_cache, c.v_cache, c.table, torch.tensor([at + n], dtype=torch.int32, device="cuda"), starts_of([n]))
        # both are off by their result's rounding and their weights', 2^-8 each of the result and of weights times values (at most 5 here)
        assert ((part.float() - whole[at:at + n].float()).abs() <= 2.0**-7 * whole[at:at + n].float().abs() + 2.0**-6).all()
        at += n


def test_rows_without_anything_to_see_and_rows_of_none():
    """More new tokens than the length counts: the first of them see nothing and become 0.  Rows behind the last sequence stay."""
    c = cache([5, 0, 70], 2, 16, 64, bf16, seed=5)
    for counts in ([9, 4, 200], [3, 2, 4]):
        lengths = torch.tensor([5, -3, 2**30], dtype=torch.int32, device="cuda")  # (clamped to 0 and to the table)
        c.device_lengths = lengths
        q = queries(counts, 4, 64, bf16, 5, spare=50)
        out = torch.full_like(q, 3.0)
        table = c.table.clone()
        got = ops.paged_attention_chunk(q, c.k_cache, c.v_cache, table, lengths, starts_of(counts), out=out)
        assert got is out and (out[sum(counts):] == 3).all()
        n = 5
        hidden = max(counts[0] - n, 0)
        assert (out[:hidden] == 0).all() and (out[counts[0]:counts[0] + counts[1]] == 0).all() and (out[hidden:counts[0]] != 0).any()
        k, v = (c.rows(cache, 0, 5).double() for cache in (c.k_cache, c.v_cache))
        want, allowed = statement(q[counts[0] - 1].cpu(), k, v, 0.125)
        assert ((out[counts[0] - 1].cpu().double() - want).abs() <= allowed).all()


@pytest.mark.parametrize("dtype,G", [(bf16, 1), (f32, 2), (e4m3, 4), (f16, 4)])
def test_pages_that_hold_nothing(dtype, G):
    """Positions on such pages are left out, wherever they lie."""
    for lengths, counts in (([200, 90], [150, 20]), ([200, 90], [2, 3])):
        c = cache(lengths, 2, 16, 64, dtype, seed=6)
        q = queries(counts, 2 * G, 64, dtype, 6)
        keep = [torch.ones(n, dtype=torch.bool) for n in lengths]
        for b, page in ((0, 0), (0, 5), (0, 12), (1, 1), (1, 2)):
            c.table[b, page] = (-1, c.pages, 2**31 - 1, -(2**31))[page % 4]
            keep[b][16 * page:16 * page + 16] = False
        out = ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of(counts)).cpu().double()
        at = 0
        for b, n in enumerate(lengths):
            k, v = (c.rows(cache, b, n).double() for cache in (c.k_cache, c.v_cache))
            for i in range(counts[b]):
                live = keep[b].clone()
                live[n - counts[b] + i + 1:] = False
                want, allowed = statement(q[at + i].cpu(), k[:, live], v[:, live], 0.125)
                assert ((out[at + i] - want).abs() <= allowed).all(), (b, i)
            at += counts[b]


@pytest.mark.parametrize("dtype", [bf16, f16, f32, e4m3])
@pytest.mark.parametrize("counts", [[150, 40], [4, 3]])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, counts, bad):
    """A key and a value of a later token hold infinities or NaN: rows before it are what they are without, rows behind it see them."""
    if dtype == e4m3:
        bad = math.nan
    lengths = [260, 45]
    c = cache(lengths, 2, 16, 64, dtype, seed=8)
    q = queries(counts, 4, 64, dtype, 8)
    call = lambda: ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of(counts))  # noqa: E731
    clean = call()
    at = lengths[0] - counts[0] // 2  # a position within the chunk
    page, slot = int(c.table[0, at // 16]), at % 16
    c.v_cache[page, 0, slot, 5] = bad
    c.v_cache[page, 1, slot, 60] = bad
    dirty = call()
    row = at - (lengths[0] - counts[0])
    assert torch.equal(dirty[:row], clean[:row]) and torch.equal(dirty[counts[0]:], clean[counts[0]:])
    hit = torch.zeros(4, 64, dtype=torch.bool, device="cuda")
    hit[:2, 5] = hit[2:, 60] = True
    assert not torch.isfinite(dirty[row:counts[0], hit]).any()
    assert torch.equal(dirty[row:counts[0], ~hit], clean[row:counts[0], ~hit])
    if dtype != e4m3:
        c.v_cache[page, 0, slot, 5] = c.v_cache[page, 1, slot, 60] = 0.0
        clean = call()
    c.k_cache[page, 0, slot, 7] = math.nan
    dirty = call()
    assert torch.equal(dirty[:row], clean[:row]) and torch.equal(dirty[row:counts[0], 2:], clean[row:counts[0], 2:]) if dtype != e4m3 else True
    assert torch.isnan(dirty[row:counts[0], :2]).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7, 1e-30])
@pytest.mark.parametrize("dtype", [bf16, f32, e4m3])
def test_scales_of_any_sign(scale, dtype):
    for counts in ([20, 50], [1, 3]):
        c = cache([90, 50], 2, 16, 64, dtype, seed=9, scales=(0.5, 3.0) if dtype == e4m3 else (1.0, 1.0))
        q, out = run(c, counts, 4, scale=scale)
        check(q, c, counts, out, scale=scale, rows=SOME)


@pytest.mark.parametrize("dtype", [bf16, f16, f32])
def test_scores_far_apart_and_long_flat_rows(dtype):
    """Maxima that grow by hundreds along the row, and rows whose many small weights add up."""
    c = cache([1200], 1, 16, 64, dtype, seed=10)
    grows = torch.linspace(0.0, 40.0, 1200)
    k = c.rows(c.k_cache, 0, 1200).clone()
    k[0, :, 0] = grows.to(dtype)
    for t in range(1200):
        c.k_cache[int(c.table[0, t // 16]), 0, t % 16, 0] = grows[t].to(dtype).item()
    q = queries([130], 2, 64, dtype, 10)
    q[:, 0, 0], q[:, 1, 0] = 30.0, -30.0
    out = ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of([130]))
    check(q, c, [130], out, rows=SOME)


def test_a_table_much_wider_than_the_sequences():
    c = ref.Cache([5, 40, 129], 2, 16, 64, bf16, seed=8)
    wide = torch.full((3, 4000), -1, dtype=torch.int32, device="cuda")
    wide[:, : c.P] = c.table
    for counts in ([5, 3, 100], [1, 1, 1]):
        q = queries(counts, 2, 64, bf16, 8)
        check(q, c, counts, ops.paged_attention_chunk(q, c.k_cache, c.v_cache, wide, c.device_lengths, starts_of(counts)), rows=SOME)


def test_many_sequences():
    lengths = [(7 * b) % 50 + 1 for b in range(300)]
    counts = [min(n, (3 * b) % 5) for b, n in enumerate(lengths)]
    c = cache(lengths, 1, 8, 32, bf16, seed=11)
    q, out = run(c, counts, 2)
    check(q, c, counts, out)
    c = cache([1] * 5000, 1, 1, 8, f32, seed=12)
    q, out = run(c, [1] * 5000, 1)
    want = c.v[:, 0, 0]  # p v / p: a rounding of each product and of the quotient
    assert ((out[:, 0].cpu() - want).abs() <= 4 * 2.0**-24 * want.abs()).all()


def test_strided_queries_and_results():
    c = cache([100, 33], 2, 16, 64, bf16, seed=13)
    counts = [60, 5]
    qkv = queries(counts, 10, 64, bf16, 13)
    store = torch.full((65, 7, 70), 5.0, dtype=bf16, device="cuda")
    out = store[:, 2:6, 3:67]
    ops.paged_attention_chunk(qkv[:, 3:7], c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of(counts), out=out)
    check(qkv[:, 3:7], c, counts, out, rows=SOME)
    store[:, 2:6, 3:67] = 5.0
    assert (store == 5).all()


@pytest.mark.parametrize("counts", [[2000, 1, 40], [300, 1, 40], [4, 1, 2]])
def test_the_result_may_take_the_place_of_the_queries(counts):
    c = cache([2300, 700, 900], 2, 16, 64, bf16, seed=19)
    q, want = run(c, counts, 8)
    got = ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of(counts), out=q)
    assert got is q and torch.equal(q, want)


def test_starts_that_make_no_sense_stay_within_the_rows():
    c = cache([100, 33, 50], 2, 16, 64, bf16, seed=14)
    q = queries([90], 4, 64, bf16, 14)
    for starts in ([5, 3, 2000, -7], [-5, 2**31 - 1, -(2**31), 90], [0, 0, 0, 0], [90, 90, 90, 90]):
        out = torch.empty_like(q)
        ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    torch.cuda.synchronize()


def test_results_repeat_themselves_and_graphs_have_workspaces_of_their_own():
    cs = [cache([3000, 100], 2, 16, 128, bf16, seed=15 + i) for i in range(2)]
    counts = [5, 3]
    qs = [queries(counts, 8, 128, bf16, 15 + i) for i in range(2)]
    starts = starts_of(counts)
    call = lambda i: ops.paged_attention_chunk(qs[i], cs[i].k_cache, cs[i].v_cache, cs[i].table, cs[i].device_lengths, starts)  # noqa: E731
    for i in range(2):
        assert torch.equal(call(i), call(i))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(i))
    g = torch.Generator(device="cuda").manual_seed(16)
    for _ in range(4):
        for i in range(2):
            qs[i].copy_(torch.randn(qs[i].shape, device="cuda", generator=g))
        graphs[0].replay()
        graphs[1].replay()
        wants = [call(0), call(1)]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1])
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, wants[i]) for i in range(2) for x in got[i])


def test_a_workspace_of_the_caller():
    c = cache([3000], 2, 16, 64, f16, seed=17)
    q = queries([2], 4, 64, f16, 17)
    need = ops.paged_attention_chunk_workspace_bytes(q, c.k_cache, c.v_cache, c.table)
    store = torch.full((need + 256,), 77, dtype=torch.uint8, device="cuda")
    at = -store.data_ptr() % 256
    ws = store[at:at + need]
    want = ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of([2]))
    got = ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of([2]), workspace=ws)
    assert torch.equal(got, want) and (store[at + need:] == 77).all() and (store[:at] == 77).all()
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_attention_chunk(q, c.k_cache, c.v_cache, c.table, c.device_lengths, starts_of([2]), workspace=ws[:-256])
