"""What the operators on packed tokens launch at the limits of their sizes, on any machine: launches within what a device takes (fewer than 2^32
threads), or a refusal.  The calls run on a recorder in the place of the HIP runtime, in a process of its own."""

import math
import multiprocessing
import random
import struct

import pytest

from tests import recorded_launches as rec

BF16, F32, E4M3 = rec._lib.BF16, rec._lib.F32, rec._lib.F8E4M3
K, V, TABLE, Q, OUT, LENGTHS, STARTS, WORKSPACE = (n << 50 for n in range(1, 9))  # far apart, aligned


@pytest.fixture(scope="module")
def recorded(tmp_path_factory):
    """recorded(check, *args): check(recorder, *args) in a process whose library launches nothing."""
    so = rec.build(tmp_path_factory.mktemp("recorder"))
    with multiprocessing.get_context("spawn").Pool(1) as pool:
        yield lambda check, *args: pool.apply(_on_recorder, (so, check, args))


_recorder = None


def _on_recorder(so, check, args):
    global _recorder
    _recorder = _recorder or rec.Recorder(so)
    return check(_recorder, *args)


def _cache(heads, d, positions, size=16, dtype=BF16, pad=0, pages=64):
    row, columns = d + pad, -(-positions // size)
    strides = (heads * size * row, size * row, row)
    return struct.pack(rec._lib.PAGED_CACHE_FORMAT, K, V, TABLE, columns, *strides, *strides, pages, columns, size, heads, d, dtype, 1.0, 1.0)


def _within(launches):
    return all(launch.grid > 0 and launch.grid * launch.block < 2**32 for launch in launches)


def _chunk(r, cache, N, B, H, d, dtype=BF16):
    need = r.lib.lh_hip_paged_attention_chunk_workspace_bytes(cache, N, B, H)
    rc, launches = r.calls("lh_hip_paged_attention_chunk", cache, OUT, Q, H * d, d, H * d, d, LENGTHS, STARTS, N, B, H, 0.1, dtype, WORKSPACE if need else None,
                           need, None)
    return rc, launches, r.lib.lh_hip_last_error().decode()


def _few_tokens_among_many_sequences(r):
    for B in (2**12, 2**12 + 1, 2**16, 2**18, 2**20 - 1):
        for N in (1, 8, 300):
            for positions in (16, 16384, 2**20, 2**30):
                rc, launches, said = _chunk(r, _cache(8, 128, positions), N, B, 8, 128)
                assert rc == 0 and launches and _within(launches), (B, N, positions, said, [(x.grid, x.block) for x in launches])


def test_few_tokens_among_many_sequences(recorded):
    """Above 4096 sequences idle ones have workgroups, too: the shares of positions are as many as a launch has room for."""
    recorded(_few_tokens_among_many_sequences)


def _attention_of_any_size(r):
    rng = random.Random(3)
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi))))  # noqa: E731
    refused = 0
    for _ in range(20000):
        heads, G, B, N = log(1, 300), log(1, 64), log(1, 2**20), log(1, 2**29)
        dtype, d = rng.choice([BF16, F32, E4M3]), rng.choice([64, 96, 128, 200, 256])
        rc, launches, said = _chunk(r, _cache(heads, d, log(1, 2**24), dtype=dtype), N, B, heads * G, d, BF16 if dtype == E4M3 else dtype)
        case = (heads, G, B, N, dtype, d, said)
        if rc == 0:
            assert launches and _within(launches), case
        else:
            refused += 1
            sizes = N * heads * G >= 2**32 or N * G >= 2**31 - 256
            assert "bad sizes" in said if sizes else ("too many rows" in said or "bad sizes" in said) and (N * G / 16 + B) * heads >= 2**24, case
    assert 1000 < refused < 15000


def test_attention_of_any_size_is_launched_or_refused(recorded):
    recorded(_attention_of_any_size)


def _one_workspace_for_caches_of_any_strides(r):
    """Sized with rows that are padded and pages of any size, for calls on contiguous ones, and the other way round."""
    rng = random.Random(6)
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi))))  # noqa: E731
    for _ in range(10000):
        heads, G, B, N = log(1, 32), log(1, 16), log(1, 200), log(1, 4096)
        dtype, d = rng.choice([BF16, F32, E4M3]), rng.choice([64, 96, 128, 200, 256, 100, 37])
        size = rng.choice([16, 48, 128])
        positions = size * log(1, 2**17 // size)
        caches = [_cache(heads, d, positions, size=size, dtype=dtype, pad=pad) for pad in (0, 1, 8)]
        needs = {r.lib.lh_hip_paged_attention_chunk_workspace_bytes(cache, N, B, heads * G) for cache in caches}
        assert len(needs) == 1, (heads, G, B, N, dtype, d, size, positions, needs)
        need = needs.pop()
        for cache in caches:
            rc, _ = r.calls("lh_hip_paged_attention_chunk", cache, OUT, Q, heads * G * d, d, heads * G * d, d, LENGTHS, STARTS, N, B, heads * G, 0.1,
                            BF16 if dtype == E4M3 else dtype, WORKSPACE if need else None, need, None)
            assert rc == 0, (heads, G, B, N, dtype, d, size, positions, need, r.lib.lh_hip_last_error())


def test_one_workspace_for_caches_of_any_strides(recorded):
    recorded(_one_workspace_for_caches_of_any_strides)


def _norms_of_any_size(r):
    """Rows of up to 512 and 1024 columns are four a workgroup, others one."""
    for C in (1, 512, 513, 1024, 1025, 2048, 2049, 4096, 8192, 8193, 16384, 16385, 2**29):
        for M in (1, 5, 2**22 - 5, 2**22, 2**24 - 1, 2**24 + 3, 2**26 - 1, 2**26, 2**26 + 1, 2**31 - 1):
            for x_dtype, residual, out_dtype, scales in ((BF16, None, BF16, None), (F32, Q, F32, None), (BF16, Q, E4M3, STARTS)):
                rc, launches = r.calls("lh_hip_rms_norm", OUT, K, V, residual, residual, scales, 1.0, M, C, C, C, C, C, 1e-5, x_dtype, x_dtype, out_dtype, None)
                case = (C, M, x_dtype, out_dtype, r.lib.lh_hip_last_error(), [(x.grid, x.block) for x in launches])
                assert rc == 0 and _within(launches), case
                rows = 4 if C <= 1024 else 1
                assert sum(x.grid for x in launches) == -(-M // rows) and len(launches) == 1 + (M - 1) // (2**32 * rows // launches[0].block - 4), case


def test_norms_of_any_size(recorded):
    recorded(_norms_of_any_size)


def _turns_and_pages_of_any_size(r):
    rng = random.Random(4)
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi))))  # noqa: E731
    turn = struct.pack(rec._lib.ROTARY_FORMAT, LENGTHS, STARTS, 2, 0, 1.0)
    for _ in range(5000):
        N, H, d = log(1, 2**31 - 1), log(1, 2**20 - 1), rng.randint(2, 256)
        rc, launches = r.calls("lh_hip_rotary", OUT, Q, H * d, d, H * d, d, turn, N, H, d, BF16, None)
        assert (rc == 0 and launches and _within(launches)) or N * H * (d + 30) >= 2**34, (N, H, d)
        rc, launches = r.calls("lh_hip_kv_store", _cache(8, d, 16), Q, Q, 8 * d, d, 8 * d, d, LENGTHS, OUT, Q, H * d, d, H * d, d, turn, N, H, BF16, None)
        assert (rc == 0 and launches and _within(launches)) or N * (H + 16) * (d + 30) >= 2**34, (N, H, d)
        B, N = log(1, 2**20 - 1), log(1, 2**30 - 1)
        rc, launches = r.calls("lh_hip_kv_pages", TABLE, 4, LENGTHS, LENGTHS, LENGTHS, K, V, STARTS, OUT, Q, B, 4, 1000, 16, N, None)
        assert rc == 0 and launches and _within(launches), (B, N)


def test_turns_and_pages_of_any_size(recorded):
    recorded(_turns_and_pages_of_any_size)


def _stores_without_a_table(r):
    for table, stride, columns in ((0, 0, 0), (0, 0, 2**31), (TABLE, 1, 4)):
        cache = struct.pack(rec._lib.PAGED_CACHE_FORMAT, K, V, table, stride, *(2048, 1024, 64), *(2048, 1024, 64), 9, columns, 16, 2, 64, BF16, 1.0, 1.0)
        rc, launches = r.calls("lh_hip_kv_store", cache, Q, Q, 128, 64, 128, 64, LENGTHS, None, None, 0, 0, 0, 0, None, 5, 0, BF16, None)
        assert rc == 0 and len(launches) == 1, (table, columns, r.lib.lh_hip_last_error())
        if not table:  # (what reads one still asks for it)
            assert r.calls("lh_hip_paged_attention_chunk", cache, OUT, Q, 128, 64, 128, 64, LENGTHS, STARTS, 5, 1, 2, 0.1, BF16, None, 0, None)[0] != 0


def test_stores_read_no_table(recorded):
    recorded(_stores_without_a_table)
