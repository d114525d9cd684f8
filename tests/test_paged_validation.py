"""The operators over a paged cache and sampling refuse mismatched calls before any device work (host side; no GPU needed): what
is well formed gets as far as the device check."""

import ctypes
import math

import pytest
import torch

from lighthouse_amd import _lib, ops

bf16, f32, f16, e4m3, i32 = torch.bfloat16, torch.float32, torch.float16, torch.float8_e4m3fn, torch.int32
ON_GPU = "expected tensors on the GPU"


def z(*shape, dtype=f32):
    return torch.zeros(*shape, dtype=dtype)


def cache(dtype=bf16, pages=6, heads=2, size=4, d=8):
    return z(pages, heads, size, d, dtype=dtype), z(pages, heads, size, d, dtype=dtype), z(3, 2, dtype=i32)


def refused(match, call, *args, **options):
    with pytest.raises(ValueError, match=match):
        call(*args, **options)


def test_a_cache_is_refused():
    k, v, table = cache()
    q, n = z(3, 4, 8, dtype=bf16), z(3, dtype=i32)
    call = ops.paged_attention
    refused(ON_GPU, call, q, k, v, table, n)
    refused("same shape", call, q, k, v[:5], table, n)
    refused("same shape", call, q, k[0], v[0], table, n)
    refused("one dtype", call, q, k, v.to(f16), table, n)
    refused("one dtype", call, q, k.double(), v.double(), table, n)
    refused("head dimension of 1 to 256", call, z(3, 4, 264, dtype=bf16), z(6, 2, 4, 264, dtype=bf16), z(6, 2, 4, 264, dtype=bf16), table, n)
    refused("must hold something", call, q, k[:0], v[:0], table, n)
    refused("innermost stride", call, q, z(6, 2, 8, 4, dtype=bf16).transpose(2, 3), v, table, n)
    refused("rows overlap", call, q, z(6, 2, 1, 8, dtype=bf16).expand(6, 2, 4, 8), v, table, n)
    refused("block_table", call, q, k, v, table.long(), n)
    refused("block_table", call, q, k, v, table[:2], n)
    refused("block_table", call, q, k, v, z(3, dtype=i32), n)
    refused("block_table", call, q, k, v, z(3, 0, dtype=i32), n)
    refused("innermost stride", call, q, k, v, z(2, 3, dtype=i32).t(), n)
    refused("rows of block_table overlap", call, q, k, v, z(1, 2, dtype=i32).expand(3, 2), n)
    long = z(1, 1, 2**20, 8, dtype=bf16)
    refused("positions", call, q[:, :1], long, long, z(3, 2**11, dtype=i32), n)
    refused("belong to a cache", call, q, k, v, table, n, k_scale=2.0)
    for bad in (0.0, -1.0, math.inf, math.nan, 1e39):
        refused("positive", call, q, k.to(e4m3), v.to(e4m3), table, n, v_scale=bad)
    refused(ON_GPU, call, q, k.to(e4m3), v.to(e4m3), table, n, k_scale=0.5, v_scale=2.0)


def test_kv_append_rejections():
    k, v, table = cache()
    x, at = z(3, 2, 5, 8, dtype=bf16), z(3, dtype=i32)
    refused(ON_GPU, ops.kv_append, x, x, k, v, table, at)
    refused(ON_GPU, ops.kv_append, x, x, k, v, table, at, counts=at)
    refused("same shape", ops.kv_append, x, x[:, :, :4], k, v, table, at)
    refused("same shape", ops.kv_append, x, x.to(f16), k, v, table, at)
    refused("heads of 8", ops.kv_append, x[:, :1], x[:, :1], k, v, table, at)
    refused("heads of 7", ops.kv_append, x[..., :7], x[..., :7], k, v, table, at)
    refused("cache's dtype", ops.kv_append, x.float(), x.float(), k, v, table, at)
    refused("cache's dtype", ops.kv_append, x.to(e4m3), x.to(e4m3), k.to(e4m3), v.to(e4m3), table, at)
    refused(ON_GPU, ops.kv_append, x.float(), x.float(), k.to(e4m3), v.to(e4m3), table, at)
    refused("innermost stride", ops.kv_append, z(3, 2, 8, 5, dtype=bf16).transpose(2, 3), x, k, v, table, at)
    refused("positions", ops.kv_append, x, x, k, v, table, at[:2])
    refused("positions", ops.kv_append, x, x, k, v, table, at.long())
    refused("counts", ops.kv_append, x, x, k, v, table, at, counts=z(4, dtype=i32))


def test_paged_attention_rejections():
    k, v, table = cache()
    q, n = z(3, 4, 8, dtype=bf16), z(3, dtype=i32)
    call = ops.paged_attention
    refused(r"\[B, H, d\]", call, q[0], k, v, table, n)
    refused("head dimension", call, q[..., :7], k, v, table, n)
    refused("no multiple", call, q[:, :3], k, v, table, n)
    refused("no multiple", call, q[:, :0], k, v, table, n)
    refused("cache's dtype", call, q.float(), k, v, table, n)
    refused("cache's dtype", call, q.float(), k.to(e4m3), v.to(e4m3), table, n)
    refused("unsupported|cache's dtype", call, q.to(e4m3), k.to(e4m3), v.to(e4m3), table, n)
    refused("out must have", call, q, k, v, table, n, out=z(3, 4, 8))
    refused("out must have", call, q, k, v, table, n, out=z(3, 4, 9, dtype=bf16))
    refused("rows of out overlap", call, q, k, v, table, n, out=z(3, 1, 8, dtype=bf16).expand(3, 4, 8))
    refused("innermost stride", call, z(3, 8, 4, dtype=bf16).transpose(1, 2), k, v, table, n)
    refused("lengths", call, q, k, v, table, n[:2])
    refused("lengths", call, q, k, v, table, n.long())
    refused(ON_GPU, call, q, k, v, table, n, weights=z(3, 2, 8))
    refused("weights must be", call, q, k, v, table, n, weights=z(3, 2, 7))
    refused("weights must be", call, q, k, v, table, n, weights=z(3, 4, 8))
    refused("weights must be", call, q, k, v, table, n, weights=z(3, 2, 8, dtype=bf16))
    refused("rows must not overlap", call, q, k, v, table, n, weights=z(1, 1, 8).expand(3, 2, 8))


def test_kv_evict_rejections():
    k, v, table = cache()
    w, n = z(3, 2, 8), z(3, dtype=i32)
    call = ops.kv_evict
    refused(ON_GPU, call, k, v, w, table, n, 4)
    refused(ON_GPU, call, k, v, w, table, n, 4, recent=4, out=n)
    for budget, recent in ((0, 0), (-1, 0), (4, 5), (4, -1)):
        refused("budget", call, k, v, w, table, n, budget, recent=recent)
    refused("weights must be", call, k, v, w[:, :, :7], table, n, 4)
    refused("lengths", call, k, v, w, table, n.long(), 4)
    refused("lengths", call, k, v, w, table, z(3, 1, dtype=i32), 4)
    refused("block_table", call, k, v, w, table, n[:2], 4)
    refused("out", call, k, v, w, table, n, 4, out=n.long())
    assert ops.kv_evict_workspace_bytes(k, table, 100) == ops.kv_evict_workspace_bytes(k, table, 8) >= 3 * 2 * 8 * 4


def test_sample_rejections():
    x, u = z(3, 50), z(3)
    refused(ON_GPU, ops.sample, x, u)
    refused(ON_GPU, ops.sample, x.to(bf16), u, temperature=z(3), top_k=z(3, dtype=i32), top_p=z(3), min_p=z(3))
    refused(r"\[B, V\]", ops.sample, x[0], u)
    refused(r"\[B, V\]", ops.sample, x.double(), u)
    refused(r"\[B, V\]", ops.sample, x[:, :0], u)
    refused("innermost stride", ops.sample, z(50, 3).t(), u)
    refused("rows of logits overlap", ops.sample, z(1, 50).expand(3, 50), u)
    refused("uniform must have shape", ops.sample, x, z(4))
    refused("uniform must be", ops.sample, x, u.double())
    refused("temperature must be", ops.sample, x, u, temperature=z(3, dtype=bf16))
    refused("top_k must be", ops.sample, x, u, top_k=z(3))
    refused("top_p must have shape", ops.sample, x, u, top_p=z(2))
    refused("min_p must be contiguous", ops.sample, x, u, min_p=z(6)[::2])
    refused("out must be", ops.sample, x, u, out=z(3, dtype=i32))
    for option in ("temperature", "top_p", "min_p"):
        refused(ON_GPU, ops.sample, x, u, **{option: 1e39})  # (more than a float holds: infinite)
        refused("could not convert", ops.sample, x, u, **{option: "much"})


def test_the_c_entry_points_refuse_without_a_gpu():
    lib = _lib.load()
    st = _lib.Strides3(64, 32, 8)

    def paged(**changes):
        c = _lib.PagedCache(4096, 8192, 12288, 2, st, st, 6, 2, 4, 2, 8, _lib.BF16, 1.0, 1.0)
        for name, value in changes.items():
            setattr(c, name, value)
        return ctypes.byref(c)

    def attention(c, q=4096, B=3, H=4, dtype=_lib.BF16, ws=None, size=0, weights=None):
        return lib.lh_hip_paged_attention(c, 4096, q, 32, 8, 32, 8, 4096, weights, 16, 8, B, H, 1.0, dtype, ws, size, None)

    bad = {"k": None, "block_table": None, "n_pages": 0, "max_pages": 2**30, "page_size": 0, "n_kv_heads": 0, "d": 257, "dtype": _lib.I8,
           "table_stride": 1, "k_scale": 0.0, "v_scale": math.inf, "sk": _lib.Strides3(64, 32, 7)}
    for name, value in bad.items():
        assert attention(paged(**{name: value})) == _lib.LH_ERR_INVALID, name
        assert lib.lh_hip_kv_append(paged(**{name: value}), 4096, 4096, 64, 32, 8, 64, 32, 8, 4096, None, 3, 5, _lib.BF16, None) == _lib.LH_ERR_INVALID
        assert lib.lh_hip_kv_evict(paged(**{name: value}), 4096, 16, 8, 4096, 4096, 3, 4, 0, 4096, 1 << 20, None) == _lib.LH_ERR_INVALID
        assert lib.lh_hip_paged_attention_workspace_bytes(paged(**{name: value}), 3, 4, 1) == 0
    assert attention(None) == _lib.LH_ERR_INVALID and attention(paged(), q=None) == _lib.LH_ERR_INVALID
    assert attention(paged(), H=3) == _lib.LH_ERR_INVALID and b"no multiple" in lib.lh_hip_last_error()
    assert attention(paged(), dtype=_lib.F16) == _lib.LH_ERR_INVALID
    assert attention(paged(), weights=4096) == _lib.LH_ERR_INVALID and b"workspace" in lib.lh_hip_last_error()
    long = paged(max_pages=2**20, table_stride=2**20)
    assert lib.lh_hip_paged_attention(long, 4096, 4096, 32, 8, 32, 8, 4096, 4096, 2**23, 2**22, 256, 2, 1.0, _lib.BF16, None, 0, None) == _lib.LH_ERR_INVALID
    assert b"too many weights" in lib.lh_hip_last_error()
    need = lib.lh_hip_paged_attention_workspace_bytes(paged(), 3, 4, 1)
    assert need > 0 and need % 256 == 0
    assert attention(paged(), weights=4096, ws=4096, size=need - 1) == _lib.LH_ERR_INVALID
    assert attention(paged(), weights=4096, ws=4096 + 16, size=need) == _lib.LH_ERR_INVALID
    assert lib.lh_hip_kv_append(paged(), None, 4096, 64, 32, 8, 64, 32, 8, 4096, None, 3, 5, _lib.BF16, None) == _lib.LH_ERR_INVALID
    assert lib.lh_hip_kv_append(paged(), 4096, 4096, 64, 32, 8, 64, 32, 8, 4096, None, 2**20, 2**20, _lib.BF16, None) == _lib.LH_ERR_INVALID
    assert lib.lh_hip_kv_evict(paged(), 4096, 16, 8, 4096, 4096, 3, 4, 5, 4096, 1 << 20, None) == _lib.LH_ERR_INVALID
    assert lib.lh_hip_kv_evict(paged(), 4096, 16, 7, 4096, 4096, 3, 4, 0, 4096, 1 << 20, None) == _lib.LH_ERR_INVALID
    assert lib.lh_hip_kv_evict(paged(), 4096, 16, 8, 4096, 4096, 3, 4, 0, 4096, 16, None) == _lib.LH_ERR_INVALID
    opts = _lib.SampleOpts(temperature_all=1.0, top_p_all=1.0)
    for args in ((None, 4096, 4096, 3, 50, 50, _lib.F32), (4096, 4096, 4096, 3, 0, 50, _lib.F32), (4096, 4096, 4096, 3, 50, 49, _lib.F32),
                 (4096, 4096, 4096, 3, 50, 50, _lib.F8E4M3), (4096, 4096, 4096, -1, 50, 50, _lib.F32)):
        assert lib.lh_hip_sample(*args, ctypes.byref(opts), None, 0, None) == _lib.LH_ERR_INVALID
    assert lib.lh_hip_sample(4096, 4096, 4096, 3, 50, 50, _lib.F32, None, None, 0, None) == _lib.LH_ERR_INVALID
    assert lib.lh_hip_sample(4096, 4096, 4096, 2**17, 2**19, 2**19, _lib.F32, ctypes.byref(opts), 4096, 1 << 40, None) == _lib.LH_ERR_INVALID
    assert b"bad shape" in lib.lh_hip_last_error()
    assert lib.lh_hip_sample_workspace_bytes(3, 8192) == 0
    need = lib.lh_hip_sample_workspace_bytes(3, 8193)
    for ws, size in ((None, need), (4096, need - 1), (4096 + 16, need)):
        assert lib.lh_hip_sample(4096, 4096, 4096, 3, 8193, 8193, _lib.F32, ctypes.byref(opts), ws, size, None) == _lib.LH_ERR_INVALID
        assert b"workspace" in lib.lh_hip_last_error()


def test_sizes_beyond_every_limit_need_no_workspace_and_are_refused():
    """Products of sizes that pass 64 bits do not come out as something small."""
    lib = _lib.load()
    st = _lib.Strides3(64, 32, 8)
    c = ctypes.byref(_lib.PagedCache(4096, 8192, 12288, 2, st, st, 6, 2, 4, 2, 8, _lib.BF16, 1.0, 1.0))
    opts = _lib.SampleOpts(temperature_all=1.0, top_p_all=1.0)
    for B, H in ((2**62, 4), (2**40, 2**26), (2**32, 2**32), (2**20, 2), (-3, 4), (3, -4)):
        assert lib.lh_hip_paged_attention_workspace_bytes(c, B, H, 1) == 0
        assert lib.lh_hip_paged_attention(c, 4096, 4096, 32, 8, 32, 8, 4096, None, 0, 0, B, H, 1.0, _lib.BF16, None, 0, None) == _lib.LH_ERR_INVALID
    for B, heads, budget in ((2**62, 4, 4), (2**33, 2**31, 8), (2, 2**62, 2), (2, 2, 2**62), (2**16, 1, 4)):
        assert lib.lh_hip_kv_evict_workspace_bytes(B, heads, budget) == 0
    for B in (2**62, 2**33, 2**18):
        assert lib.lh_hip_kv_evict(c, 4096, 16, 8, 4096, 4096, B, 4, 0, 4096, 1 << 40, None) == _lib.LH_ERR_INVALID
        assert lib.lh_hip_kv_append(c, 4096, 4096, 64, 32, 8, 64, 32, 8, 4096, None, B, 2**31, _lib.BF16, None) == _lib.LH_ERR_INVALID
        assert lib.lh_hip_sample_workspace_bytes(B, 20000) == 0
        assert lib.lh_hip_sample(4096, 4096, 4096, B, 20000, 20000, _lib.F32, ctypes.byref(opts), 4096, 1 << 40, None) == _lib.LH_ERR_INVALID


def test_packed_structs_are_laid_out_like_the_c_ones():
    import struct

    values = list(range(1, 18))
    packed = struct.pack(_lib.PAGED_CACHE_FORMAT, *values[:15], 2, 3.5, 4.5)
    c = _lib.PagedCache.from_buffer_copy(packed)
    assert len(packed) == ctypes.sizeof(c)
    assert [c.k, c.v, c.block_table, c.table_stride, c.sk.z, c.sk.h, c.sk.t, c.sv.z, c.sv.h, c.sv.t, c.n_pages, c.max_pages,
            c.page_size, c.n_kv_heads, c.d, c.dtype, c.k_scale, c.v_scale] == [*values[:15], 2, 3.5, 4.5]
    packed = struct.pack(_lib.SAMPLE_OPTS_FORMAT, 1, 2, 3, 4, 0.5, 6, 0.25, 0.125)
    o = _lib.SampleOpts.from_buffer_copy(packed)
    assert len(packed) == ctypes.sizeof(o)
    assert [o.temperature, o.top_k, o.top_p, o.min_p, o.temperature_all, o.top_k_all, o.top_p_all, o.min_p_all] == [1, 2, 3, 4, 0.5, 6, 0.25, 0.125]


def test_tensors_of_another_device_are_refused(monkeypatch):
    class On:
        def __init__(self, index):
            self.index, self.is_cuda, self.device = index, index >= 0, f"cuda:{index}"

        def get_device(self):
            return self.index

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    ops._on_current_device(On(0), None, On(0))
    refused("on one device", ops._on_current_device, On(0), On(1))
    refused("current device", ops._on_current_device, On(1), None, On(1))
    refused(ON_GPU, ops._on_current_device, On(-1), On(-1))
    refused(ON_GPU, ops._on_current_device, On(0), On(-1))


def test_shares_of_the_widest_tables():
    """Positions of the table and of a share add up to more than 2^31: there are as many shares all the same."""
    lib = _lib.load()
    size, pages = 65536, 32766
    st = _lib.Strides3(size * 64, size * 64, 64)
    c = _lib.PagedCache(4096, 8192, 12288, pages, st, st, 2, pages, size, 1, 64, _lib.BF16, 1.0, 1.0)
    per_share = 64 * 4 + 8  # sums of a head, maximum and sum
    need = lib.lh_hip_paged_attention_workspace_bytes(ctypes.byref(c), 1, 1, 0)
    assert need >= 1024 * per_share and need <= 4096 * per_share
    # With heads for every CU a share is the table, and nothing is joined.
    assert lib.lh_hip_paged_attention_workspace_bytes(ctypes.byref(c), 2**14, 1, 0) == 0


@pytest.mark.parametrize("B,heads,d,size,pages,dtype", [(4, 8, 128, 16, 256, _lib.F16), (32, 1, 128, 16, 256, _lib.BF16), (1, 12, 64, 16, 63, _lib.BF16),
                                                        (2, 2, 256, 64, 100, _lib.F32), (3, 4, 128, 32, 700, _lib.F8E4M3)])
@pytest.mark.parametrize("weights", [0, 1])
def test_a_workspace_serves_a_cache_of_any_alignment(B, heads, d, size, pages, dtype, weights):
    """Sized with keys and values at multiples of 16 bytes, it holds a call with a view that begins elsewhere, and the other way round."""
    lib = _lib.load()
    st = _lib.Strides3(heads * size * d, size * d, d)
    need = [lib.lh_hip_paged_attention_workspace_bytes(ctypes.byref(_lib.PagedCache(4096 + k, 8192 + v, 12288, pages, st, st, 9, pages, size, heads, d, dtype, 1.0, 1.0)),
                                                       B, 4 * heads, weights) for k, v in ((0, 0), (8, 0), (0, 8), (8, 8))]
    assert len(set(need)) == 1 and need[0] % 256 == 0


def test_kv_evict_refuses_a_workspace_that_is_not_aligned():
    lib = _lib.load()
    st = _lib.Strides3(64, 32, 8)
    c = ctypes.byref(_lib.PagedCache(4096, 8192, 12288, 2, st, st, 6, 2, 4, 2, 8, _lib.BF16, 1.0, 1.0))
    need = lib.lh_hip_kv_evict_workspace_bytes(3, 2, 4)
    for ws in (4096 + 1, 4096 + 4, 4096 + 128):
        assert lib.lh_hip_kv_evict(c, 4096, 16, 8, 4096, 4096, 3, 4, 0, ws, need, None) == _lib.LH_ERR_INVALID
        assert b"aligned" in lib.lh_hip_last_error()
