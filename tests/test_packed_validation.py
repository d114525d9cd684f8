"""The operators on packed tokens refuse mismatched calls before any device work (host side; no GPU needed): what is well formed gets as
far as the device check."""

import ctypes
import math

import pytest
import torch

from lighthouse_amd import _lib, ops

bf16, f32, f16, e4m3, i32, i64, f64 = torch.bfloat16, torch.float32, torch.float16, torch.float8_e4m3fn, torch.int32, torch.int64, torch.float64
ON_GPU = "expected tensors on the GPU"


def z(*shape, dtype=f32):
    return torch.zeros(*shape, dtype=dtype)


def refused(match, call, *args, **options):
    with pytest.raises(ValueError, match=match):
        call(*args, **options)


def test_kv_pages_rejections():
    table, n, free, one = z(3, 4, dtype=i32), z(3, dtype=i32), z(12, dtype=i32), z(1, dtype=i32)
    call = ops.kv_pages
    refused(ON_GPU, call, table, n, n, free, one, 16, 8)
    refused(ON_GPU, call, table, n, n, free, one, 16, 0, out=n)
    refused("block_table must be", call, table.long(), n, n, free, one, 16, 8)
    refused("block_table must be", call, table[0], n, n, free, one, 16, 8)
    refused("block_table must be", call, table[:, :0], n, n, free, one, 16, 8)
    refused("innermost stride", call, z(4, 3, dtype=i32).t(), n, n, free, one, 16, 8)
    refused("rows of block_table overlap", call, z(1, 4, dtype=i32).expand(3, 4), n, n, free, one, 16, 8)
    refused("lengths must be", call, table, n[:2], n, free, one, 16, 8)
    refused("lengths must be", call, table, n.long(), n, free, one, 16, 8)
    refused("counts must be", call, table, n, z(4, dtype=i32), free, one, 16, 8)
    refused("counts must be", call, table, n, z(3), free, one, 16, 8)
    refused("free_pages", call, table, n, n, free.long(), one, 16, 8)
    refused("free_pages", call, table, n, n, free[:0], one, 16, 8)
    refused("free_pages", call, table, n, n, free.view(3, 4), one, 16, 8)
    refused("free_pages", call, table, n, n, free[::2], one, 16, 8)
    refused("n_free", call, table, n, n, free, n, 16, 8)
    refused("n_free", call, table, n, n, free, one.long(), 16, 8)
    refused("positions", call, table, n, n, free, one, 0, 8)
    refused("positions", call, table, n, n, free, one, 2**30, 8)
    refused("tokens", call, table, n, n, free, one, 16, -1)
    refused("tokens", call, table, n, n, free, one, 16, 2**30)
    refused("out must be", call, table, n, n, free, one, 16, 8, out=n.long())


def test_rotary_rejections():
    x, at, f = z(5, 3, 8, dtype=bf16), z(5, dtype=i32), z(4, dtype=f64)
    call = ops.rotary
    refused(ON_GPU, call, x, at, f)
    refused(ON_GPU, call, x, at, f[:1], interleaved=True, amplitude=2.0, out=x)
    refused("x must be", call, x[0], at, f)
    refused("x must be", call, x.double(), at, f)
    refused("x must be", call, x.to(e4m3), at, f)
    refused("innermost stride", call, z(5, 8, 3).transpose(1, 2), at, f)
    refused("positions", call, x, at[:4], f)
    refused("positions", call, x, at.long(), f)
    refused("freqs", call, x, at, f.float())
    refused("freqs", call, x, at, z(5, dtype=f64))
    refused("freqs", call, x, at, f[:0])
    refused("freqs", call, x, at, z(8, dtype=f64)[::2])
    refused("freqs", call, z(5, 3, 1), at, f)
    refused("shape and dtype", call, x, at, f, out=z(5, 3, 8))
    refused("shape and dtype", call, x, at, f, out=z(5, 3, 9, dtype=bf16))
    refused("rows of out overlap", call, x, at, f, out=z(5, 1, 8, dtype=bf16).expand(5, 3, 8))
    refused("rows of out overlap", call, x, at, f, out=z(1, 3, 8, dtype=bf16).expand(5, 3, 8))
    refused("rows of out overlap", call, x, at, f, out=torch.as_strided(z(500, dtype=bf16), (5, 3, 8), (8, 16, 1)))
    refused("innermost stride", call, x, at, f, out=z(5, 8, 3, dtype=bf16).transpose(1, 2))
    refused(ON_GPU, call, x, at, f, out=z(3, 5, 8, dtype=bf16).transpose(0, 1))
    for bad in (0, 3, -2):
        refused("even number", ops.rotary_frequencies, bad, device="cpu")
    refused("positive", ops.rotary_frequencies, 8, base=0.0, device="cpu")
    refused("positive", ops.rotary_frequencies, 8, factor=-1.0, device="cpu")
    refused("positive", ops.rotary_frequencies, 8, context=100, low=4.0, high=4.0, device="cpu")


def test_kv_store_rejections():
    k = z(5, 2, 8, dtype=bf16)
    cache, slots, at, f = z(6, 2, 4, 8, dtype=bf16), z(5, dtype=i64), z(5, dtype=i32), z(4, dtype=f64)
    q = z(5, 6, 8, dtype=bf16)
    turn = {"positions": at, "freqs": f}
    call = ops.kv_store
    refused(ON_GPU, call, k, k, cache, cache, slots)
    refused(ON_GPU, call, k, k, cache, cache, slots, q=q, q_out=q, **turn)
    refused(ON_GPU, call, k.float(), k.float(), cache.to(e4m3), cache.to(e4m3), slots, k_scale=2.0)
    refused("k must be", call, k[0], k[0], cache, cache, slots)
    refused("same shape", call, k, k[:, :1], cache, cache, slots)
    refused("same shape", call, k, k.float(), cache, cache, slots)
    refused("innermost stride", call, k, z(5, 8, 2, dtype=bf16).transpose(1, 2), cache, cache, slots)
    refused("heads of 8", call, k[:, :1], k[:, :1], cache, cache, slots)
    refused("heads of 7", call, k[..., :7], k[..., :7], cache, cache, slots)
    refused("cache's dtype", call, k.float(), k.float(), cache, cache, slots)
    refused("belong to a cache", call, k, k, cache, cache, slots, k_scale=2.0)
    refused("positive", call, k, k, cache.to(e4m3), cache.to(e4m3), slots, v_scale=math.nan)
    refused("same shape", call, k, k, cache, cache[:5], slots)
    refused("slots", call, k, k, cache, cache, slots.int())
    refused("slots", call, k, k, cache, cache, slots[:4])
    refused("slots", call, k, k, cache, cache, z(10, dtype=i64)[::2])
    refused("go together", call, k, k, cache, cache, slots, positions=at)
    refused("go together", call, k, k, cache, cache, slots, freqs=f)
    refused("positions", call, k, k, cache, cache, slots, positions=at[:3], freqs=f)
    refused("freqs", call, k, k, cache, cache, slots, positions=at, freqs=z(5, dtype=f64))
    refused("to be turned", call, k, k, cache, cache, slots, q=q)
    refused("q_out needs q", call, k, k, cache, cache, slots, q_out=q, **turn)
    refused("q must have", call, k, k, cache, cache, slots, q=q[:4], **turn)
    refused("q must have", call, k, k, cache, cache, slots, q=q[..., :6], **turn)
    refused("q must have", call, k, k, cache, cache, slots, q=q.float(), **turn)
    refused("q must be", call, k, k, cache, cache, slots, q=q[0], **turn)
    refused("q_out must have", call, k, k, cache, cache, slots, q=q, q_out=q.float(), **turn)
    refused("rows of q_out", call, k, k, cache, cache, slots, q=q, q_out=z(1, 6, 8, dtype=bf16).expand(5, 6, 8), **turn)


def test_paged_attention_chunk_rejections():
    k, table = z(6, 2, 4, 8, dtype=bf16), z(3, 2, dtype=i32)
    q, n, s = z(7, 4, 8, dtype=bf16), z(3, dtype=i32), z(4, dtype=i32)
    call = ops.paged_attention_chunk
    refused(ON_GPU, call, q, k, k, table, n, s)
    refused(ON_GPU, call, q, k.to(e4m3), k.to(e4m3), table, n, s, k_scale=0.5, v_scale=2.0)
    refused("q must be", call, q[0], k, k, table, n, s)
    refused("q must be", call, q.to(e4m3), k.to(e4m3), k.to(e4m3), table, n, s)
    refused("head dimension", call, q[..., :7], k, k, table, n, s)
    refused("no multiple", call, q[:, :3], k, k, table, n, s)
    refused("no multiple", call, q[:, :0], k, k, table, n, s)
    refused("cache's dtype", call, q.float(), k, k, table, n, s)
    refused("cache's dtype", call, q.float(), k.to(e4m3), k.to(e4m3), table, n, s)
    refused("lengths", call, q, k, k, table, n[:2], s)
    refused("lengths", call, q, k, k, table, n.long(), s)
    refused("starts", call, q, k, k, table, n, n)
    refused("starts", call, q, k, k, table, n, s.long())
    refused("block_table", call, q, k, k, table.long(), n, s)
    refused("same shape", call, q, k, k[:5], table, n, s)
    refused("shape and dtype", call, q, k, k, table, n, s, out=z(7, 4, 8))
    refused("rows of out overlap", call, q, k, k, table, n, s, out=z(7, 1, 8, dtype=bf16).expand(7, 4, 8))
    refused("innermost stride", call, z(7, 8, 4, dtype=bf16).transpose(1, 2), k, k, table, n, s)
    wide = z(3, 4000, dtype=i32)
    assert ops.paged_attention_chunk_workspace_bytes(q, k, k, wide) > 0
    assert ops.paged_attention_chunk_workspace_bytes(q, k, k, table) == 0


def test_rms_norm_rejections():
    x, g, r = z(4, 16, dtype=bf16), z(16), z(4, 16)
    call = ops.rms_norm
    refused(ON_GPU, call, x, g)
    refused(ON_GPU, call, x, g, residual=r, residual_out=r, out_dtype=e4m3, scale=0.5)
    refused(ON_GPU, call, x, g, residual=x, out_dtype=e4m3, row_scales=z(4))
    refused(ON_GPU, call, x, g, out=x)
    refused(r"\[M, C\]", call, x[0], g)
    refused(r"\[M, C\]", call, x.double(), g)
    refused(r"\[M, C\]", call, x[:, :0], g[:0])
    refused("gamma", call, x, g[:8])
    refused("gamma", call, x, g.to(bf16))
    refused("x: innermost stride", call, z(16, 4).t(), g)
    refused("x: rows overlap", call, z(1, 16).expand(4, 16), g)
    refused("out must be torch", call, x, g, out=r, out_dtype=bf16)
    refused("out must be float32", call, x, g, out_dtype=f64)
    refused("out must have", call, x, g, out=z(4, 17))
    refused("out: rows overlap", call, x, g, out=z(1, 16).expand(4, 16))
    refused("residual must have", call, x, g, residual=r[:3])
    refused("residual must be", call, x, g, residual=r.to(f16))
    refused("residual_out must have the dtype", call, x, g, residual=r, residual_out=x)
    refused("residual_out must have shape", call, x, g, residual=r, residual_out=r[:3])
    refused("needs residual", call, x, g, residual_out=r)
    refused("scale belongs", call, x, g, scale=0.5)
    for bad in (0.0, -1.0, math.inf, math.nan):
        refused("scale belongs", call, x, g, out_dtype=e4m3, scale=bad)
    refused("row_scales", call, x, g, out_dtype=e4m3, row_scales=z(3))
    refused("row_scales", call, x, g, row_scales=z(4))
    refused("row_scales", call, x, g, out_dtype=e4m3, scale=1.0, row_scales=z(4))


def test_the_entry_points_check_for_themselves():
    lib = _lib.load()
    p = ctypes.create_string_buffer(4096)
    at = ctypes.addressof(p)

    def says(text, rc):
        assert rc == _lib.LH_ERR_INVALID and text in lib.lh_hip_last_error().decode()

    pages = lambda **o: lib.lh_hip_kv_pages(*({"table": at, "stride": 4, "lengths": at, "counts": at, "out": at, "free": at, "n": at, "starts": at, "pos": at, "slots": at,  # noqa: E731
                                               "B": 2, "P": 4, "pages": 9, "size": 16, "N": 3} | o).values(), None)
    says("null pointer", pages(table=None))
    says("null pointer", pages(slots=None))
    says("overlap", pages(stride=3))
    says("bad page counts", pages(size=0))
    says("bad page counts", pages(P=2**27))
    says("bad counts", pages(B=2**20))
    says("bad counts", pages(N=-1))
    turn = lambda turned=8: ops._PACK_ROTARY(at, at, turned, 0, 1.0)  # noqa: E731
    says("cannot turn", lib.lh_hip_rotary(at, at, 8, 8, 8, 8, turn(7), 1, 1, 8, _lib.BF16, None))
    says("cannot turn", lib.lh_hip_rotary(at, at, 8, 8, 8, 8, turn(10), 1, 1, 8, _lib.BF16, None))
    says("null pointer", lib.lh_hip_rotary(None, at, 8, 8, 8, 8, turn(), 1, 1, 8, _lib.BF16, None))
    says("unsupported", lib.lh_hip_rotary(at, at, 8, 8, 8, 8, turn(), 1, 1, 8, _lib.F8E4M3, None))
    says("bad sizes", lib.lh_hip_rotary(at, at, 8, 8, 8, 8, turn(), -1, 1, 8, _lib.BF16, None))
    cache = ops._PACK_CACHE(at, at, at, 2, 64, 32, 8, 64, 32, 8, 4, 2, 4, 2, 8, _lib.BF16, 1.0, 1.0)
    says("to be turned", lib.lh_hip_kv_store(cache, at, at, 16, 8, 16, 8, at, at, at, 8, 8, 8, 8, None, 1, 1, _lib.BF16, None))
    says("cache's dtype", lib.lh_hip_kv_store(cache, at, at, 16, 8, 16, 8, at, None, None, 0, 0, 0, 0, None, 1, 0, _lib.F16, None))
    says("null pointer", lib.lh_hip_kv_store(cache, at, at, 16, 8, 16, 8, None, None, None, 0, 0, 0, 0, None, 1, 0, _lib.BF16, None))
    chunk = lambda H=4, N=3, B=2, scale=1.0, dtype=_lib.BF16, q=at: lib.lh_hip_paged_attention_chunk(cache, at, q, 32, 8, 32, 8, at, at, N, B, H, scale, dtype, None, 0, None)  # noqa: E731
    says("no multiple", chunk(H=3))
    says("bad sizes", chunk(N=2**30))
    says("bad sizes", chunk(B=2**20))
    says("cache's dtype", chunk(dtype=_lib.F16))
    says("null pointer", chunk(q=None))
    says("finite", chunk(scale=math.inf))
    says("finite", chunk(scale=math.nan))
    wide = ops._PACK_CACHE(at, at, at, 4000, 64, 32, 8, 64, 32, 8, 4, 4000, 4, 2, 8, _lib.BF16, 1.0, 1.0)
    says("workspace", lib.lh_hip_paged_attention_chunk(wide, at, at, 32, 8, 32, 8, at, at, 3, 2, 4, 1.0, _lib.BF16, None, 0, None))
    norm = lambda out=at, residual=None, after=None, scales=None, scale=1.0, C=16, xd=_lib.BF16, rd=_lib.F32, od=_lib.BF16: lib.lh_hip_rms_norm(  # noqa: E731
        out, at, at, residual, after, scales, scale, 4, C, 16, 16, 16, 16, 1e-5, xd, rd, od, None)
    says("null pointer", norm(out=None))
    says("bad sizes", norm(C=0))
    says("unsupported x", norm(xd=_lib.F8E4M3))
    says("unsupported out", norm(od=_lib.I32))
    says("place for its sum", norm(residual=at))
    says("place for its sum", norm(after=at))
    says("must be f32", norm(residual=at, after=at, rd=_lib.F16))
    says("positive scale", norm(od=_lib.F8E4M3, scale=0.0))
    says("positive scale", norm(od=_lib.F8E4M3, scale=math.nan))
    says("positive scale", norm(scales=at))


def test_the_entry_point_of_the_norm_checks_its_row_strides():
    lib = _lib.load()
    p = ctypes.create_string_buffer(4096)
    at = ctypes.addressof(p)
    norm = lambda M=4, strides=(16, 16, 16, 16), residual=at: lib.lh_hip_rms_norm(  # noqa: E731
        at, at, at, residual, residual, None, 1.0, M, 16, *strides, 1e-5, _lib.BF16, _lib.F32, _lib.BF16, None)
    for strides in ((15, 16, 16, 16), (16, 16, 16, 15)):  # (of out and residual_out)
        for M in (4, 2):
            assert norm(M, strides) == _lib.LH_ERR_INVALID and "rows of a result overlap" in lib.lh_hip_last_error().decode()
    assert norm(0, (0, 0, 0, 0)) == 0
