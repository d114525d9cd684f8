"""Torch-tensor front end of the C ABI: launches on torch's current stream, no allocation
except outputs the caller did not pass.  Used by the torch ingress path, the benchmark and
the tests; every function goes straight to liblighthouse_hip.so.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _lib
from .utils.numpy import lh_dtype


def _stream() -> int:
    """Raw handle of torch's current stream on the current device (the accessors torch's own
    extensions use: no Stream object is built per launch; torch is up, the call's tensors are on the GPU)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _need_cuda(*tensors) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("expected tensors on the GPU")


# The C side sees pointers and sizes only, so everything it cannot check is checked here, before
# any device work: a mismatched call must raise, not read or write outside a buffer.
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _tuned_db():
    """The active tuned-parameter database (None when there is none); the import is deferred so that
    loading this module does not read the database file."""
    global _active_db
    if _active_db is None:
        from .tuning.tile_db import active_db

        _active_db = active_db
    return _active_db()


_active_db = None
_DTYPE_NAMES = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}


def _rows_aligned16(*tensors) -> bool:
    """Base address and every stride but the innermost are multiples of 16 bytes."""
    for t in tensors:
        if t is None:
            continue
        per = 16 // t.element_size()
        if t.data_ptr() % 16 or any(s % per for s in t.stride()[:-1]):
            return False
    return True


def _is_matrix(t, rows, cols, what: str) -> None:
    if t.shape != (rows, cols):
        raise ValueError(f"{what} must have shape [{rows}, {cols}], got {tuple(t.shape)}")
    if t.stride(1) != 1 and cols != 1:
        raise ValueError(f"{what}: innermost stride must be 1")
    if t.stride(0) < cols and rows != 1:
        raise ValueError(f"{what}: rows overlap (stride {t.stride(0)} < {cols} columns)")


def _is_vector(t, n, dtype, what: str) -> None:
    if t.shape != (n,):
        raise ValueError(f"{what} must have shape [{n}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if t.stride(0) != 1 and n != 1:
        raise ValueError(f"{what} must be contiguous")


def _same_dense(out, x, what: str) -> None:
    if out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError(f"{what}: out must have the shape and dtype of the input ({tuple(x.shape)}, {x.dtype})")
    if not x.is_contiguous() or not out.is_contiguous():
        raise ValueError(f"{what} expects contiguous tensors")


def device_info() -> dict:
    info = _lib.DeviceInfo()
    _lib.check(_lib.load().lh_hip_device_info(ctypes.byref(info)), "device_info")
    return {
        "arch": info.arch.decode(), "name": info.name.decode(), "compute_units": info.compute_units,
        "clock_khz": info.clock_khz, "memory_clock_khz": info.memory_clock_khz,
        "memory_bus_bits": info.memory_bus_bits, "lds_bytes_per_cu": info.lds_bytes_per_cu,
        "wavefront_size": info.wavefront_size, "hbm_bytes": info.hbm_bytes,
    }


def gemm(a, b, bias=None, *, out=None, out_dtype=None, relu=False, gelu=False, accumulate_c=False,
         transpose_a=False, transpose_b=False, tile=None, split_k=None, residual=None, workspace=None):
    """out = epilogue(A @ B); see lh_hip_gemm.  `tile=(bm, bn)` requests a workgroup tile and
    `split_k` (1 = never, 2 / 4 / 8) a cut along K for the 16-bit kernels (f32 inputs take the tiles
    128x128, 128x64 and 64x64 and no cut); with neither given the
    tuned-parameter database is asked, then the library's own choice applies;
    `residual` [M, N] is added to A @ B before the epilogue (lh_hip_gemm_residual) and is left intact;
    `workspace` (uint8, see gemm_workspace_bytes) makes the call take its temporary memory from
    there instead of the library's pool (lh_hip_gemm_ws)."""
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("gemm expects 2-D tensors")
    if a.stride(1) != 1 or b.stride(1) != 1:
        raise ValueError("innermost stride must be 1")
    if a.dtype not in _FLOATS:
        raise ValueError(f"unsupported A/B dtype {a.dtype}")
    if a.dtype != b.dtype:
        raise ValueError("A and B must have the same dtype")
    M, K = (a.shape[1], a.shape[0]) if transpose_a else a.shape
    N = b.shape[0] if transpose_b else b.shape[1]
    if not ((b.shape[1] if transpose_b else b.shape[0]) == K):
        raise ValueError(f"B has {b.shape[1] if transpose_b else b.shape[0]} rows of K, A has {K}")
    _require(a.stride(0) >= a.shape[1] and b.stride(0) >= b.shape[1], "rows of A or B overlap")
    if out is None:
        if accumulate_c:
            raise ValueError("accumulate_c needs an explicit out tensor")
        out = torch.empty((M, N), dtype=out_dtype or a.dtype, device=a.device)
    _is_matrix(out, M, N, "out")
    _require(out.dtype in (torch.float32, a.dtype), "out must be float32 or have the A/B dtype")
    if bias is not None:
        if bias.dtype != out.dtype:
            raise ValueError("bias must have the output dtype")
        _is_vector(bias, N, out.dtype, "bias")
    if residual is not None:
        if accumulate_c or workspace is not None:
            raise ValueError("residual excludes accumulate_c and workspace")
        if tuple(residual.shape) != (M, N) or residual.dtype != out.dtype or residual.stride(1) != 1 \
                or residual.stride(0) != out.stride(0):
            raise ValueError("residual must be an [M, N] matrix of the output dtype with the output's row stride")
    if workspace is not None:
        _require(workspace.dtype == torch.uint8 and workspace.dim() == 1 and workspace.is_contiguous(),
                 "workspace must be a contiguous uint8 vector")
    _need_cuda(a, b, bias, out, residual, workspace)
    flags = ((_lib.GEMM_HAS_BIAS if bias is not None else 0) | (_lib.GEMM_HAS_RELU if relu else 0)
             | (_lib.GEMM_HAS_GELU if gelu else 0) | (_lib.GEMM_ACCUMULATE_C if accumulate_c else 0)
             | (_lib.GEMM_TRANSPOSE_A if transpose_a else 0) | (_lib.GEMM_TRANSPOSE_B if transpose_b else 0))
    if tile is None and split_k is None and not transpose_a:  # (a transposed B runs on the same kernels in place)
        db = _tuned_db()  # tuned parameters for this shape, if the database has any
        if db is not None and db.entries:
            tile, split_k = db.lookup_gemm(_DTYPE_NAMES[a.dtype], M, N, K)
            # (a request needs aligned rows; tuned entries assume them)
            if (tile is not None or split_k is not None) and not _rows_aligned16(a, b, out, bias):
                tile = split_k = None
    if tile is not None:
        allowed = _lib.GEMM_TILES_F32 if a.dtype == torch.float32 else _lib.GEMM_TILES_16BIT
        if tuple(tile) not in allowed:
            raise ValueError(f"unsupported tile {tile} for {_DTYPE_NAMES[a.dtype]} inputs; choose from {sorted(allowed)}")
        flags |= _lib.GEMM_TILES[tuple(tile)]
    if split_k is not None:
        if a.dtype == torch.float32 and split_k != 0:
            raise ValueError("split_k applies to 16-bit inputs")
        if split_k not in _lib.GEMM_SPLITK:
            raise ValueError(f"unsupported split_k {split_k}; choose from {sorted(_lib.GEMM_SPLITK)}")
        flags |= _lib.GEMM_SPLITK[split_k]
    bias_ptr = bias.data_ptr() if bias is not None else None
    if residual is not None:
        _lib.check(_lib.load().lh_hip_gemm_residual(
            out.data_ptr(), residual.data_ptr(), a.data_ptr(), b.data_ptr(), bias_ptr, M, N, K,
            a.stride(0), b.stride(0), out.stride(0), lh_dtype(a.dtype), lh_dtype(out.dtype), flags, _stream()), "gemm")
        return out
    if workspace is not None:
        _lib.check(_lib.load().lh_hip_gemm_ws(
            out.data_ptr(), a.data_ptr(), b.data_ptr(), bias_ptr, M, N, K, a.stride(0), b.stride(0), out.stride(0),
            lh_dtype(a.dtype), lh_dtype(out.dtype), flags, workspace.data_ptr() if workspace.numel() else None,
            workspace.numel(), _stream()), "gemm")
        return out
    _lib.check(_lib.load().lh_hip_gemm(
        out.data_ptr(), a.data_ptr(), b.data_ptr(), bias_ptr,
        M, N, K, a.stride(0), b.stride(0), out.stride(0), lh_dtype(a.dtype), lh_dtype(out.dtype), flags, _stream()),
        "gemm")
    return out


def gemm_workspace_bytes(M, N, K, dtype, out_dtype=None, *, lda=None, ldb=None, ldc=None, bias=False, relu=False,
                         gelu=False, accumulate_c=False, transpose_a=False, transpose_b=False, tile=None, split_k=None,
                         operands=None) -> int:
    """Bytes of temporary memory `gemm(..., workspace=...)` needs for this problem (0 for most).
    `tile` and `split_k` are the requests of the `gemm` call the workspace is for (a requested cut
    along K needs its f32 blocks whatever the library would have chosen itself).  The plain query
    assumes 16-byte aligned operands; `operands=(out, a, b, bias_or_None)` asks for those tensors,
    whose alignment then counts (an unaligned operand runs on a padded copy in the workspace)."""
    flags = ((_lib.GEMM_HAS_BIAS if bias else 0) | (_lib.GEMM_HAS_RELU if relu else 0)
             | (_lib.GEMM_HAS_GELU if gelu else 0) | (_lib.GEMM_ACCUMULATE_C if accumulate_c else 0)
             | (_lib.GEMM_TRANSPOSE_A if transpose_a else 0) | (_lib.GEMM_TRANSPOSE_B if transpose_b else 0))
    if tile is not None:
        if tuple(tile) not in _lib.GEMM_TILES:
            raise ValueError(f"unsupported tile {tile}")
        flags |= _lib.GEMM_TILES[tuple(tile)]
    if split_k is not None:
        if split_k not in _lib.GEMM_SPLITK:
            raise ValueError(f"unsupported split_k {split_k}; choose from {sorted(_lib.GEMM_SPLITK)}")
        flags |= _lib.GEMM_SPLITK[split_k]
    lda = lda or (M if transpose_a else K)
    ldb = ldb or (K if transpose_b else N)
    if operands is not None:
        out, a, b, bias_t = operands
        if (bias_t is not None) != bool(bias):
            raise ValueError("operands and the bias flag disagree")
        return int(_lib.load().lh_hip_gemm_workspace_bytes_for(
            out.data_ptr(), a.data_ptr(), b.data_ptr(), bias_t.data_ptr() if bias_t is not None else None, M, N, K,
            a.stride(0), b.stride(0), out.stride(0), lh_dtype(dtype), lh_dtype(out_dtype or dtype), flags))
    return int(_lib.load().lh_hip_gemm_workspace_bytes(M, N, K, lda, ldb, ldc or N, lh_dtype(dtype),
                                                       lh_dtype(out_dtype or dtype), flags))


def gemm_fp8(a_q, b_q, scale_a: float, scale_b: float, *, out=None, out_dtype=torch.bfloat16, workspace=None):
    """out = out_dtype((Aq @ Bq)_f32 * scale_a * scale_b); see lh_hip_gemm_fp8 (lh_hip_gemm_fp8_ws
    with a `workspace`)."""
    _require(a_q.dim() == 2 and b_q.dim() == 2, "gemm_fp8 expects 2-D tensors")
    _require(a_q.dtype == torch.float8_e4m3fn and b_q.dtype == torch.float8_e4m3fn,
             "gemm_fp8 expects float8_e4m3fn operands")
    M, K = a_q.shape
    N = b_q.shape[1]
    if not (b_q.shape[0] == K):
        raise ValueError(f"B has {b_q.shape[0]} rows, A has {K} columns")
    _require(a_q.stride(1) == 1 and b_q.stride(1) == 1, "innermost stride must be 1")
    _require(a_q.stride(0) >= K and b_q.stride(0) >= N, "rows of A or B overlap")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=a_q.device)
    _is_matrix(out, M, N, "out")
    _require(out.dtype in (torch.bfloat16, torch.float32), "out must be bfloat16 or float32")
    _need_cuda(a_q, b_q, out, workspace)
    if workspace is not None:
        _require(workspace.dtype == torch.uint8 and workspace.dim() == 1 and workspace.is_contiguous(),
                 "workspace must be a contiguous uint8 vector")
        _lib.check(_lib.load().lh_hip_gemm_fp8_ws(
            out.data_ptr(), a_q.data_ptr(), b_q.data_ptr(), float(scale_a), float(scale_b), M, N, K,
            a_q.stride(0), b_q.stride(0), out.stride(0), lh_dtype(out.dtype),
            workspace.data_ptr() if workspace.numel() else None, workspace.numel(), _stream()), "gemm_fp8")
        return out
    _lib.check(_lib.load().lh_hip_gemm_fp8(
        out.data_ptr(), a_q.data_ptr(), b_q.data_ptr(), float(scale_a), float(scale_b), M, N, K,
        a_q.stride(0), b_q.stride(0), out.stride(0), lh_dtype(out.dtype), _stream()), "gemm_fp8")
    return out


def gemm_fp8_workspace_bytes(M, N, K, out_dtype=torch.bfloat16, *, lda=None, ldb=None, ldc=None) -> int:
    """Bytes of temporary memory `gemm_fp8(..., workspace=...)` needs; the row strides default to
    those of contiguous operands."""
    return int(_lib.load().lh_hip_gemm_fp8_workspace_bytes(M, N, K, lda or K, ldb or N, ldc or N, lh_dtype(out_dtype)))


def _strides3(t) -> _lib.Strides3:
    return _lib.Strides3(t.stride(0), t.stride(1), t.stride(2))


def _strides3_of(*tensors):
    """Those of each tensor; tensors laid out alike share one (each costs 0.5 us to make)."""
    first = tensors[0].stride()
    shared = _lib.Strides3(*first[:3])
    return [shared if t.stride() == first else _strides3(t) for t in tensors]


def _attention_request(rows_per_wave, stages, kv_split, scale_in_f32) -> int:
    """The bits of the causal word that ask for a kernel variant."""
    if not ((rows_per_wave or 0) in _lib.ATTN_ROWS and (stages or 0) in _lib.ATTN_STAGES and (kv_split or 0) in _lib.ATTN_KSPLIT):
        raise ValueError(f"rows_per_wave must be one of {sorted(_lib.ATTN_ROWS)[1:]}, stages one of {sorted(_lib.ATTN_STAGES)[1:]}, "
                         f"kv_split one of {sorted(_lib.ATTN_KSPLIT)[1:]}")
    return (_lib.ATTN_ROWS[rows_per_wave or 0] | _lib.ATTN_STAGES[stages or 0] | _lib.ATTN_KSPLIT[kv_split or 0]
            | (_lib.ATTN_SCALE_F32 if scale_in_f32 else 0))


def attention(q, k, v, *, causal=False, scale=None, out=None, rows_per_wave=None, stages=None, kv_split=None,
              workspace=None, scale_in_f32=False):
    """Fused attention forward on [Z,H,T,d] tensors (any strides with unit stride along d).
    `rows_per_wave` (32 or 64), `stages` (3 or 4, K/V ring of the 32-row kernel) and `kv_split`
    (2: two wave groups per workgroup on halves of the key range, 1: never) request a
    kernel variant for 16-bit tensors with head dimension 64; with none given the
    tuned-parameter database is asked, then the library chooses by shape.
    `workspace` (uint8, see attention_workspace_bytes) makes the call take its temporary memory
    from there instead of the library's pool (lh_hip_attention_ws).
    `scale_in_f32` (16-bit tensors, head dimension 64): Q stays as stored and every score is scaled
    in f32, the reference's rounding points exactly (LH_ATTN_SCALE_F32; about 7 % slower). Without it
    most problems multiply Q by the scale once and round it to the element type again; those with few
    query rows scale in f32 all the same."""
    if q.dim() != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("attention expects Q, K, V of equal 4-D shape [Z,H,T,d]")
    _require(q.dtype in _FLOATS and k.dtype == q.dtype and v.dtype == q.dtype,
             "attention expects Q, K, V of one dtype (float32, bfloat16 or float16)")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have the shape and dtype of Q")
    if q.stride(3) != 1 or k.stride(3) != 1 or v.stride(3) != 1 or out.stride(3) != 1:
        raise ValueError("innermost stride must be 1")
    _need_cuda(q, k, v, out)
    Z, H, T, d = q.shape
    if rows_per_wave is None and stages is None and kv_split is None and d == 64 and q.dtype != torch.float32:
        db = _tuned_db()
        if db is not None and db.entries:
            rows_per_wave, stages, kv_split = db.lookup_attention("bf16" if q.dtype == torch.bfloat16 else "f16", Z * H, T, d, causal)
            if (rows_per_wave or stages or kv_split) and not _rows_aligned16(q, k, v, out):
                rows_per_wave = stages = kv_split = None
    word = _lib.ATTN_CAUSAL if causal else 0
    if rows_per_wave or stages or kv_split or scale_in_f32:
        word |= _attention_request(rows_per_wave, stages, kv_split, scale_in_f32)
    if workspace is not None:
        _require(workspace.dtype == torch.uint8 and workspace.dim() == 1 and workspace.is_contiguous(),
                 "workspace must be a contiguous uint8 vector")
        _need_cuda(workspace)
        _lib.check(_lib.load().lh_hip_attention_ws(
            out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), Z, H, T, d,
            _strides3(out), _strides3(q), _strides3(k), _strides3(v),
            float(scale) if scale is not None else 1.0 / math.sqrt(d), word, lh_dtype(q.dtype),
            workspace.data_ptr() if workspace.numel() else None, workspace.numel(), _stream()), "attention")
        return out
    _lib.check(_lib.load().lh_hip_attention(
        out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), Z, H, T, d,
        *_strides3_of(out, q, k, v),
        float(scale) if scale is not None else 1.0 / math.sqrt(d), word, lh_dtype(q.dtype), _stream()),
        "attention")
    return out


def attention_workspace_bytes(Z, H, T, d, dtype, *, causal=False, rows_per_wave=None, stages=None, kv_split=None,
                              scale_in_f32=False) -> int:
    """Bytes of temporary memory `attention(..., workspace=...)` needs for contiguous [Z,H,T,d]
    tensors: the partial results of a key range split between workgroups, which the library
    chooses for 16-bit problems with few query blocks and long sequences; 0 for everything else
    and for every call that requests a kernel variant."""
    word = ((_lib.ATTN_CAUSAL if causal else 0) | _lib.ATTN_ROWS[rows_per_wave or 0] | _lib.ATTN_STAGES[stages or 0]
            | _lib.ATTN_KSPLIT[kv_split or 0] | (_lib.ATTN_SCALE_F32 if scale_in_f32 else 0))
    st = _lib.Strides3(H * T * d, T * d, d)
    return int(_lib.load().lh_hip_attention_workspace_bytes(Z, H, T, d, st, st, st, st, word, lh_dtype(dtype)))


def layer_norm(x, gamma, beta, eps=1e-5, *, out=None, out_dtype=None):
    _require(x.dim() == 2, "layer_norm expects a 2-D input")
    M, N = x.shape
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or x.dtype, device=x.device)
    if gamma.dtype != torch.float32 or beta.dtype != torch.float32:
        raise ValueError("gamma and beta must be float32")
    _is_vector(gamma, N, torch.float32, "gamma")
    _is_vector(beta, N, torch.float32, "beta")
    if not (tuple(out.shape) == (M, N)):
        raise ValueError(f"out must have shape [{M}, {N}]")
    if not x.is_contiguous() or not out.is_contiguous():
        raise ValueError("layer_norm expects contiguous tensors")
    _need_cuda(x, gamma, beta, out)
    _lib.check(_lib.load().lh_hip_layer_norm(
        out.data_ptr(), x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), M, N, float(eps),
        lh_dtype(x.dtype), lh_dtype(out.dtype), _stream()), "layer_norm")
    return out


def softmax(x, *, out=None):
    _require(x.dim() == 2, "softmax expects a 2-D input")
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    _same_dense(out, x, "softmax")
    _need_cuda(x, out)
    M, N = x.shape
    _lib.check(_lib.load().lh_hip_softmax(out.data_ptr(), x.data_ptr(), M, N, lh_dtype(x.dtype), _stream()), "softmax")
    return out


def gelu_tanh(x, *, out=None):
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    _same_dense(out, x, "gelu_tanh")
    _need_cuda(x, out)
    _lib.check(_lib.load().lh_hip_gelu_tanh(out.data_ptr(), x.data_ptr(), x.numel(), lh_dtype(x.dtype), _stream()),
               "gelu_tanh")
    return out


def bias_act(x, bias, relu=False, *, out=None):
    _require(x.dim() == 2, "bias_act expects a 2-D input")
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    _same_dense(out, x, "bias_act")
    M, N = x.shape
    _is_vector(bias, N, x.dtype, "bias")
    _need_cuda(x, bias, out)
    _lib.check(_lib.load().lh_hip_bias_act(out.data_ptr(), x.data_ptr(), bias.data_ptr(), M, N, 1 if relu else 0,
                                           lh_dtype(x.dtype), _stream()), "bias_act")
    return out


def add(a, b, *, out=None):
    out = torch.empty(a.shape, dtype=a.dtype, device=a.device) if out is None else out
    _same_dense(out, a, "add")
    _same_dense(b, a, "add (second operand)")
    _need_cuda(a, b, out)
    _lib.check(_lib.load().lh_hip_add(out.data_ptr(), a.data_ptr(), b.data_ptr(), a.numel(), lh_dtype(a.dtype),
                                      _stream()), "add")
    return out


def cast(x, dtype, *, out=None):
    out = torch.empty(x.shape, dtype=dtype, device=x.device) if out is None else out
    _require(tuple(out.shape) == tuple(x.shape) and out.dtype == dtype, "cast: out must have the input's shape and the target dtype")
    _require(x.is_contiguous() and out.is_contiguous(), "cast expects contiguous tensors")
    _need_cuda(x, out)
    _lib.check(_lib.load().lh_hip_cast(out.data_ptr(), x.data_ptr(), x.numel(), lh_dtype(x.dtype), lh_dtype(dtype),
                                       _stream()), "cast")
    return out


BLOCK_PARAM_NAMES = ("ln1_g", "ln1_b", "w_qkv", "b_qkv", "w_o", "b_o", "ln2_g", "ln2_b", "w_fc", "b_fc", "w_proj",
                     "b_proj", "w_q", "w_k", "w_v")


def _block_opts(dtype, causal, activation, bias_dtype, hidden):
    acts = {"gelu_tanh": _lib.ACT_GELU_TANH, "relu": _lib.ACT_RELU}
    if activation not in acts:
        raise ValueError(f"activation must be one of {sorted(acts)}")
    return _lib.NanoGPTBlockOpts(1 if causal else 0, acts[activation], lh_dtype(bias_dtype or dtype), int(hidden))


def _block_params(params: dict, C: int, n_head: int):
    """Validate one block's parameter tensors and pack their pointers.  Returns (struct, dtype,
    bias dtype or None, hidden).  (Runs for every block of every call: a block of few rows takes the device about 25 us,
    so messages are put together only to be raised.)"""
    if C % n_head != 0:
        raise ValueError(f"C={C} is not a multiple of n_head={n_head}")
    get = params.get
    w = {name: get(name) for name in ("w_qkv", "w_q", "w_k", "w_v", "w_o", "w_fc", "w_proj")}
    fused = w["w_qkv"] is not None
    if not fused and (w["w_q"] is None or w["w_k"] is None or w["w_v"] is None):
        raise ValueError("the block needs w_qkv or all of w_q, w_k, w_v")
    dtype = (w["w_qkv"] if fused else w["w_q"]).dtype
    if dtype not in _FLOATS:
        raise ValueError(f"unsupported weight dtype {dtype}")
    hidden = params["w_fc"].shape[1] if params["w_fc"].dim() == 2 else -1
    for name, shape in (("w_qkv", (C, 3 * C)), ("w_q", (C, C)), ("w_k", (C, C)), ("w_v", (C, C)), ("w_o", (C, C)),
                        ("w_fc", (C, hidden)), ("w_proj", (hidden, C))):
        t = w[name]
        if t is None:
            if name in ("w_o", "w_fc", "w_proj"):
                raise ValueError(f"missing block parameter {name}")
            continue
        if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}, got {tuple(t.shape)} {t.dtype}")
    for name in ("ln1_g", "ln1_b", "ln2_g", "ln2_b"):
        _is_vector(params[name], C, torch.float32, name)
    bias_dtype = None
    for name, n in (("b_qkv", 3 * C), ("b_o", C), ("b_fc", hidden), ("b_proj", C)):
        t = get(name)
        if t is None:
            continue
        bias_dtype = bias_dtype or t.dtype
        if t.dtype != dtype and t.dtype != torch.float32:
            raise ValueError(f"{name} must be float32 or have the weight dtype")
        _is_vector(t, n, bias_dtype, name)
    pointers = [None if get(name) is None else params[name].data_ptr() for name in BLOCK_PARAM_NAMES]
    return _lib.NanoGPTBlockParams(*pointers), dtype, bias_dtype, hidden


def nanogpt_block_workspace_bytes(B, T, C, dtype, *, causal=True, activation="gelu_tanh", bias_dtype=None,
                                  hidden=0) -> int:
    o = _block_opts(dtype, causal, activation, bias_dtype, hidden)
    return int(_lib.load().lh_hip_nanogpt_block_workspace_bytes(B, T, C, lh_dtype(dtype), ctypes.byref(o)))


def _workspace(workspace, need, device):
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if not (workspace.dtype == torch.uint8 and workspace.dim() == 1 and workspace.is_contiguous() and workspace.numel() >= need):
        raise ValueError(f"workspace must be a contiguous uint8 vector of at least {need} bytes")
    return workspace


def nanogpt_block(x, params: dict, n_head: int, *, eps=1e-5, out=None, workspace=None, causal=True,
                  activation="gelu_tanh"):
    """One GPT-2 block forward. x: [B,T,C] float32; params: tensors named BLOCK_PARAM_NAMES with
    weights stored [in,out] in float32, bfloat16 or float16 (LayerNorm parameters float32; biases
    float32 or the weight type, or absent).  Either `w_qkv` [C,3C] or `w_q`, `w_k`, `w_v` [C,C] each.
    The defaults are the benchmark's block; `causal=False, activation="relu"` with separate
    projections and float32 biases is the reference's (examples/xegpu/nanoGPT_payload.py:299-317)."""
    _require(x.dim() == 3 and x.dtype == torch.float32 and x.is_contiguous(), "x must be a contiguous float32 [B,T,C] tensor")
    B, T, C = x.shape
    p, dtype, bias_dtype, hidden = _block_params(params, C, n_head)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _same_dense(out, x, "nanogpt_block")
    o = _block_opts(dtype, causal, activation, bias_dtype, hidden)
    _need_cuda(x, out, workspace, *[t for t in params.values() if t is not None])
    need = int(_lib.load().lh_hip_nanogpt_block_workspace_bytes(B, T, C, lh_dtype(dtype), ctypes.byref(o)))
    workspace = _workspace(workspace, need, x.device)
    _lib.check(_lib.load().lh_hip_nanogpt_block(
        out.data_ptr(), x.data_ptr(), ctypes.byref(p), B, T, C, n_head, float(eps), lh_dtype(dtype), ctypes.byref(o),
        workspace.data_ptr(), workspace.numel(), _stream()), "nanogpt_block")
    return out


def nanogpt_forward(x, layers: list, lnf_g, lnf_b, lm_w, lm_b, n_head: int, *, eps=1e-5, out=None, workspace=None,
                    causal=True, activation="gelu_tanh"):
    """n blocks + final LayerNorm + lm_head. x: [B,T,C] float32; `layers`: one parameter dict per
    block (see nanogpt_block); lm_w [C, vocab] in the blocks' dtype and lm_b [vocab] (or None) in
    their bias dtype. Returns float32 logits [B,T,vocab]."""
    _require(x.dim() == 3 and x.dtype == torch.float32 and x.is_contiguous(), "x must be a contiguous float32 [B,T,C] tensor")
    B, T, C = x.shape
    if not (lm_w.dim() == 2 and lm_w.shape[0] == C and lm_w.is_contiguous()):
        raise ValueError(f"lm_w must be a contiguous [{C}, vocab] matrix")
    vocab = lm_w.shape[1]
    dtype = lm_w.dtype
    packed = [_block_params(p, C, n_head) for p in layers]
    for _, dt, _, _ in packed:
        _require(dt == dtype, "every block must have lm_w's dtype")
    bias_dtype = next((b for _, _, b, _ in packed if b is not None), lm_b.dtype if lm_b is not None else None)
    hidden = packed[0][3] if packed else 0
    _require(all(h == hidden for _, _, _, h in packed), "every block must have the same MLP width")
    _require(all(b in (None, bias_dtype) for _, _, b, _ in packed), "every block must have the same bias dtype")
    _is_vector(lnf_g, C, torch.float32, "lnf_g")
    _is_vector(lnf_b, C, torch.float32, "lnf_b")
    if lm_b is not None:
        _is_vector(lm_b, vocab, bias_dtype, "lm_b")
    if out is None:
        out = torch.empty((B, T, vocab), dtype=torch.float32, device=x.device)
    if not (tuple(out.shape) == (B, T, vocab) and out.dtype == torch.float32 and out.is_contiguous()):
        raise ValueError(f"out must be a contiguous float32 [{B}, {T}, {vocab}] tensor")
    o = _block_opts(dtype, causal, activation, bias_dtype, hidden)
    _need_cuda(x, out, workspace, lnf_g, lnf_b, lm_w, lm_b, *[t for p in layers for t in p.values() if t is not None])
    need = int(_lib.load().lh_hip_nanogpt_forward_workspace_bytes(B, T, C, vocab, lh_dtype(dtype), ctypes.byref(o)))
    workspace = _workspace(workspace, need, x.device)
    blocks = (_lib.NanoGPTBlockParams * max(len(layers), 1))(*[p for p, _, _, _ in packed])
    _lib.check(_lib.load().lh_hip_nanogpt_forward(
        out.data_ptr(), x.data_ptr(), blocks, len(layers), lnf_g.data_ptr(), lnf_b.data_ptr(), lm_w.data_ptr(),
        lm_b.data_ptr() if lm_b is not None else None, B, T, C, n_head, vocab, float(eps), lh_dtype(dtype),
        ctypes.byref(o), workspace.data_ptr(), workspace.numel(), _stream()), "nanogpt_forward")
    return out


# ---- generation over a paged key / value cache ------------------------------------------------------------------------
_CACHE_DTYPES = (torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn)
_SAMPLE_OPTIONS = ("temperature", "top_k", "top_p", "min_p")
_PACK_SAMPLE = struct.Struct(_lib.SAMPLE_OPTS_FORMAT).pack
_PACK_CACHE = struct.Struct(_lib.PAGED_CACHE_FORMAT).pack
_PACK_ROTARY = struct.Struct(_lib.ROTARY_FORMAT).pack
_F32_MAX = torch.finfo(torch.float32).max
_LH_DTYPE = {t: lh_dtype(t) for t in (torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn)}  # (in front of launches of a few microseconds)


def _on_current_device(*tensors) -> None:
    """Launches go to the current device's stream: tensors of another device would be read there through the wrong one."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            _need_cuda(*tensors)
            raise ValueError(f"expected tensors on one device, got {tensors[0].device} and {t.device}")
    if device < 0:
        raise ValueError("expected tensors on the GPU")
    if device != torch._C._cuda_getDevice():
        raise ValueError(f"expected tensors on the current device (cuda:{torch._C._cuda_getDevice()}), got {tensors[0].device}")


def _is_index(t, n, what: str) -> None:
    if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 vector of {n}, got {tuple(t.shape)} {t.dtype}")


def _paged_cache(k_cache, v_cache, block_table, B, k_scale, v_scale):
    """Checks a cache and its block table for B sequences: (lh_paged_cache as bytes, kv heads, d, positions of the table).
    (Runs in front of launches of a few microseconds: plain conditions, the struct packed in one go.)"""
    shape, dtype = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must have the same shape [pages, kv heads, page size, d]")
    if dtype not in _CACHE_DTYPES or v_cache.dtype != dtype:
        raise ValueError("k_cache and v_cache must have one dtype (float32, bfloat16, float16 or float8_e4m3fn)")
    pages, heads, size, d = shape
    if not (1 <= d <= 256 and pages and heads and size):
        raise ValueError(f"the cache must hold something, with a head dimension of 1 to 256, got {tuple(shape)}")
    sk, sv = k_cache.stride(), v_cache.stride()
    for st in (sk,) if sv == sk else (sk, sv):
        if st[3] != 1 and d != 1:
            raise ValueError("k_cache and v_cache: innermost stride must be 1")
        if (st[0] < d and pages > 1) or (st[1] < d and heads > 1) or (st[2] < d and size > 1):
            raise ValueError("k_cache and v_cache: rows overlap")
    if block_table is None:  # (for calls that name slots, which read none)
        rows, step, table = (B, 0), 0, 0
    else:
        table = block_table.data_ptr()
        rows = block_table.shape
        if len(rows) != 2 or rows[0] != B or rows[1] < 1 or block_table.dtype != torch.int32:
            raise ValueError(f"block_table must be an int32 tensor of shape [{B}, pages of a sequence], got {tuple(rows)} {block_table.dtype}")
        step, inner = block_table.stride()
        if inner != 1 and rows[1] > 1:
            raise ValueError("block_table: innermost stride must be 1")
        if step < rows[1]:
            if B > 1:
                raise ValueError("rows of block_table overlap")
            step = rows[1]
    if rows[1] * size >= 2**31 - 65536:
        raise ValueError("the block table must hold fewer than 2^31 - 65536 positions")
    if not (k_scale == 1.0 and v_scale == 1.0):
        if dtype != torch.float8_e4m3fn:
            raise ValueError("k_scale and v_scale belong to a cache of float8_e4m3fn")
        if not (0.0 < k_scale <= _F32_MAX and 0.0 < v_scale <= _F32_MAX):
            raise ValueError("k_scale and v_scale must be positive numbers")
    return (_PACK_CACHE(k_cache.data_ptr(), v_cache.data_ptr(), table, step, *sk[:3], *sv[:3], pages, rows[1], size,
                        heads, d, _LH_DTYPE[dtype], k_scale, v_scale), heads, d, rows[1] * size)


def _cache_weights(weights, B, heads, capacity):
    shape = weights.shape
    if weights.dtype != torch.float32 or len(shape) != 3 or shape[0] != B or shape[1] != heads or shape[2] < capacity:
        raise ValueError(f"weights must be a float32 tensor of shape [{B}, {heads}, {capacity} or more], got {tuple(shape)} {weights.dtype}")
    st = weights.stride()
    if (st[2] != 1 and shape[2] != 1) or (heads > 1 and st[1] < capacity) or (B > 1 and st[0] < capacity):
        raise ValueError("weights: innermost stride must be 1, and rows must not overlap")
    return st


def kv_append(k, v, k_cache, v_cache, block_table, positions, *, counts=None, k_scale=1.0, v_scale=1.0):
    """Writes the keys and values of new tokens into a paged cache and returns (k_cache, v_cache).

    k, v: [B, kv heads, T, d] (any strides with unit stride along d, so a projection's output can be passed as a view) in the cache's
    dtype; for a cache of float8_e4m3fn in float32, bfloat16 or float16, of which it holds e4m3(x / scale), clamped to +-448.
    k_cache, v_cache: [pages, kv heads, page size, d], any strides with unit stride along d.  block_table int32 [B, P]: position t of
    sequence b lies on page block_table[b, t // size], slot t % size.  Token t goes to position positions[b] + t (int32 [B]) if
    t < counts[b] (int32 [B]; None: all do).  Positions outside the table, and pages outside the cache (-1 for an entry not in use), are left out.
    Every token needs a slot of its own."""
    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or v.shape != shape or v.dtype != dtype:
        raise ValueError("k and v must have the same shape [B, kv heads, T, d] and dtype")
    B, heads, T, d = shape
    cache, cache_heads, cache_d, _ = _paged_cache(k_cache, v_cache, block_table, B, k_scale, v_scale)
    if heads != cache_heads or d != cache_d:
        raise ValueError(f"k and v have {heads} heads of {d}, the cache {cache_heads} of {cache_d}")
    if dtype not in _FLOATS or (dtype != k_cache.dtype and k_cache.dtype != torch.float8_e4m3fn):
        raise ValueError("k and v must have the cache's dtype (float32, bfloat16 or float16 for a cache of float8_e4m3fn)")
    sk, sv = k.stride(), v.stride()
    if d != 1 and (sk[3] != 1 or sv[3] != 1):
        raise ValueError("innermost stride must be 1")
    _is_index(positions, B, "positions")
    if counts is not None:
        _is_index(counts, B, "counts")
    _on_current_device(k, v, k_cache, v_cache, block_table, positions, counts)
    if B and T:
        _lib.check(_lib.load().lh_hip_kv_append(
            cache, k.data_ptr(), v.data_ptr(), *sk[:3], *sv[:3], positions.data_ptr(),
            counts.data_ptr() if counts is not None else None, B, T, lh_dtype(dtype), _stream()), "kv_append")
    return k_cache, v_cache


def _vector_workspace(workspace, need, like):
    """The caller's workspace or, from torch's allocator, one that a captured graph keeps for itself.  To be held until the launch is
    enqueued: from then on the allocator hands the memory out again only to work that follows on this stream."""
    if workspace is None:
        return like.new_empty(need, dtype=torch.uint8)
    _on_current_device(workspace)
    if not (workspace.dtype == torch.uint8 and workspace.dim() == 1 and workspace.is_contiguous() and workspace.numel() >= need
            and workspace.data_ptr() % 256 == 0):
        raise ValueError(f"workspace must be a contiguous uint8 vector of at least {need} bytes, 256-byte aligned")
    return workspace


def paged_attention(q, k_cache, v_cache, block_table, lengths, *, scale=None, out=None, weights=None, k_scale=1.0, v_scale=1.0,
                    workspace=None):
    """Attention of one new token of every sequence over its paged cache (laid out as for kv_append): out[b, h] =
    softmax(scale q[b, h] . k_t over t < lengths[b]) v_t, 0 where nothing is there.

    q, out: [B, H, d] (unit stride along d) in the cache's dtype, or bfloat16 / float16 for a cache of float8_e4m3fn, whose codes stand for
    code * k_scale and code * v_scale.  H is a multiple of the cache's heads; head h reads head h // (H // kv heads).  lengths int32 [B]
    counts the new token once it has been appended.  scale: 1 / sqrt(d) if None.  `weights`, float32 [B, kv heads, N] with N at least the
    positions of the block table: weights[b, g, t] grows by the probabilities of position t, added over the heads of group g
    (what kv_evict goes by).  `workspace` (uint8, see paged_attention_workspace_bytes): temporary memory, otherwise
    torch's allocator is asked; two calls that overlap in time need one each."""
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3:
        raise ValueError("paged_attention expects q of shape [B, H, d]")
    B, H, d = shape
    cache, heads, cache_d, capacity = _paged_cache(k_cache, v_cache, block_table, B, k_scale, v_scale)
    if d != cache_d:
        raise ValueError(f"q has a head dimension of {d}, the cache of {cache_d}")
    if H == 0 or H % heads:
        raise ValueError(f"{H} heads are no multiple of the cache's {heads}")
    if dtype not in _FLOATS or (dtype != k_cache.dtype and (k_cache.dtype != torch.float8_e4m3fn or dtype == torch.float32)):
        raise ValueError("q must have the cache's dtype (bfloat16 or float16 for a cache of float8_e4m3fn)")
    sq = q.stride()
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype:
        raise ValueError("out must have the shape and dtype of q")
    so = out.stride()
    if d != 1 and (so[2] != 1 or sq[2] != 1):
        raise ValueError("innermost stride must be 1")
    if (H > 1 and so[1] < d) or (B > 1 and so[0] < d):
        raise ValueError("rows of out overlap")
    _is_index(lengths, B, "lengths")
    w_ptr, w_b, w_h = None, 0, 0
    if weights is not None:
        w_b, w_h, _ = _cache_weights(weights, B, heads, capacity)
        w_ptr = weights.data_ptr()
    _on_current_device(q, k_cache, v_cache, block_table, lengths, out, weights)
    if B == 0:
        return out
    lib = _lib.load()
    need = lib.lh_hip_paged_attention_workspace_bytes(cache, B, H, w_ptr is not None)
    if need:
        workspace = _vector_workspace(workspace, need, q)
    _lib.check(lib.lh_hip_paged_attention(
        cache, out.data_ptr(), q.data_ptr(), so[0], so[1], sq[0], sq[1], lengths.data_ptr(), w_ptr, w_b, w_h, B, H,
        1.0 / math.sqrt(d) if scale is None else scale, lh_dtype(dtype),
        workspace.data_ptr() if need else None, need, _stream()), "paged_attention")
    return out


def paged_attention_workspace_bytes(q, k_cache, v_cache, block_table, *, weights=False) -> int:
    """Bytes of temporary memory that paged_attention takes for these tensors (only their shapes, strides and types matter);
    `weights`: whether the call passes any."""
    cache = _paged_cache(k_cache, v_cache, block_table, q.shape[0], 1.0, 1.0)[0]
    return int(_lib.load().lh_hip_paged_attention_workspace_bytes(cache, q.shape[0], q.shape[1], 1 if weights else 0))


def kv_evict(k_cache, v_cache, weights, block_table, lengths, budget, *, recent=0, out=None, workspace=None):
    """Shrinks every sequence longer than `budget` to it and returns the new lengths (int32 [B]; written to `out` if given, which may be
    `lengths`).  Of each kv head the last `recent` positions stay, and of the others the budget - recent with the largest weight
    (ties: the lowest positions; NaN is below every number).  Keys, values and weights of what stays move up, in order; weights behind
    them up to the old length become 0.  Every position below the length must lie on a page of its own; lengths are clamped to 0 and the
    positions of the block table.
    Cache, block table and weights are those of kv_append and paged_attention; `workspace` as there (kv_evict_workspace_bytes)."""
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    _is_index(lengths, B, "lengths")
    cache, heads, _, capacity = _paged_cache(k_cache, v_cache, block_table, B, 1.0, 1.0)
    w_b, w_h, _ = _cache_weights(weights, B, heads, capacity)
    budget, recent = int(budget), int(recent)
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"budget must be at least 1 and recent between 0 and the budget, got {budget} and {recent}")
    if out is None:
        out = lengths.new_empty(B)
    _is_index(out, B, "out")
    _on_current_device(k_cache, v_cache, weights, block_table, lengths, out)
    if B == 0:
        return out
    lib = _lib.load()
    need = lib.lh_hip_kv_evict_workspace_bytes(B, heads, min(budget, capacity))
    workspace = _vector_workspace(workspace, need, lengths)
    _lib.check(lib.lh_hip_kv_evict(cache, weights.data_ptr(), w_b, w_h, lengths.data_ptr(), out.data_ptr(), B, min(budget, capacity),
                                   min(recent, capacity), workspace.data_ptr(), need, _stream()), "kv_evict")
    return out


def kv_evict_workspace_bytes(k_cache, block_table, budget) -> int:
    """Bytes of temporary memory that kv_evict takes for this cache and block table."""
    capacity = block_table.shape[1] * k_cache.shape[2]
    return int(_lib.load().lh_hip_kv_evict_workspace_bytes(block_table.shape[0], k_cache.shape[1], min(int(budget), capacity)))


def sample(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, workspace=None):
    """The next token of every row of logits [B, V] (float32, bfloat16 or float16, rows of any stride): int64 [B].

    With w = exp((x - max) / temperature) in 64 bits (to 6e-12; sums of them to 2^-33 of the whole) and the words in falling order of x
    (equal ones: lowest index first): the first top_k words stay, of those the shortest beginning with at least top_p of their mass, of those the ones with w >= min_p;
    the first always does.  The token is the lowest index whose running sum of w over what stayed, by index, exceeds uniform[b] (float32
    [B], in [0, 1)) times their sum.  temperature <= 0: the largest logit.  top_k <= 0, top_p >= 1 and min_p <= 0 keep everything.
    NaN and -inf are no words, a +inf leaves only those, a row without words gives -1.
    Each setting is a number or a tensor [B] on the GPU (int32 for top_k, float32 for the others).  `workspace` as for paged_attention
    (sample_workspace_bytes; rows of up to 8192 words need none)."""
    if logits.dim() != 2 or logits.dtype not in _FLOATS or logits.shape[1] < 1:
        raise ValueError("sample expects logits of shape [B, V] in float32, bfloat16 or float16")
    B, V = logits.shape
    if logits.stride(1) != 1 and V != 1:
        raise ValueError("innermost stride must be 1")
    if B > 1 and logits.stride(0) < V:
        raise ValueError("rows of logits overlap")
    _is_vector(uniform, B, torch.float32, "uniform")
    pointers, numbers, vectors = [0, 0, 0, 0], [1.0, 0, 1.0, 0.0], []
    for i, value in enumerate((temperature, top_k, top_p, min_p)):
        if isinstance(value, torch.Tensor):
            _is_vector(value, B, torch.int32 if i == 1 else torch.float32, _SAMPLE_OPTIONS[i])
            pointers[i] = value.data_ptr()
            vectors.append(value)
        else:
            numbers[i] = max(0, min(int(value), 2**31 - 1)) if i == 1 else value
    try:
        options = _PACK_SAMPLE(*pointers, *numbers)
    except (OverflowError, struct.error):  # more than a float holds is infinite
        options = _PACK_SAMPLE(*pointers, *(x if i == 1 else ctypes.c_float(float(x)).value for i, x in enumerate(numbers)))
    if out is None:
        out = logits.new_empty(B, dtype=torch.int64)
    _is_vector(out, B, torch.int64, "out")
    _on_current_device(logits, uniform, out, *vectors)
    if B == 0:
        return out
    lib = _lib.load()
    need = lib.lh_hip_sample_workspace_bytes(B, V)
    if need:
        workspace = _vector_workspace(workspace, need, logits)
    _lib.check(lib.lh_hip_sample(
        out.data_ptr(), logits.data_ptr(), uniform.data_ptr(), B, V, max(logits.stride(0), V), lh_dtype(logits.dtype),
        options, workspace.data_ptr() if need else None, need, _stream()), "sample")
    return out


def sample_workspace_bytes(B, V) -> int:
    """Bytes of temporary memory that sample takes for B rows of V words."""
    return int(_lib.load().lh_hip_sample_workspace_bytes(B, V))


# ---- packed tokens of many sequences over a paged cache ------------------------------------------------------------------------
def kv_pages(block_table, lengths, counts, free_pages, n_free, page_size, tokens, *, out=None):
    """The pages of a step, and where its packed tokens lie: (lengths int32 [B], starts int32 [B + 1], positions int32 [tokens], slots int64 [tokens]).

    Sequence b has `lengths[b]` positions (int32 [B]) and gets `counts[b]` tokens (int32 [B]), or has ended, where that is negative: its
    length becomes 0.  block_table (int32 [B, P]) is updated: its first entries are the pages that the new length needs, those behind
    them -1, as at the beginning; a page is one sequence's.  free_pages (int32, one entry for every page of the cache) begins with the n_free (int32 [1]) pages that no sequence
    has; both are updated.  Pages that are needed no longer go back first, in the order of sequences and positions; then missing ones are taken from
    the list's end.  A sequence whose pages, with those that the ones before it miss, are more than there are, whose length would
    pass the table or whose rows pass `tokens`, is refused: pages and length stay, its rows have no place.
    Row i of the `tokens` packed ones belongs to the sequence with starts[b] <= i < starts[b + 1]; its position is positions[i], its slot (page *
    page_size + slot of the page) slots[i], -1 both where it has no place.  `out` receives the lengths (may be `lengths`)."""
    rows = block_table.shape
    if len(rows) != 2 or rows[1] < 1 or block_table.dtype != torch.int32:
        raise ValueError(f"block_table must be an int32 tensor of shape [sequences, pages of a sequence], got {tuple(rows)} {block_table.dtype}")
    B, P = rows
    step, inner = block_table.stride()
    if inner != 1 and P > 1:
        raise ValueError("block_table: innermost stride must be 1")
    if step < P and B > 1:
        raise ValueError("rows of block_table overlap")
    _is_index(lengths, B, "lengths")
    _is_index(counts, B, "counts")
    if free_pages.dim() != 1 or free_pages.shape[0] < 1:
        raise ValueError("free_pages must be an int32 vector with an entry for every page of the cache")
    _is_index(free_pages, free_pages.shape[0], "free_pages")
    _is_index(n_free, 1, "n_free")
    size, tokens = int(page_size), int(tokens)
    if size < 1 or P * size >= 2**31 - 65536:
        raise ValueError("the block table must hold fewer than 2^31 - 65536 positions, with at least one on a page")
    if not 0 <= tokens < 2**30:
        raise ValueError(f"tokens must be between 0 and 2^30, got {tokens}")
    if out is None:
        out = lengths.new_empty(B)
    _is_index(out, B, "out")
    _on_current_device(block_table, lengths, counts, free_pages, n_free, out)
    starts, positions = lengths.new_empty(B + 1), lengths.new_empty(tokens)
    slots = lengths.new_empty(tokens, dtype=torch.int64)
    _lib.check(_lib.load().lh_hip_kv_pages(
        block_table.data_ptr(), step, lengths.data_ptr(), counts.data_ptr(), out.data_ptr(), free_pages.data_ptr(), n_free.data_ptr(),
        starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), B, P, free_pages.shape[0], size, tokens, _stream()), "kv_pages")
    return out, starts, positions, slots


def rotary_frequencies(turned, *, base=10000.0, factor=1.0, context=None, low=1.0, high=32.0, device="cuda"):
    """Radians a position for the pairs of columns of `rotary`: float64 [turned / 2], base^(-2 i / turned).

    For contexts `factor` times as long as those a model has seen: without `context` every frequency is divided by the factor.  With it (the
    length that was seen) those that turn at most `low` times over it are divided, those that turn at least `high` times stay, between
    them the two are mixed in proportion."""
    turned = int(turned)
    if turned < 2 or turned % 2:
        raise ValueError(f"an even number of columns turns, got {turned}")
    if not (base > 0 and factor > 0 and (context is None or (context > 0 and low < high))):
        raise ValueError("base, factor and context must be positive, low below high")
    f = base ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned)
    if context is None:
        f = f / factor
    else:
        stays = ((f * context / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = stays * f + (1.0 - stays) * f / factor
    return f.to(device)


def _packed_rows(t, what: str):
    """(shape, strides of token and head) of a [N, heads, d] tensor."""
    shape, st = t.shape, t.stride()
    if len(shape) != 3 or t.dtype not in _FLOATS:
        raise ValueError(f"{what} must be a float32, bfloat16 or float16 tensor of shape [tokens, heads, d], got {tuple(shape)} {t.dtype}")
    if st[2] != 1 and shape[2] != 1:
        raise ValueError("innermost stride must be 1")
    return shape, st


def _row_stride(t, rows, cols, what: str) -> int:
    """Stride of the rows of a [rows, cols] matrix."""
    shape, st = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != rows or shape[1] != cols:
        raise ValueError(f"{what} must have shape [{rows}, {cols}], got {tuple(shape)}")
    if st[1] != 1 and cols != 1:
        raise ValueError(f"{what}: innermost stride must be 1")
    if st[0] < cols and rows != 1:
        raise ValueError(f"{what}: rows overlap (stride {st[0]} < {cols} columns)")
    return st[0]


def _packed_out(out, x, shape, what: str):
    """(the result of a call on x [N, heads, d], with rows of its own; its strides)."""
    if out is None:
        return x.new_empty(shape), (shape[1] * shape[2], shape[2])
    if out.shape != shape or out.dtype != x.dtype:
        raise ValueError(f"{what} must have the shape and dtype of its input")
    (n, heads, d), st = shape, out.stride()
    if d != 1 and st[2] != 1:
        raise ValueError("innermost stride must be 1")
    if n and heads and ((heads > 1 and st[1] < d) or (n > 1 and st[0] < d) or (n > 1 and heads > 1 and st[0] < (heads - 1) * st[1] + d and st[1] < (n - 1) * st[0] + d)):
        raise ValueError(f"rows of {what} overlap")
    return out, st


def _turn(positions, freqs, N, d, interleaved, amplitude):
    _is_index(positions, N, "positions")
    half = freqs.numel()
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not 1 <= half <= d // 2 or not freqs.is_contiguous():
        raise ValueError(f"freqs must be a contiguous float64 vector of 1 to {d // 2}, got {tuple(freqs.shape)} {freqs.dtype}")
    return _PACK_ROTARY(positions.data_ptr(), freqs.data_ptr(), 2 * half, 1 if interleaved else 0, amplitude)


def rotary(x, positions, freqs, *, interleaved=False, amplitude=1.0, out=None):
    """Rotary positions: of every head of x [N, heads, d] (any strides with unit stride along d) the column pairs (i, i + R / 2), or (2 i, 2 i + 1)
    if `interleaved`, turn by positions[n] * freqs[i]: (a cos - b sin, b cos + a sin), times `amplitude`.  freqs: float64 [R / 2] (see
    rotary_frequencies), radians a position; columns from R on stay.  positions: int32 [N].  `out` may be x.
    Turning by -freqs takes a gradient from the result to x (at the same amplitude), and at amplitude 1 the result back to x."""
    shape, sx = _packed_rows(x, "x")
    N, heads, d = shape
    turn = _turn(positions, freqs, N, d, interleaved, amplitude)
    out, so = _packed_out(out, x, shape, "out")
    _on_current_device(x, positions, freqs, out)
    if N and heads:
        _lib.check(_lib.load().lh_hip_rotary(out.data_ptr(), x.data_ptr(), so[0], so[1], sx[0], sx[1], turn, N, heads, d, _LH_DTYPE[x.dtype],
                                             _stream()), "rotary")
    return out


def kv_store(k, v, k_cache, v_cache, slots, *, q=None, q_out=None, positions=None, freqs=None, interleaved=False, amplitude=1.0, k_scale=1.0,
             v_scale=1.0):
    """Keys and values of packed tokens into their slots of a paged cache (see kv_pages): returns (k_cache, v_cache).

    k, v: [N, kv heads, d] (any strides with unit stride along d, so a projection's output can be passed as views) in the cache's dtype, or in
    float32, bfloat16 or float16 for a cache of float8_e4m3fn, which holds e4m3(x / scale), clamped to +-448.  k_cache, v_cache:
    [pages, kv heads, page size, d] as for kv_append.  slots int64 [N]: page * page size + slot; a token whose slot lies outside the cache (-1)
    is left out, two tokens must not share one.  With `positions` and `freqs` the keys turn on their way (see rotary).  `q` [N, H, d] turns
    with them, all rows of it, into `q_out` (which may be q; otherwise made here): then the result is (q_out, k_cache, v_cache)."""
    shape, sk = _packed_rows(k, "k")
    N, heads, d = shape
    dtype = k.dtype
    if v.shape != shape or v.dtype != dtype:
        raise ValueError("k and v must have the same shape [tokens, kv heads, d] and dtype")
    sv = v.stride()
    if d != 1 and sv[2] != 1:
        raise ValueError("innermost stride must be 1")
    cache, cache_heads, cache_d = _paged_cache(k_cache, v_cache, None, 1, k_scale, v_scale)[:3]
    if heads != cache_heads or d != cache_d:
        raise ValueError(f"k and v have {heads} heads of {d}, the cache {cache_heads} of {cache_d}")
    if dtype != k_cache.dtype and k_cache.dtype != torch.float8_e4m3fn:
        raise ValueError("k and v must have the cache's dtype (float32, bfloat16 or float16 for a cache of float8_e4m3fn)")
    if slots.dtype != torch.int64 or slots.dim() != 1 or slots.numel() != N or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 vector of {N}, got {tuple(slots.shape)} {slots.dtype}")
    if (positions is None) != (freqs is None):
        raise ValueError("positions and freqs go together")
    turn = None if freqs is None else _turn(positions, freqs, N, d, interleaved, amplitude)
    H, sq, so = 0, (0, 0), (0, 0)
    if q is not None:
        if turn is None:
            raise ValueError("q is passed to be turned: positions and freqs are missing")
        q_shape, sq = _packed_rows(q, "q")
        rows, H, q_d = q_shape
        if rows != N or q_d != d or q.dtype != dtype:
            raise ValueError(f"q must have shape [{N}, heads, {d}] and the dtype of k, got {tuple(q_shape)} {q.dtype}")
        q_out, so = _packed_out(q_out, q, q_shape, "q_out")
    elif q_out is not None:
        raise ValueError("q_out needs q")
    _on_current_device(k, v, k_cache, v_cache, slots, q, q_out, positions, freqs)
    if N:
        _lib.check(_lib.load().lh_hip_kv_store(
            cache, k.data_ptr(), v.data_ptr(), sk[0], sk[1], sv[0], sv[1], slots.data_ptr(), q_out.data_ptr() if H else None,
            q.data_ptr() if H else None, so[0], so[1], sq[0], sq[1], turn, N, H, _LH_DTYPE[dtype], _stream()), "kv_store")
    return (k_cache, v_cache) if q is None else (q_out, k_cache, v_cache)


def paged_attention_chunk(q, k_cache, v_cache, block_table, lengths, starts, *, scale=None, out=None, k_scale=1.0, v_scale=1.0, workspace=None):
    """Causal attention of packed chunks of new tokens over their sequences' paged caches (laid out as for kv_append).

    q, out: [N, H, d] (unit stride along d) in the cache's dtype, or bfloat16 / float16 for a cache of float8_e4m3fn, whose codes stand for
    code * k_scale and code * v_scale.  H is a multiple of the cache's heads; head h reads head h // (H // kv heads).  Sequence b has the rows
    starts[b] .. starts[b + 1] - 1 (int32 [B + 1], from 0 up); the last one is at position lengths[b] - 1 (int32 [B]: the new tokens count, and
    have been stored), the others right before it, and each sees the positions up to its own: softmax(scale q . k_t) v_t, 0 where it sees none.
    What lies at positions that a row does not see does not matter to it.  Rows from starts[B] on stay as they were.  scale: 1 / sqrt(d) if None.
    `out` may be q, but not another view of its memory.  `workspace` (uint8, see paged_attention_chunk_workspace_bytes): temporary memory, otherwise torch's allocator is asked; two
    calls that overlap in time need one each."""
    shape, sq = _packed_rows(q, "q")
    N, H, d = shape
    dtype = q.dtype
    B = block_table.shape[0]
    cache, heads, cache_d, _ = _paged_cache(k_cache, v_cache, block_table, B, k_scale, v_scale)
    if d != cache_d:
        raise ValueError(f"q has a head dimension of {d}, the cache of {cache_d}")
    if H == 0 or H % heads:
        raise ValueError(f"{H} heads are no multiple of the cache's {heads}")
    if dtype != k_cache.dtype and (k_cache.dtype != torch.float8_e4m3fn or dtype == torch.float32):
        raise ValueError("q must have the cache's dtype (bfloat16 or float16 for a cache of float8_e4m3fn)")
    _is_index(lengths, B, "lengths")
    _is_index(starts, B + 1, "starts")
    out, so = _packed_out(out, q, shape, "out")
    _on_current_device(q, k_cache, v_cache, block_table, lengths, starts, out)
    if N == 0 or B == 0:
        return out
    lib = _lib.load()
    need = lib.lh_hip_paged_attention_chunk_workspace_bytes(cache, N, B, H)
    if need:
        workspace = _vector_workspace(workspace, need, q)
    _lib.check(lib.lh_hip_paged_attention_chunk(
        cache, out.data_ptr(), q.data_ptr(), so[0], so[1], sq[0], sq[1], lengths.data_ptr(), starts.data_ptr(), N, B, H,
        1.0 / math.sqrt(d) if scale is None else scale, _LH_DTYPE[dtype], workspace.data_ptr() if need else None, need, _stream()),
        "paged_attention_chunk")
    return out


def paged_attention_chunk_workspace_bytes(q, k_cache, v_cache, block_table) -> int:
    """Bytes of temporary memory that paged_attention_chunk takes for these tensors (only their shapes and types matter).  Fewer tokens or sequences
    may take more: a workspace for several calls is the largest of theirs."""
    cache = _paged_cache(k_cache, v_cache, block_table, block_table.shape[0], 1.0, 1.0)[0]
    return int(_lib.load().lh_hip_paged_attention_chunk_workspace_bytes(cache, q.shape[0], block_table.shape[0], q.shape[1]))


def rms_norm(x, gamma, eps=1e-5, *, residual=None, residual_out=None, out=None, out_dtype=None, scale=None, row_scales=None):
    """Root-mean-square norm of the rows of x [M, C]: s / sqrt(mean(s^2) + eps) * gamma with s = x + residual (x where there is none), in f32.

    x: float32, bfloat16 or float16, rows of any stride; gamma: float32 [C].  `residual` [M, C], float32 or of the dtype of x, becomes s, or
    stays where `residual_out` (of its dtype) receives it.  out_dtype (default: that of x): float32, bfloat16, float16 or float8_e4m3fn; that one holds
    e4m3(y / scale), clamped to +-448: with `scale` given (a number: what gemm_fp8 takes as scale_a) the result is `out`; without, every row has
    the scale max |y| / 448 of its own (1 for a row of zeros) and the result is (out, row_scales), float32 [M]."""
    dtype, shape = x.dtype, x.shape
    if len(shape) != 2 or dtype not in _FLOATS or shape[1] < 1:
        raise ValueError("rms_norm expects x of shape [M, C] in float32, bfloat16 or float16")
    M, C = shape
    _is_vector(gamma, C, torch.float32, "gamma")
    if out is None:
        out = x.new_empty(shape) if out_dtype is None or out_dtype == dtype else x.new_empty(shape, dtype=out_dtype)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise ValueError(f"out must be {out_dtype}, got {out.dtype}")
    to = out.dtype
    if to not in _CACHE_DTYPES:
        raise ValueError("out must be float32, bfloat16, float16 or float8_e4m3fn")
    ld_out, ld_x = _row_stride(out, M, C, "out"), _row_stride(x, M, C, "x")
    r, r_out, ld_r, ld_r_out, r_dtype = None, None, 0, 0, 0
    if residual is not None:
        ld_r = ld_r_out = _row_stride(residual, M, C, "residual")
        if residual.dtype != dtype and residual.dtype != torch.float32:
            raise ValueError("residual must be float32 or have the dtype of x")
        if residual_out is None:
            residual_out = residual
        elif residual_out.dtype != residual.dtype:
            raise ValueError("residual_out must have the dtype of residual")
        else:
            ld_r_out = _row_stride(residual_out, M, C, "residual_out")
        r, r_out, r_dtype = residual.data_ptr(), residual_out.data_ptr(), _LH_DTYPE[residual.dtype]
    elif residual_out is not None:
        raise ValueError("residual_out needs residual")
    coded = to == torch.float8_e4m3fn
    if scale is not None and not (coded and 0.0 < scale <= _F32_MAX):
        raise ValueError("scale belongs to a result of float8_e4m3fn, and must be a positive number")
    if coded and scale is None:
        if row_scales is None:
            row_scales = gamma.new_empty(M)
        _is_vector(row_scales, M, torch.float32, "row_scales")
    elif row_scales is not None:
        raise ValueError("row_scales belong to a result of float8_e4m3fn without a scale")
    _on_current_device(x, gamma, residual, residual_out, out, row_scales)
    if M:
        _lib.check(_lib.load().lh_hip_rms_norm(
            out.data_ptr(), x.data_ptr(), gamma.data_ptr(), r, r_out, None if row_scales is None else row_scales.data_ptr(), scale or 1.0, M, C,
            ld_out, ld_x, ld_r, ld_r_out, eps, _LH_DTYPE[dtype], r_dtype, _LH_DTYPE[to], _stream()), "rms_norm")
    return out if row_scales is None else (out, row_scales)


def release_scratch() -> None:
    """Free the library's pool of temporary buffers on the current device (waits for the device)."""
    _lib.check(_lib.load().lh_hip_release_scratch(), "release_scratch")
