"""ctypes binding of libhmx.so (the C ABI declared in include/hmx.h).

The library is loaded lazily on first use.  There is no CPU fallback: calling
an op without the built library, or with tensors that are not on a GPU,
raises.  Status codes from the C side map to the Python exception types the
reference ops raise (ValueError / NotImplementedError / RuntimeError).
"""
from __future__ import annotations

import ctypes
import functools
import itertools
import os
from pathlib import Path

import numpy as np
import torch

LIB_PATH = Path(__file__).resolve().parent / "libhmx.so"

HMX_OK, HMX_EINVAL, HMX_EUNSUPPORTED, HMX_EHIP = 0, 1, 2, 3
HMX_F32, HMX_BF16, HMX_F16 = 0, 1, 2

_DTYPE_CODE = {torch.float32: HMX_F32, torch.bfloat16: HMX_BF16, torch.float16: HMX_F16}

_P = ctypes.c_void_p
_I32 = ctypes.c_int32
_I64 = ctypes.c_int64
_F32 = ctypes.c_float

# name -> argtypes (restype is int unless listed in _RESTYPES)
SIGNATURES: dict[str, list] = {
    "hmx_abi_version": [],
    "hmx_last_error": [],
    "hmx_gdn_gating": [_P, _I32, _P, _I64, _I64, _P, _I64, _I64, _I32, _P, _I32, _P, _P, _I32,
                       _I64, _I32, _F32, _F32, _P],
    "hmx_gdn_recurrent_fwd": [_P, _I64, _P, _I64, _P, _I64, _I32, _P, _I32, _P, _I32, _I32, _P,
                              _P, _I64, _P, _I64, _I32,
                              _P, _P, _I64, _P,
                              _I64, _I64, _I64, _I32, _I32, _I32, _I32,
                              _F32, _I32, _I32, _P, _P, _P],
    "hmx_gdn_chunk_fwd": [_P, _I64, _P, _I64, _P, _I64, _I32, _P, _I32, _P, _I32, _P,
                          _P, _P, _I64, _I32, _P, _P,
                          _P, _I32, _I32, _I32, _I32, _I32, _I32, _F32,
                          _I32, _I32, _F32, _P, ctypes.c_size_t, _P, _P, _P],
    "hmx_gdn_chunk_workspace_bytes": [_I32, _I32, _I32, _I32],
    "hmx_gdn_chunk_fwd_noalloc": [_P, _I64, _P, _I64, _P, _I64, _I32, _P, _I32, _P, _I32, _P,
                                  _P, _P, _I64, _I32, _P, _P,
                                  _P, _I32, _I32, _I32, _I32, _I32, _I32, _F32,
                                  _I32, _I32, _F32, _P, _P, _P],
    "hmx_gka_gating": [_P, _I32, _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I32, _P, _I32,
                       _P, _P, _P, _I32, _I64, _I32, _F32, _F32, _P],
    "hmx_gka_decode_fwd": [_P, _I64, _P, _I64, _P, _I64, _I32, _P, _I32, _P, _I32, _P, _I32, _P,
                           _P, _I64, _P, _I64, _P, _I64, _P, _I64, _I32,
                           _P, _P, _I64, _I64, _I64, _I64, _I32, _I32, _I32, _I32,
                           _I32, _F32, _F32, _P, _P, _P],
    "hmx_gka_chunk_fwd": [_P, _I64, _P, _I64, _P, _I64, _I32, _P, _I32, _P, _I32, _P, _I32,
                          _P, _I32, _P,
                          _P, _P, _I64, _I32, _P, _P, _I64, _I32, _P, _P,
                          _P, _I32, _I32, _I32, _I32, _I32, _I32, _I32,
                          _I32, _F32, _F32, _I32, _P, ctypes.c_size_t, _P, _P, _P],
    "hmx_gka_chunk_workspace_bytes": [_I32, _I32, _I32, _I32],
    "hmx_gka_cheb_fwd": [_P, _I64, _P, _I64, _I32, _P, _I32, _P, _P, _P, _P, _I32, _I32, _I32,
                         _I32, _I32, _I32, _F32, _P, ctypes.c_size_t, _P],
    "hmx_gka_cheb_bwd": [_P, _I64, _P, _P, _I64, _I32, _P, _I32, _P, _P, _P, _P, _P, _I32, _I32,
                         _I32, _I32, _I32, _I64, _I32, _F32, _I32, _P, ctypes.c_size_t, _P,
                         ctypes.c_size_t, _P],
    "hmx_gka_cheb_bwd_workspace_bytes": [_I32, _I32, _I64],
    "hmx_gka_train_fwd": [_P, _P, _P, _I32, _P, _I32, _P, _I32, _P, _I32, _P, _P, _P, _P, _P,
                          _P, _I32, _I32, _I32, _I32, _I32, _I32, _F32, _F32, _P,
                          ctypes.c_size_t, _P],
    "hmx_gka_train_bwd": [_P, _P, _P, _I32, _P, _I32, _P, _I32, _P, _I32, _P, _P, _P, _P, _P, _P,
                          _P, _P, _P, _P, _I32, _I32, _I32, _I32, _I32, _I64, _I32, _F32, _F32,
                          _I32, _P, ctypes.c_size_t, _P, ctypes.c_size_t, _P],
    "hmx_gka_train_bwd_workspace_bytes": [_I32, _I32, _I64],
    "hmx_gdn_train_fwd": [_P, _I64, _P, _P, _I64, _P, _I32, _P, _I32, _P, _P, _P, _P, _I32,
                          _I32, _I32, _F32, _I32, _I32, _F32, _P, ctypes.c_size_t, _P, _P, _P],
    "hmx_gdn_train_bwd": [_P, _I64, _P, _P, _I64, _P, _I32, _P, _I32, _P, _I64, _P, _P, _P, _P,
                          _I32, _I32, _P, _I32, _I32, _F32, _I32, _F32, _I32, _P, _P, _P, _P,
                          _P, _P, _P, ctypes.c_size_t, _P],
    "hmx_gdn_train_bwd_workspace_bytes": [_I32, _I32, _I32, _I32],
    "hmx_plan_segments": [_I32, _P, _I32, _I32, _I64, _I32, _I32, _I32, _P, _I32, _P, _P],
    "hmx_plan_segments_bounds": [_I32, _P, _I32, _I64, _I32, _I32, _I32, _P, _I32, _P, _P],
    "hmx_ssd_chunk_fwd": [_P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I32,
                          _P, _I32, _I64, _I64, _P, _P, _P, _P, _I64, _I64,
                          _P, _I64, _I64, _P, _P, _I64, _I32, _P, _P, _P, _I32, _I32,
                          _I32, _I32, _I32, _I32, _I32, _I32, _I32, _F32, _F32, _P, ctypes.c_size_t,
                          _P],
    "hmx_ssd_chunk_workspace_bytes": [_I32, _I32, _I32, _I32, _I32],
    "hmx_ssd_chunk_bwd": [_P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I32,
                          _P, _I32, _I64, _I64, _P, _P, _P, _P, _I64, _I64,
                          _P, _I64, _I64, _P, _P, _P, _I32, _P, _I32,
                          _I32, _I32, _I32, _I32, _I32, _I32, _I32, _F32, _F32,
                          _P, _P, _P, _I32, _P, _P, _P, _P, _P, _P, _P, ctypes.c_size_t, _P],
    "hmx_ssd_chunk_bwd_workspace_bytes": [_I32, _I32, _I32, _I32],
    "hmx_causal_conv1d_fwd": [_P, _I64, _P, _I64, _I32, _P, _I32, _I32, _P, _I32, _P, _I64, _I64,
                              _I32, _P, _I32, _I64, _P, _P, _I32, _I32, _I32, _P],
    "hmx_causal_conv1d_update": [_P, _I64, _P, _I64, _I32, _P, _I32, _I32, _P, _I32, _P, _I64,
                                 _I64, _I32, _P, _I32, _I32, _I32, _I32, _P],
    "hmx_causal_conv1d_update_spec": [_P, _I64, _P, _I64, _I32, _P, _I32, _I32, _P, _I32, _P,
                                      _I64, _I64, _I32, _P, _P, _P, _I32, _I64, _I32, _I32,
                                      _I32, _P],
    "hmx_causal_conv1d_fwd_blocks": [_P, _I64, _P, _I64, _I32, _P, _I32, _I32, _P, _I32, _P,
                                     _I64, _I64, _I32, _P, _I32, _I64, _P, _I64, _I32, _P, _P,
                                     _P, _P, _P, _I32, _I32, _I32, _I32, _P],
    "hmx_causal_conv1d_update_blocks": [_P, _I64, _P, _I64, _I32, _P, _I32, _I32, _P, _I32, _P,
                                        _I64, _I64, _I32, _P, _I64, _I32, _P, _P, _I32, _I32,
                                        _I32, _I32, _P],
    "hmx_rms_norm_gated": [_P, _I64, _P, _I64, _I32, _P, _I32, _P, _I64, _I64, _I32, _F32, _I32, _P],
    "hmx_ssd_state_update": [_P, _I32, _I64, _P, _I32, _I64, _I64, _I64,
                             _P, _I32, _I64, _I64, _I64, _P, _I64, _I64, _I64,
                             _P, _I32, _I64, _I64, _P, _I32, _I64, _I64,
                             _P, _I64, _I64, _P, _I64, _I64,
                             _P, _I32, _I64, _I64, _I64, _P, _I32, _I64, _I64, _I64,
                             _P, _P, _I32, _I32, _I32, _I32, _I32, _I32, _I32, _I32, _I32, _P],
    "hmx_append_paged_kv": [_P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I32, _P, _I64, _I64,
                            _P, _P, _I32, _P, _I32, _P, _I32, _I64, _I64, _I32, _I32, _I64, _I32,
                            _I32, _I32, _P],
    "hmx_paged_attention_decode": [_P, _I64, _I64, _I32, _P, _I64, _I64, _P, _I32, _I32, _I32,
                                   _I32, _F32, _P, ctypes.c_size_t, _P],
    "hmx_paged_attention_decode_workspace_bytes": [_I32, _I32, _I32, _I32, _I64],
    "hmx_causal_attention": [_P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I32, _P, _I64, _I64,
                             _P, _P, _I32, _I64, _I32, _I32, _I32, _F32, _I32, _P, ctypes.c_size_t, _P],
    "hmx_causal_attention_workspace_bytes": [_I32, _I64, _I32, _I32, _I32, _I32],
    "hmx_causal_attention_bwd": [_P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I32, _P, _I64,
                                 _I64, _P, _I64, _I64, _P, _P, _I32, _I64, _I32, _I32, _I32, _F32,
                                 _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _P, _P],
    "hmx_paged_causal_attention": [_P, _I64, _I64, _I32, _P, _I64, _I64, _P, _P, _I32, _I64, _I32,
                                   _I32, _I32, _F32, _I32, _P, ctypes.c_size_t, _P],
    "hmx_paged_causal_attention_workspace_bytes": [_I32, _I64, _I32, _I32, _I32, _I64],
}
_RESTYPES = {"hmx_last_error": ctypes.c_char_p, "hmx_gdn_chunk_workspace_bytes": ctypes.c_size_t,
             "hmx_gka_chunk_workspace_bytes": ctypes.c_size_t,
             "hmx_gka_cheb_bwd_workspace_bytes": ctypes.c_size_t,
             "hmx_gka_train_bwd_workspace_bytes": ctypes.c_size_t,
             "hmx_gdn_train_bwd_workspace_bytes": ctypes.c_size_t,
             "hmx_ssd_chunk_workspace_bytes": ctypes.c_size_t,
             "hmx_ssd_chunk_bwd_workspace_bytes": ctypes.c_size_t,
             "hmx_paged_attention_decode_workspace_bytes": ctypes.c_size_t,
             "hmx_causal_attention_workspace_bytes": ctypes.c_size_t,
             "hmx_paged_causal_attention_workspace_bytes": ctypes.c_size_t}



class GatedNorm(ctypes.Structure):
    """hmx_gated_norm (include/hmx.h): the optional output-norm epilogue."""
    _fields_ = [("gate", _P), ("gate_token_stride", _I64), ("gate_head_stride", _I64),
                ("weight", _P), ("weight_dtype", _I32), ("eps", _F32)]


def gated_norm(gate: torch.Tensor | None, weight: torch.Tensor, eps: float, V: int):
    """ctypes pointer to an hmx_gated_norm for a gate viewed as [tokens, H, V]
    (None: no epilogue requested -> returns None, i.e. NULL)."""
    w = weight.contiguous()
    if w.numel() != V:
        raise ValueError(f"o_norm weight has {w.numel()} elements, expected {V}")
    s = GatedNorm(None if gate is None else gate.data_ptr(),
                  0 if gate is None else gate.stride(0), 0 if gate is None else gate.stride(1),
                  w.data_ptr(), dtype_code(w), float(eps))
    s._keep = (gate, w)   # the tensors outlive the call
    return ctypes.pointer(s)


class GateProj(ctypes.Structure):
    """hmx_gate_proj (include/hmx.h): gates formed from the raw projections."""
    _fields_ = [("A_log", _P), ("A_log_dtype", _I32), ("dt_bias", _P), ("dt_bias_dtype", _I32),
                ("a", _P), ("a_token_stride", _I64), ("a_head_stride", _I64),
                ("b", _P), ("b_token_stride", _I64), ("b_head_stride", _I64),
                ("alpha_in", _P), ("alpha_token_stride", _I64), ("alpha_head_stride", _I64),
                ("in_dtype", _I32), ("softplus_beta", _F32), ("softplus_threshold", _F32),
                ("beta_scale", _F32), ("alpha_add", _F32), ("alpha_zero", _I32),
                ("gk_from_g", _I32)]


def gate_proj(pg):
    """ctypes pointer to an hmx_gate_proj for an hmx.ops.ProjGates (None -> NULL)."""
    if pg is None:
        return None
    ts = [t for t in (pg.a, pg.b, pg.alpha_in) if t is not None]
    if not ts:
        raise ValueError("ProjGates needs at least one of a, b, alpha_in")
    in_dt = ts[0].dtype
    for t in ts:
        if t.dim() != 2 or t.dtype != in_dt:
            raise ValueError("ProjGates a / b / alpha_in must be [tokens, heads] of one dtype")
    require_gpu(pg.A_log, pg.dt_bias, *ts)
    st = lambda t: (0, 0) if t is None else (t.stride(0), t.stride(1))
    s = GateProj(ptr(pg.A_log), 0 if pg.A_log is None else dtype_code(pg.A_log),
                 ptr(pg.dt_bias), 0 if pg.dt_bias is None else dtype_code(pg.dt_bias),
                 ptr(pg.a), *st(pg.a), ptr(pg.b), *st(pg.b), ptr(pg.alpha_in), *st(pg.alpha_in),
                 _DTYPE_CODE[in_dt], float(pg.softplus_beta), float(pg.softplus_threshold),
                 float(pg.beta_scale), float(pg.alpha_add), int(bool(pg.alpha_zero)),
                 int(bool(pg.gk_from_g)))
    s._keep = (pg.A_log, pg.dt_bias, *ts)
    return ctypes.pointer(s)


class PagedKV(ctypes.Structure):
    """hmx_paged_kv (include/hmx.h): a paged key/value cache and its sequences."""
    _fields_ = [("k", _P), ("k_page_stride", _I64), ("k_token_stride", _I64),
                ("k_head_stride", _I64), ("v", _P), ("v_page_stride", _I64),
                ("v_token_stride", _I64), ("v_head_stride", _I64), ("table", _P),
                ("table_stride", _I64), ("seq_lens", _P), ("table_width", _I32),
                ("num_pages", _I32), ("page_size", _I32)]


def paged_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor | None = None,
             seq_lens: torch.Tensor | None = None):
    """ctypes pointer to an hmx_paged_kv of caches [pages, page size, HKV, D]; strides of
    dimensions of one, which are never used and may be anything, go as 0."""
    n = k_cache.shape
    if k_cache.is_contiguous() and v_cache.is_contiguous():
        hs = n[3]
        ts = n[2] * hs
        ks = vs = (n[1] * ts, ts, hs)
    else:
        ks, vs = ([x if m > 1 else 0 for x, m in zip(t.stride()[:3], n)] for t in (k_cache, v_cache))
    return ctypes.pointer(PagedKV(
        k_cache.data_ptr(), *ks, v_cache.data_ptr(), *vs, ptr(table),
        0 if table is None else table.stride(0), ptr(seq_lens),
        0 if table is None else table.shape[1], n[0], n[1]))


_lib = None


class HmxLibraryMissing(RuntimeError):
    pass


def load(path: str | os.PathLike | None = None):
    """Load (once) and return the ctypes handle with argtypes installed."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise HmxLibraryMissing(
            f"libhmx.so not found at {p}; build it with `python hybrid-model-factory_amd/hmx/build.py`")
    lib = ctypes.CDLL(str(p))
    for name, argtypes in SIGNATURES.items():
        try:
            fn = getattr(lib, name)
        except AttributeError:
            raise HmxLibraryMissing(
                f"{p} is older than this package (it has no {name}); build it again with "
                f"`python hybrid-model-factory_amd/hmx/build.py`") from None
        fn.argtypes = argtypes
        fn.restype = _RESTYPES.get(name, ctypes.c_int)
    if path is None:
        _lib = lib
    return lib


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPE_CODE[t.dtype]
    except KeyError:
        raise NotImplementedError(f"unsupported dtype {t.dtype}") from None


def ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def stream_of(t: torch.Tensor):
    """torch's current stream on the tensor's device, as the raw handle: building a
    torch.cuda.Stream object for it takes 2.1 us, this 0.1.  A tensor off the GPU raises
    (the raw call would take its index -1 for the current device)."""
    index = t.get_device()
    if index < 0:
        raise ValueError(f"expected a tensor on a GPU, got one on {t.device}")
    return torch._C._cuda_getCurrentRawStream(index)


PLAN_GDN, PLAN_GKA, PLAN_SSD = 0, 1, 2


def plan_segments(op: int, bounds: list[tuple[int, int]], tokens: int, H: int, cu_count: int,
                  segment_chunks: int | None = None) -> tuple[np.ndarray, int]:
    """The segment table of a chunked prefill (hmx_plan_segments_bounds, host code)
    as an int32 [rows, 8] array, and the chunks of all sequences."""
    table, nblk = segment_plan(op, bounds, tokens, H, cu_count, segment_chunks)
    return table.copy(), nblk


def segment_plan(op: int, bounds: list[tuple[int, int]], tokens: int, H: int, cu_count: int,
                 segment_chunks: int | None = None) -> tuple[np.ndarray, int]:
    """plan_segments with a read-only table.  It depends on the sizes alone, and the last
    few distinct ones are kept, shared by all callers and threads: lengths planned
    before take 1 us (4 for 256 sequences) and new ones 10 (48), where asking the library
    for the table's size first and keeping none takes 12 (84) for any."""
    args = (tokens, H, cu_count, segment_chunks or 0)
    try:
        return _plan(op, tuple(bounds), *args)
    except TypeError:      # bounds as lists or an array
        return _plan(op, tuple(map(tuple, bounds)), *args)


@functools.lru_cache(maxsize=64)
def _plan(op: int, bounds: tuple, tokens: int, H: int, cu_count: int, segment_chunks: int):
    n = len(bounds)
    tokens, H, cu_count = int(tokens), int(H), int(cu_count)
    be = np.fromiter(itertools.chain.from_iterable(bounds), np.int64, 2 * n)
    nrows, nblk = ctypes.c_int32(0), ctypes.c_int32(0)
    args = (op, be.ctypes.data, n, tokens, H, cu_count, int(segment_chunks))

    def build(rows):
        table = np.empty((rows, 8), dtype=np.int32)
        call("hmx_plan_segments_bounds", *args, table.ctypes.data, rows, ctypes.byref(nrows),
             ctypes.byref(nblk))
        return table

    # one call into a table that holds what the planner makes of it without
    # segment_chunks (a row a sequence, or up to four workgroups a CU); a larger
    # table's size comes back in nrows
    room = n + max(0, 4 * cu_count // max(H, 1))
    try:
        table = build(room)[:nrows.value]
    except ValueError:
        if nrows.value <= room:
            raise
        table = build(nrows.value)
    return read_only(table), nblk.value


def read_only(a: np.ndarray) -> np.ndarray:
    """``a``, marked read-only: a plan kept for several callers."""
    a.flags.writeable = False
    return a


def require_gpu(*tensors: torch.Tensor | None) -> None:
    """The product path runs only on the GPU: refuse CPU tensors loudly."""
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("hmx ops run only on GPU tensors (no CPU fallback); got a "
                               f"{t.device} tensor")


def call(name: str, *args) -> None:
    lib = load()
    rc = getattr(lib, name)(*args)
    if rc == HMX_OK:
        return
    msg = (lib.hmx_last_error() or b"").decode(errors="replace")
    if rc == HMX_EINVAL:
        raise ValueError(msg)
    if rc == HMX_EUNSUPPORTED:
        raise NotImplementedError(msg)
    raise RuntimeError(msg)
