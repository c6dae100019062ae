"""Python binding of the GQA attention C ABI (include/tkm_attn.h, libtkm_attn.so).

Mirrors the reference's GQA op (``GQA(q=, kv=, d=, causal=)``, reference
src/tkm_core.c:83-95) as it is executed by the runtime: forward at
src/tkm_gpu.cu:1252-1265, backward at src/tkm_gpu.cu:1389-1404.  Tensors are
torch device tensors (torch is used only for device memory and streams); every
call goes through ctypes into the HIP library and launches on the caller's
current torch stream.  There is no fallback: if the library is missing or a
call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
import re

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
LIB_PATH = os.path.join(PKG, "libtkm_attn.so")
HEADER = os.path.join(ROOT, "include", "tkm_attn.h")

F16, BF16 = 0, 1
BWD_DELTA, BWD_DKDV, BWD_DQ, BWD_DQ_DELTA = 0, 1, 2, 3

_vp = ctypes.c_void_p
_i = ctypes.c_int
_lib = None


class _Kv(ctypes.Structure):
    """tkm_attn_kv"""
    _fields_ = [(n, _vp) for n in ("k", "v", "table", "len", "weight")] + [
        (n, _i) for n in ("B", "Hkv", "D", "page", "max_pages", "num_pages", "dtype")]


class _RopeParams(ctypes.Structure):
    """tkm_attn_rope_params"""
    _fields_ = [("rot", _i), ("layout", _i), ("scaling", _i)] + [
        (n, ctypes.c_double) for n in ("theta", "scale", "original", "low", "high", "factor")]


class _Rope(ctypes.Structure):
    """tkm_attn_rope"""
    _fields_ = [("rot", _i), ("layout", _i), ("factor", ctypes.c_float), ("turns", ctypes.c_uint64 * 64)]


class _Pages(ctypes.Structure):
    """tkm_attn_pages"""
    _fields_ = [(n, _vp) for n in ("free", "n_free", "held")]


class _Plan(ctypes.Structure):
    """tkm_attn_plan"""
    _fields_ = [(n, _vp) for n in ("n_new", "row_start", "seq", "pos", "slot")]


class AttnError(RuntimeError):
    """A tkm_attn_* call returned a non-zero status."""

    def __init__(self, fn: str, status: int, message: str):
        super().__init__(f"{fn} failed with status {status}: {message}")
        self.status = status


def header_functions() -> list:
    """Names of the functions include/tkm_attn.h declares."""
    with open(HEADER) as f:
        text = f.read()
    return re.findall(r"TKM_ATTN_API\s+[\w\s\*]+?\b(tkm_attn_\w+)\s*\(", text)


def lib() -> ctypes.CDLL:
    """Load libtkm_attn.so (built by tokamak_amd.build); raises if absent."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -m tokamak_amd.build` "
            "(the attention path has no non-HIP implementation)")
    L = ctypes.CDLL(LIB_PATH)
    L.tkm_attn_fwd.argtypes = [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, ctypes.c_float, _i, _i, _vp]
    L.tkm_attn_fwd.restype = _i
    L.tkm_attn_bwd_workspace_bytes.argtypes = [_i, _i, _i]
    L.tkm_attn_bwd_workspace_bytes.restype = ctypes.c_size_t
    bwd_args = [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, ctypes.c_float, _i, _i,
                _vp, ctypes.c_size_t, _vp]
    L.tkm_attn_bwd.argtypes = bwd_args
    L.tkm_attn_bwd.restype = _i
    L.tkm_attn_bwd_stage.argtypes = [_i] + bwd_args
    L.tkm_attn_bwd_stage.restype = _i
    L.tkm_attn_status_string.argtypes = [_i]
    L.tkm_attn_status_string.restype = ctypes.c_char_p
    L.tkm_attn_last_error.restype = ctypes.c_char_p
    L.tkm_attn_version.restype = _i
    L.tkm_attn_init.restype = _i
    L.tkm_attn_asm_available.restype = _i
    L.tkm_attn_last_kernels.restype = ctypes.c_uint
    kv = ctypes.POINTER(_Kv)
    L.tkm_attn_kv_append.argtypes = [kv, _vp, _i, _i, _vp, _vp, _vp]
    L.tkm_attn_kv_append.restype = _i
    L.tkm_attn_decode_workspace_bytes.argtypes = [kv, _i, _i]
    L.tkm_attn_decode_workspace_bytes.restype = ctypes.c_size_t
    L.tkm_attn_decode.argtypes = [kv, _vp, ctypes.c_longlong, _vp, _vp, _i, ctypes.c_float, _i, _vp, ctypes.c_size_t, _vp]
    L.tkm_attn_decode.restype = _i
    L.tkm_attn_kv_evict.argtypes = [kv, kv, _vp, _i, _i, _i, _vp]
    L.tkm_attn_kv_evict.restype = _i
    ll, rope, plan = ctypes.c_longlong, ctypes.POINTER(_Rope), ctypes.POINTER(_Plan)
    L.tkm_attn_rope_init.argtypes = [ctypes.POINTER(_RopeParams), rope]
    L.tkm_attn_rope_init.restype = _i
    L.tkm_attn_rope_from_freqs.argtypes = [ctypes.POINTER(ctypes.c_double), _i, _i, ctypes.c_double, rope]
    L.tkm_attn_rope_from_freqs.restype = _i
    L.tkm_attn_rope_rows.argtypes = [rope, _vp, ll, _vp, ll, _vp] + [_i] * 7 + [_vp]
    L.tkm_attn_rope_rows.restype = _i
    L.tkm_attn_kv_plan.argtypes = [kv, ctypes.POINTER(_Pages), _vp, _vp, plan, _i, _vp]
    L.tkm_attn_kv_plan.restype = _i
    L.tkm_attn_kv_append_rows.argtypes = [kv, rope, _vp, ll, _vp, ll, plan, _i, _i, _vp]
    L.tkm_attn_kv_append_rows.restype = _i
    L.tkm_attn_chunk_workspace_bytes.argtypes = [kv, _i, _i]
    L.tkm_attn_chunk_workspace_bytes.restype = ctypes.c_size_t
    L.tkm_attn_chunk.argtypes = [kv, _vp, ll, _vp, _vp, _i, _vp, _vp, _i, ctypes.c_float, _i, _i, _vp, ctypes.c_size_t, _vp]
    L.tkm_attn_chunk.restype = _i
    _lib = L
    return L


# Bits of tkm_attn_last_kernels (include/tkm_attn.h)
KERNEL_BITS = {"fwd_asm": 1, "fwd_hip": 2, "dq_asm": 4, "dq_hip": 8, "dkdv_asm": 16,
               "dkdv_hip": 32, "delta_hip": 64, "decode": 128, "join": 256, "weights": 512, "append": 1024,
               "evict": 2048, "rope": 4096, "plan": 8192, "chunk": 16384}


def init() -> None:
    """Load the gfx950 assembly kernels on the current device (tkm_attn_init); raises if a
    code object fails to load."""
    _check("tkm_attn_init", lib().tkm_attn_init())


def asm_available() -> bool:
    return bool(lib().tkm_attn_asm_available())


def last_kernels() -> list:
    """Names of the kernels the calling thread's last tkm_attn_* call launched."""
    bits = int(lib().tkm_attn_last_kernels())
    return [n for n, b in KERNEL_BITS.items() if bits & b]


def _check(fn: str, rc: int, L=None) -> None:
    if rc != 0:
        raise AttnError(fn, rc, (L or lib()).tkm_attn_last_error().decode())


@functools.lru_cache(maxsize=64)
def default_scale(D: int) -> float:
    """1/sqrtf(D) in fp32, as the reference dispatch passes (tkm_gpu.cu:1258)."""
    import numpy as np
    return float(np.float32(1.0) / np.sqrt(np.float32(D)))


def _dtype_code(t) -> int:
    import torch
    if t.dtype == torch.float16:
        return F16
    if t.dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"attention tensors must be float16 or bfloat16, got {t.dtype}")


# Addresses go to ctypes as plain ints (c_void_p argtypes take them), and the current stream's handle
# comes from torch's C entry: the wrapper objects cost more host time than a small call's kernels.
def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(stream):
    if stream is not None:
        return stream.cuda_stream
    import torch
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _check_tensor(name, t, numel, device, dtype=None):
    if (t.is_cuda and t.numel() == numel and t.is_contiguous() and (dtype is None or t.dtype == dtype)
            and t.device == device):
        return
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.numel() != numel:
        raise ValueError(f"{name} has {t.numel()} elements, expected {numel}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")


def gqa_fwd(qkv, B, S, Hq, Hkv, D, causal=True, kv_len=None, scale=None,
            out=None, lse=None, stream=None):
    """O [B,S,Hq*D] and LSE [B,Hq,S] (fp32) of packed qkv [B,S,(Hq+2Hkv)*D]."""
    import torch
    dev = qkv.device
    _check_tensor("qkv", qkv, B * S * (Hq + 2 * Hkv) * D, dev)
    dt = _dtype_code(qkv)
    if out is None:
        out = torch.empty((B, S, Hq * D), dtype=qkv.dtype, device=dev)
    else:
        _check_tensor("out", out, B * S * Hq * D, dev, qkv.dtype)
    if lse is None:
        lse = torch.empty((B, Hq, S), dtype=torch.float32, device=dev)
    else:
        _check_tensor("lse", lse, B * Hq * S, dev, torch.float32)
    if kv_len is not None:
        _check_tensor("kv_len", kv_len, B, dev, torch.int32)
    scale = default_scale(D) if scale is None else float(scale)
    rc = lib().tkm_attn_fwd(_ptr(qkv), _ptr(out), _ptr(lse), _ptr(kv_len), B, S, Hq, Hkv, D,
                            scale, int(bool(causal)), dt, _stream(stream))
    _check("tkm_attn_fwd", rc)
    return out, lse


def bwd_workspace_bytes(B, S, Hq) -> int:
    return int(lib().tkm_attn_bwd_workspace_bytes(B, S, Hq))


def gqa_bwd(qkv, o, dout, lse, B, S, Hq, Hkv, D, causal=True, kv_len=None, scale=None,
            dqkv=None, workspace=None, stream=None, stage=None):
    """dqkv [B,S,(Hq+2Hkv)*D] (dQ | dK | dV); stage selects one backward kernel."""
    import torch
    dev = qkv.device
    _check_tensor("qkv", qkv, B * S * (Hq + 2 * Hkv) * D, dev)
    _check_tensor("o", o, B * S * Hq * D, dev, qkv.dtype)
    _check_tensor("dout", dout, B * S * Hq * D, dev, qkv.dtype)
    _check_tensor("lse", lse, B * Hq * S, dev, torch.float32)
    if kv_len is not None:
        _check_tensor("kv_len", kv_len, B, dev, torch.int32)
    dt = _dtype_code(qkv)
    if dqkv is None:
        dqkv = torch.empty_like(qkv)
    else:
        _check_tensor("dqkv", dqkv, qkv.numel(), dev, qkv.dtype)
    if workspace is None:
        wbytes = bwd_workspace_bytes(B, S, Hq)
        workspace = torch.empty(wbytes, dtype=torch.uint8, device=dev)
    else:
        wbytes = workspace.numel() * workspace.element_size()
    scale = default_scale(D) if scale is None else float(scale)
    args = (_ptr(qkv), _ptr(o), _ptr(dout), _ptr(lse), _ptr(dqkv), _ptr(kv_len), B, S, Hq, Hkv,
            D, scale, int(bool(causal)), dt, _ptr(workspace), wbytes, _stream(stream))
    if stage is None:
        _check("tkm_attn_bwd", lib().tkm_attn_bwd(*args))
    else:
        _check("tkm_attn_bwd_stage", lib().tkm_attn_bwd_stage(int(stage), *args))
    return dqkv


class _Handle:
    """Of tensors whose addresses a C struct holds: an attribute that has been set stays, for a tensor in its place would
    leave the struct with the address of memory that may be freed."""

    def __setattr__(self, name, value):
        if name in self.__dict__ and value is not self.__dict__[name]:     # c.kv_len += 1 ends in c.kv_len = c.kv_len
            raise AttributeError(f"{name} cannot be replaced: write into the tensor")
        super().__setattr__(name, value)


class KvCache(_Handle):
    """A paged key-value cache over the caller's tensors (tkm_attn_kv, include/tkm_attn.h):

    k       [num_pages, Hkv, page/32, D/32, 32, 32]  float16 or bfloat16, blocks of 32 tokens x 32 dims
    v       the same shape, its blocks 32 dims x 32 tokens
    table   [B, max_pages] int32: the pages of each sequence
    kv_len  [B] int32: the tokens each sequence holds
    weight  [B, Hkv, max_pages * page] float32 or None: attention weight gathered by each position

    The tensors stay the caller's, and are attributes here: write into them (a new page into the table, 0 into
    kv_len for a slot that starts anew), do not replace them.  Caches may share a pool (k, v)."""

    def __init__(self, k, v, table, kv_len, weight=None):
        dev = k.device
        if k.dim() != 6 or tuple(k.shape[4:]) != (32, 32) or v.shape != k.shape:
            raise ValueError("k and v must be [num_pages, Hkv, page/32, D/32, 32, 32]")
        if table.dim() != 2:
            raise ValueError("table must be [B, max_pages]")
        dt = _dtype_code(k)
        num_pages, Hkv, page, D = k.shape[0], k.shape[1], 32 * k.shape[2], 32 * k.shape[3]
        B, max_pages = table.shape
        _check_tensor("k", k, k.numel(), dev)
        _check_tensor("v", v, k.numel(), dev, k.dtype)
        _check_dtype("table", table, B * max_pages, dev, "int32")
        _check_dtype("kv_len", kv_len, B, dev, "int32")
        if weight is not None:
            _check_dtype("weight", weight, B * Hkv * max_pages * page, dev, "float32")
        self.k, self.v, self.table, self.kv_len, self.weight = k, v, table, kv_len, weight
        self.B, self.Hkv, self.D, self.page, self.max_pages, self.num_pages = B, Hkv, D, page, max_pages, num_pages
        self.dtype, self.device = k.dtype, dev
        self._c = _Kv(_ptr(k), _ptr(v), _ptr(table), _ptr(kv_len), _ptr(weight), B, Hkv, D, page, max_pages, num_pages, dt)
        self._ref = ctypes.byref(self._c)
        self._ws = {}

    @classmethod
    def empty(cls, B, max_pages, num_pages, Hkv, D, page=64, dtype=None, device="cuda", weights=False):
        """A cache of sequences without tokens; every table entry is -1 until the caller names a page."""
        import torch
        if page % 32 or D % 32:
            raise ValueError("page and D must be multiples of 32")
        blocks = (num_pages, Hkv, page // 32, D // 32, 32, 32)
        k, v = (torch.empty(blocks, dtype=dtype or torch.float16, device=device) for _ in range(2))
        return cls(k, v, torch.full((B, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(B, dtype=torch.int32, device=device),
                   torch.zeros((B, Hkv, max_pages * page), device=device) if weights else None)


def _check_dtype(name, t, numel, device, dtype):
    import torch
    _check_tensor(name, t, numel, device, getattr(torch, dtype))


class _On:
    """Where a call on tensors of one device launches and allocates: the device, which need not be the current
    one, on its current stream or the given one, which has to be that device's."""
    __slots__ = ("handle", "ctx")

    def __init__(self, device, stream):
        import torch
        if stream is not None and stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors are on {device}")
        self.ctx = torch.cuda.device(device) if stream is None else torch.cuda.stream(stream)
        self.handle = torch._C._cuda_getCurrentRawStream(device.index) if stream is None else stream.cuda_stream

    def __enter__(self):
        self.ctx.__enter__()
        return self.handle

    def __exit__(self, *a):
        return self.ctx.__exit__(*a)


def _current(device, stream):
    """The current stream's handle, or None if the call has to change device or stream (_On) first."""
    if stream is not None:
        return None
    import torch
    return torch._C._cuda_getCurrentRawStream(device.index) if torch._C._cuda_getDevice() == device.index else None


def kv_append(qkv, cache, Hq, start=None, n_new=None, stream=None):
    """Stores the K and V rows of packed qkv [B, S, (Hq+2Hkv)*D] (or [B, (Hq+2Hkv)*D]: one row a sequence) behind
    what the cache holds, or from positions start [B] int32 on; kv_len becomes the start plus n_new [B] int32
    (None: S) rows.  Page the table first: rows on positions without a page are dropped."""
    st = _current(cache.device, stream)
    if st is None:
        with _On(cache.device, stream) as st:
            return _kv_append(qkv, cache, Hq, start, n_new, st)
    return _kv_append(qkv, cache, Hq, start, n_new, st)


def _kv_append(qkv, cache, Hq, start, n_new, st):
    dev, B = cache.device, cache.B
    row = B * (Hq + 2 * cache.Hkv) * cache.D
    n = qkv.numel()
    S = n // row if row > 0 else 0
    _check_tensor("qkv", qkv, S * row if S else row, dev, cache.dtype)
    if start is not None:
        _check_tensor("start", start, B, dev, cache.kv_len.dtype)
    if n_new is not None:
        _check_tensor("n_new", n_new, B, dev, cache.kv_len.dtype)
    _check("tkm_attn_kv_append", lib().tkm_attn_kv_append(cache._ref, qkv.data_ptr(), S, Hq, _ptr(start), _ptr(n_new), st))


def decode_workspace_bytes(cache, Hq, add_weights=False) -> int:
    key = (Hq, bool(add_weights))
    if key not in cache._ws:
        cache._ws[key] = int(lib().tkm_attn_decode_workspace_bytes(cache._ref, Hq, int(key[1])))
    return cache._ws[key]


def gqa_decode(q, cache, Hq, scale=None, out=None, lse=None, add_weights=False, workspace=None, stream=None):
    """O [B, Hq*D] and LSE [B, Hq] (fp32) of one query row a sequence over the cache.  q: [B, >= Hq*D] with the Q
    heads first, rows any multiple of 8 elements apart; the packed row of the new token does as it is.
    add_weights: also add the softmax weights of every cached position to cache.weight.
    workspace: decode_workspace_bytes(cache, Hq, add_weights) bytes, allocated for the call if not given; with
    add_weights these are over B * Hq * 4 bytes for every position that the table can hold."""
    st = _current(cache.device, stream)
    if st is None:
        with _On(cache.device, stream) as st:
            return _gqa_decode(q, cache, Hq, scale, out, lse, add_weights, workspace, st)
    return _gqa_decode(q, cache, Hq, scale, out, lse, add_weights, workspace, st)


def _gqa_decode(q, cache, Hq, scale, out, lse, add_weights, workspace, st):
    import torch
    B, D, dev = cache.B, cache.D, cache.device
    rows, stride = q.shape, q.stride()
    if len(rows) != 2 or rows[0] != B or rows[1] < Hq * D or stride[1] != 1:
        raise ValueError(f"q must be [{B}, at least {Hq * D}] with contiguous rows")
    if q.device != dev or q.dtype != cache.dtype:
        raise ValueError(f"q must be {cache.dtype} on {dev}")
    if out is None:
        out = q.new_empty((B, max(0, Hq * D)))
    else:
        _check_tensor("out", out, B * Hq * D, dev, q.dtype)
    if lse is None:
        lse = torch.empty((B, max(0, Hq)), dtype=torch.float32, device=dev)
    else:
        _check_tensor("lse", lse, B * Hq, dev, torch.float32)
    if workspace is None:
        wbytes = decode_workspace_bytes(cache, Hq, add_weights)
        if wbytes:
            workspace = torch.empty(wbytes, dtype=torch.uint8, device=dev)
    else:
        _check_tensor("workspace", workspace, workspace.numel(), dev)
        wbytes = workspace.numel() * workspace.element_size()
    rc = lib().tkm_attn_decode(cache._ref, q.data_ptr(), stride[0] if B > 1 else Hq * D, out.data_ptr(), lse.data_ptr(), Hq,
                               default_scale(D) if scale is None else scale, 1 if add_weights else 0, _ptr(workspace),
                               wbytes, st)
    if rc:
        _check("tkm_attn_decode", rc)
    return out, lse


def kv_evict(cache, budget, sink=0, recent=0, dst=None, kept=None, stream=None):
    """Cuts sequences of more than `budget` tokens to the first `sink`, the last `recent` and, of the others, those
    with the largest cache.weight, each kv head by its own; in place, or into the cache `dst` (faster).  Returns kept
    [B, Hkv, budget] int32: the old position of each new one, -1 behind the last."""
    st = _current(cache.device, stream)
    if st is None:
        with _On(cache.device, stream) as st:
            return _kv_evict(cache, budget, sink, recent, dst, kept, st)
    return _kv_evict(cache, budget, sink, recent, dst, kept, st)


def _kv_evict(cache, budget, sink, recent, dst, kept, st):
    if dst is not None and dst.device != cache.device:
        raise ValueError(f"dst must be on {cache.device}")
    if kept is None:
        kept = cache.kv_len.new_empty((cache.B, cache.Hkv, max(0, budget)))
    else:
        _check_tensor("kept", kept, cache.B * cache.Hkv * budget, cache.device, cache.kv_len.dtype)
    _check("tkm_attn_kv_evict", lib().tkm_attn_kv_evict(cache._ref, None if dst is None else dst._ref, kept.data_ptr(), budget,
                                                        sink, recent, st))
    return kept


ROPE_CLEAR = 256      # TKM_ROPE_CLEAR


class Rope:
    """Rotary positions (tkm_attn_rope, include/tkm_attn.h): the first `rot` dims of a head turn, pair i by freqs[i]
    radians a position.

    layout   "halves" (dims i and i + rot/2) or "pairs" (2i and 2i + 1)
    scaling  None, or "linear", "ntk", "bands", "yarn": for contexts `scale` times longer than the `original` ones of
             training; low and high: turns over the original context (bands 1 and 4, yarn 1 and 32 if not given)
    factor   of the rotated dims; None: the scaling's own
    freqs    rot/2 frequencies in place of theta and scaling"""

    LAYOUTS = {"halves": 0, "pairs": 1}
    SCALINGS = {None: 0, "linear": 1, "ntk": 2, "bands": 3, "yarn": 4}

    def __init__(self, rot, theta=10000.0, layout="halves", scaling=None, scale=1.0, original=8192.0, low=None, high=None,
                 factor=None, freqs=None):
        if layout not in self.LAYOUTS:
            raise ValueError(f"layout must be one of {list(self.LAYOUTS)}, got {layout!r}")
        if scaling not in self.SCALINGS:
            raise ValueError(f"scaling must be one of {list(self.SCALINGS)}, got {scaling!r}")
        self._c = _Rope()
        self._ref = ctypes.byref(self._c)
        if freqs is not None:
            if scaling is not None:
                raise ValueError("freqs are taken as they are: scale them, and leave scaling out")
            freqs = [float(f) for f in freqs]
            if 2 * len(freqs) != rot:
                raise ValueError(f"{len(freqs)} frequencies for {rot} rotated dims")
            _check("tkm_attn_rope_from_freqs", lib().tkm_attn_rope_from_freqs(
                (ctypes.c_double * len(freqs))(*freqs), rot, self.LAYOUTS[layout], factor or 0.0, self._ref))
        else:
            p = _RopeParams(rot, self.LAYOUTS[layout], self.SCALINGS[scaling], theta, scale, original, 1.0 if low is None else low,
                            (32.0 if scaling == "yarn" else 4.0) if high is None else high, factor or 0.0)
            _check("tkm_attn_rope_init", lib().tkm_attn_rope_init(ctypes.byref(p), self._ref))

    @classmethod
    def of_prep(cls, desc):
        """The rotation of a qkv-prep descriptor (prep.Desc with RoPE): its frequencies, pairs over the whole head."""
        from . import prep
        r = cls.__new__(cls)
        r._c = _Rope()
        r._ref = ctypes.byref(r._c)
        _check("tkm_prep_rope", prep.lib().tkm_prep_rope(ctypes.byref(desc), r._ref))
        return r

    rot = property(lambda self: self._c.rot)
    factor = property(lambda self: self._c.factor)

    def freqs(self):
        """The frequencies as they are held, modulo a whole turn a position: floats in [0, 2 pi)."""
        return [t * (2.0 * math.pi / 2.0 ** 64) for t in self._c.turns[:self._c.rot // 2]]


def rope_fwd(x, rope, Hq, Hkv, D, pos=None, S=None, out=None, stream=None):
    """Rotates the Q and K heads of packed rows x [..., (Hq+2Hkv)*D] (rows any multiple of 8 elements apart in a 2-D
    x) to the positions pos [rows] int32, or, if these are None, to r % S of the row r; V is copied.  A row of a
    negative position stays as it is in a given out (x itself: in place), and is 0 in a new one."""
    return _rope_on(x, rope, Hq, Hkv, D, pos, S, out, 0, stream)


def rope_bwd(dout, rope, Hq, Hkv, D, pos=None, S=None, dx=None, stream=None):
    """The gradient of rope_fwd's x from that of its output: the rotation the other way.  Rows of negative positions as
    there."""
    return _rope_on(dout, rope, Hq, Hkv, D, pos, S, dx, 1, stream)


def _rope_on(x, rope, Hq, Hkv, D, pos, S, out, inverse, stream):
    st = _current(x.device, stream) if x.is_cuda else None
    if st is None:
        if not x.is_cuda:
            raise ValueError("the rows must be on a GPU")
        with _On(x.device, stream) as st:
            return _rope(x, rope, Hq, Hkv, D, pos, S, out, inverse, st)
    return _rope(x, rope, Hq, Hkv, D, pos, S, out, inverse, st)


def _rows_of(name, t, width, device, dtype, least=False):
    """(rows, stride in elements) of a tensor of rows: 2-D with contiguous rows, or contiguous."""
    if t.device != device or t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} on {device}")
    shape = t.shape
    if len(shape) == 0 or (shape[-1] < width if least else shape[-1] != width):
        raise ValueError(f"{name} must have rows of {'at least ' if least else ''}{width} elements")
    n = t.numel() // shape[-1] if shape[-1] else 0
    if len(shape) == 2:
        if t.stride(1) != 1 and shape[1] > 1:
            raise ValueError(f"{name} must have contiguous rows")
        return n, t.stride(0) if n > 1 else (shape[1] + 7) // 8 * 8
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, or of two dimensions")
    return n, shape[-1]


def _rope(x, rope, Hq, Hkv, D, pos, S, out, inverse, st):
    dt, dev, width = _dtype_code(x), x.device, (Hq + 2 * Hkv) * D
    rows, stride = _rows_of("x", x, width, dev, x.dtype)
    if pos is None:
        if S is None:
            raise ValueError("rows need positions, or the S rows of a sequence")
    else:
        _check_dtype("pos", pos, rows, dev, "int32")
    if out is None:
        out, ostride = x.new_empty(x.shape), width
        inverse |= ROPE_CLEAR
    else:
        n, ostride = _rows_of("out", out, width, dev, x.dtype)
        if n != rows:
            raise ValueError(f"out has {n} rows, expected {rows}")
    _check("tkm_attn_rope_rows", lib().tkm_attn_rope_rows(rope._ref, x.data_ptr(), stride, out.data_ptr(), ostride, _ptr(pos),
                                                          1 if S is None else S, rows, Hq, Hkv, D, dt, inverse, st))
    return out


class KvPages(_Handle):
    """The pages of a pool that no sequence has, and how many each sequence has (tkm_attn_pages): free [num_pages]
    int32, of which the first n_free [1] int32 are free, and held [B] int32.  The tensors stay the caller's, and are
    attributes here: write into them, do not replace them."""

    def __init__(self, free, n_free, held):
        dev = held.device
        _check_dtype("free", free, free.numel(), dev, "int32")
        _check_dtype("n_free", n_free, 1, dev, "int32")
        _check_dtype("held", held, held.numel(), dev, "int32")
        self.free, self.n_free, self.held, self.device = free, n_free, held, dev
        self._c = _Pages(_ptr(free), _ptr(n_free), _ptr(held))
        self._ref = ctypes.byref(self._c)

    @classmethod
    def all_free(cls, cache):
        """Of a cache whose sequences have no pages yet: page 0 is taken first."""
        import torch
        dev, n = cache.device, cache.num_pages
        return cls(torch.arange(n - 1, -1, -1, dtype=torch.int32, device=dev), torch.full((1,), n, dtype=torch.int32, device=dev),
                   torch.zeros(cache.B, dtype=torch.int32, device=dev))


class KvPlan(_Handle):
    """What a step does (tkm_attn_plan), written by kv_plan: n_new [B], row_start [B + 1], and per packed row seq, pos
    [rows], all int32, and slot [rows] int64; write into them, do not replace them."""

    def __init__(self, n_new, row_start, seq, pos, slot):
        dev, B, rows = n_new.device, n_new.numel(), slot.numel()
        _check_dtype("n_new", n_new, B, dev, "int32")
        _check_dtype("row_start", row_start, B + 1, dev, "int32")
        _check_dtype("seq", seq, rows, dev, "int32")
        _check_dtype("pos", pos, rows, dev, "int32")
        _check_dtype("slot", slot, rows, dev, "int64")
        self.n_new, self.row_start, self.seq, self.pos, self.slot = n_new, row_start, seq, pos, slot
        self.B, self.rows, self.device = B, rows, dev
        self._c = _Plan(_ptr(n_new), _ptr(row_start), _ptr(seq), _ptr(pos), _ptr(slot))
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, B, rows, device="cuda"):
        import torch
        i32 = [torch.empty(n, dtype=torch.int32, device=device) for n in (B, B + 1, rows, rows)]
        return cls(*i32, torch.empty(rows, dtype=torch.int64, device=device))


def kv_plan(cache, pages, want, rows=None, start=None, plan=None, stream=None):
    """Makes room for want [B] int32 more tokens of each sequence behind start [B] int32 (None: kv_len itself), takes
    pages from the pool and gives back what sequences no longer need, advances kv_len, and lays out the step's packed
    rows, at most `rows` of them (or as many as the given plan has).  A sequence whose pages or rows are not there gets
    none: its plan.n_new is 0.  From the first whose rows do not fit on, none gets any: cut a want of more than `rows`
    into pieces.  include/tkm_attn.h has the rules.  Returns the plan."""
    st = _current(cache.device, stream)
    if st is None:
        with _On(cache.device, stream) as st:
            return _kv_plan(cache, pages, want, rows, start, plan, st)
    return _kv_plan(cache, pages, want, rows, start, plan, st)


def _kv_plan(cache, pages, want, rows, start, plan, st):
    dev, B = cache.device, cache.B
    if plan is None:
        if rows is None or rows < 0:
            raise ValueError("a plan of how many rows?")
        plan = KvPlan.empty(B, rows, dev)
    elif rows is not None and rows != plan.rows:
        raise ValueError(f"the plan has {plan.rows} rows, not {rows}")
    if pages.device != dev or plan.device != dev:
        raise ValueError(f"pages and plan must be on {dev}")
    if pages.held.numel() != B or plan.B != B or pages.free.numel() != cache.num_pages:
        raise ValueError(f"pages and plan must be of {B} sequences and {cache.num_pages} pages")
    _check_tensor("want", want, B, dev, cache.kv_len.dtype)
    if start is not None:
        _check_tensor("start", start, B, dev, cache.kv_len.dtype)
    _check("tkm_attn_kv_plan", lib().tkm_attn_kv_plan(cache._ref, pages._ref, want.data_ptr(), _ptr(start), plan._ref, plan.rows, st))
    return plan


def kv_append_rows(qkv, cache, Hq, plan, rope=None, q=None, stream=None):
    """Stores the K and V heads of a plan's packed rows qkv [rows, (Hq+2Hkv)*D] in their slots of the cache, K rotated
    to its position if there is a rope, and returns the Q heads [rows, >= Hq*D], rotated too: a new tensor, whose rows
    of no sequence hold anything, or the given q (qkv itself: in place; without a rope and q they stay where they are).
    kv_len is the plan's business."""
    st = _current(cache.device, stream)
    if st is None:
        with _On(cache.device, stream) as st:
            return _kv_append_rows(qkv, cache, Hq, plan, rope, q, st)
    return _kv_append_rows(qkv, cache, Hq, plan, rope, q, st)


def _kv_append_rows(qkv, cache, Hq, plan, rope, q, st):
    dev, D = cache.device, cache.D
    rows, stride = _rows_of("qkv", qkv, (Hq + 2 * cache.Hkv) * D, dev, cache.dtype)
    if plan.device != dev or plan.rows != rows:
        raise ValueError(f"the plan must be of {rows} rows, on {dev}")
    if q is None:
        q = qkv if rope is None else qkv.new_empty((rows, max(0, Hq * D)))
    n, q_stride = _rows_of("q", q, Hq * D, dev, cache.dtype, least=True)
    if n != rows:
        raise ValueError(f"q has {n} rows, expected {rows}")
    if rows < 2:
        q_stride = stride      # a single row has none of its own: in place it may be of another width
    _check("tkm_attn_kv_append_rows", lib().tkm_attn_kv_append_rows(
        cache._ref, None if rope is None else rope._ref, qkv.data_ptr(), stride, q.data_ptr(), q_stride, plan._ref, rows, Hq, st))
    return q


def chunk_workspace_bytes(cache, rows, Hq) -> int:
    key = ("chunk", rows, Hq)
    if key not in cache._ws:
        if len(cache._ws) > 256:
            cache._ws.clear()
        cache._ws[key] = int(lib().tkm_attn_chunk_workspace_bytes(cache._ref, rows, Hq))
    return cache._ws[key]


def gqa_chunk(q, cache, Hq, row_start=None, n_new=None, scale=None, causal=True, window=0, out=None, lse=None, workspace=None,
              stream=None):
    """O [rows, Hq*D] and LSE [rows, Hq] (fp32) of each sequence's new rows over its cached positions, their own
    among them (append first).  q: [rows, >= Hq*D] with the Q heads first.  Sequence b has n_new[b] int32 rows from
    row_start[b] int32 on (a plan's; row_start None: at most rows / B from b * (rows / B), n_new None: rows / B), and the
    last of them stands at its last position.  causal: a row sees the positions up to its own, with a window only the last `window`
    of these.  Rows of no sequence stay as they are in out and lse (in new ones they hold anything); without rows
    nothing is launched.  No weights are gathered: eviction by weight needs gqa_decode's add_weights.
    workspace: chunk_workspace_bytes(cache, rows, Hq) bytes, allocated for the call if not given."""
    st = _current(cache.device, stream)
    if st is None:
        with _On(cache.device, stream) as st:
            return _gqa_chunk(q, cache, Hq, row_start, n_new, scale, causal, window, out, lse, workspace, st)
    return _gqa_chunk(q, cache, Hq, row_start, n_new, scale, causal, window, out, lse, workspace, st)


def _gqa_chunk(q, cache, Hq, row_start, n_new, scale, causal, window, out, lse, workspace, st):
    import torch
    D, dev, B = cache.D, cache.device, cache.B
    if len(q.shape) != 2:
        raise ValueError(f"q must be [rows, at least {Hq * D}]")
    rows, stride = _rows_of("q", q, Hq * D, dev, cache.dtype, least=True)
    i32 = cache.kv_len.dtype
    if row_start is not None and not B <= row_start.numel() <= B + 1:
        raise ValueError(f"row_start must have {B} entries, or {B + 1}")
    if row_start is not None:
        _check_tensor("row_start", row_start, row_start.numel(), dev, i32)
    if n_new is not None:
        _check_tensor("n_new", n_new, B, dev, i32)
    if out is None:
        out = q.new_empty((rows, max(0, Hq * D)))
    else:
        _check_tensor("out", out, rows * Hq * D, dev, q.dtype)
    if lse is None:
        lse = torch.empty((rows, max(0, Hq)), dtype=torch.float32, device=dev)
    else:
        _check_tensor("lse", lse, rows * Hq, dev, torch.float32)
    if rows == 0:
        return out, lse
    if workspace is None:
        wbytes = chunk_workspace_bytes(cache, rows, Hq)
        if wbytes:
            workspace = torch.empty(wbytes, dtype=torch.uint8, device=dev)
    else:
        _check_tensor("workspace", workspace, workspace.numel(), dev)
        wbytes = workspace.numel() * workspace.element_size()
    rc = lib().tkm_attn_chunk(cache._ref, q.data_ptr(), stride, _ptr(row_start), _ptr(n_new), rows, out.data_ptr(), lse.data_ptr(), Hq,
                              default_scale(D) if scale is None else scale, 1 if causal else 0, window, _ptr(workspace), wbytes, st)
    if rc:
        _check("tkm_attn_chunk", rc)
    return out, lse


def attention_flops(B, S, Hq, D, causal, kv_len=None, mode="fwd") -> float:
    """Algorithmic FLOPs (FlashAttention convention): 4*B*Hq*S*Skv*D, halved if causal,
    x2.5 for the backward, x3.5 for forward+backward; with kv_len, S*Skv -> S*mean(kv_len)."""
    skv = S if kv_len is None else sum(int(x) for x in kv_len) / len(kv_len)
    f = 4.0 * B * Hq * S * skv * D * (0.5 if causal else 1.0)
    return {"fwd": f, "bwd": 2.5 * f, "fwdbwd": 3.5 * f}[mode]


__all__ = ["gqa_fwd", "gqa_bwd", "KvCache", "kv_append", "gqa_decode", "kv_evict", "decode_workspace_bytes", "Rope", "rope_fwd", "rope_bwd", "KvPages", "KvPlan", "kv_plan", "kv_append_rows",
           "gqa_chunk", "chunk_workspace_bytes", "init", "asm_available", "last_kernels", "KERNEL_BITS", "bwd_workspace_bytes", "attention_flops", "default_scale",
           "lib", "header_functions", "AttnError", "F16", "BF16", "BWD_DELTA", "BWD_DKDV",
           "BWD_DQ", "BWD_DQ_DELTA"]
