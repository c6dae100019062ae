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
    _lib = L
    return L


# Bits of tkm_attn_last_kernels (include/tkm_attn.h)
KERNEL_BITS = {"fwd_asm": 1, "fwd_hip": 2, "dq_asm": 4, "dq_hip": 8, "dkdv_asm": 16,
               "dkdv_hip": 32, "delta_hip": 64, "decode": 128, "join": 256, "weights": 512, "append": 1024,
               "evict": 2048}


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


class KvCache:
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

    def __setattr__(self, name, value):
        if name in self.__dict__ and value is not self.__dict__[name]:     # c.kv_len += 1 ends in c.kv_len = c.kv_len
            raise AttributeError(f"{name} cannot be replaced: write into the tensor")
        super().__setattr__(name, value)

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


def attention_flops(B, S, Hq, D, causal, kv_len=None, mode="fwd") -> float:
    """Algorithmic FLOPs (FlashAttention convention): 4*B*Hq*S*Skv*D, halved if causal,
    x2.5 for the backward, x3.5 for forward+backward; with kv_len, S*Skv -> S*mean(kv_len)."""
    skv = S if kv_len is None else sum(int(x) for x in kv_len) / len(kv_len)
    f = 4.0 * B * Hq * S * skv * D * (0.5 if causal else 1.0)
    return {"fwd": f, "bwd": 2.5 * f, "fwdbwd": 3.5 * f}[mode]


__all__ = ["gqa_fwd", "gqa_bwd", "KvCache", "kv_append", "gqa_decode", "kv_evict", "decode_workspace_bytes", "init", "asm_available", "last_kernels", "KERNEL_BITS", "bwd_workspace_bytes", "attention_flops", "default_scale",
           "lib", "header_functions", "AttnError", "F16", "BF16", "BWD_DELTA", "BWD_DKDV",
           "BWD_DQ", "BWD_DQ_DELTA"]
