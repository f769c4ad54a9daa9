"""Four-bit matrices and token caches, over the C ABI: the fully connected products and the attention of a network that answers token by token.

    m = quantize_weights4(weights, group)              # load time: codes and (scale, low) pairs
    y = forward_connected4(m, x, biases, activation)   # forward_connected_layer (src-lib/connected_layer.cpp) for a few rows
    c = new_cache4(pages, kv_heads, page, dim, group)
    append4(c, k, v, table, lengths)                   # the newest tokens of every sequence into their pages
    out = attend4(c, q, table, lengths)                # their attention over all that their sequences hold

The format, and what a row of tokens stands for, are written down in include/xnor_b200.h.  torch is used for device memory and the
current stream only; every computation is a call into libxnor_b200.so.  Nothing here has a CPU path.  Calls are asynchronous, run on the
current stream of the tensors' device and may be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import torch

from . import capi

_DTYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_GROUPS = (32, 64, 128)

# A decoding step is a few small kernels, so what a call costs on the host counts: its structs are packed as bytes, in the layout of
# capi's (which takes a third of the time that filling those takes), and its checks are one expression each; only when that fails
# _refuse_* look for the fault.
_CACHE, _ROWS, _TENSOR = struct.Struct("=QQQQiiiii4x").pack, struct.Struct("=iii4xQQQ").pack, struct.Struct("=Qi4xqqq").pack
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


class _Calls:
    """The library's entry points, as functions that take packed structs."""

    def __getattr__(self, name: str):
        vp, ci, ll = C.c_void_p, C.c_int, C.c_longlong
        for entry, args in (("w4_forward", [vp, vp, ci, ci, ll, vp, vp, vp, vp, ll, vp, C.c_size_t, vp]), ("w4_scratch_bytes", [vp, ci, ci]), ("kv4_append", [vp] * 5), ("kv4_read", [vp] * 5),
                            ("kv4_attend", [vp, vp, vp, ci, C.c_float, ci, vp, vp, vp, C.c_size_t, vp]),
                            ("kv4_attend_scratch_bytes", [vp, vp, ci, ci])):
            f = capi.lib()["xnor_b200_" + entry]
            f.argtypes = args
            f.restype = C.c_size_t if entry.endswith("bytes") else ci
            setattr(self, entry, f)
        return object.__getattribute__(self, name)


_calls = _Calls()


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be fp32, fp16 or bf16, not {t.dtype}")
    return code


def _on(device: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {t.device} and {device}: all of a call's tensors are on one CUDA device")
    if device.type != "cuda":
        raise ValueError(f"tensors on {device}: this path runs on a CUDA device only")


class _Fixed:
    """What a handle was made of and checked for stays what it is."""

    def __setattr__(self, name, value):
        raise AttributeError(f"{type(self).__name__} keeps the buffers and sizes that it was made with: make another")


class Matrix4(_Fixed):
    """A packed matrix of n rows of k values (struct xnor_b200_w4_desc with its two buffers): codes uint8 [n][ceil(k/32)*16], scales fp16
    [n][ceil(k/group)][2], both contiguous."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, k: int, group: int) -> None:
        if group not in _GROUPS:
            raise ValueError(f"group must be one of {_GROUPS}, not {group}")
        if codes.dim() != 2 or codes.dtype != torch.uint8 or k <= 0 or codes.shape[0] == 0 or codes.shape[1] != (k + 31) // 32 * 16 or not codes.is_contiguous():
            raise ValueError(f"codes must be contiguous uint8 [n][{(k + 31) // 32 * 16}] for rows of {k} values")
        if scales.dtype != torch.float16 or scales.shape != (codes.shape[0], (k + group - 1) // group, 2) or not scales.is_contiguous():
            raise ValueError(f"scales must be contiguous fp16 [{codes.shape[0]}][{(k + group - 1) // group}][2]")
        if scales.device != codes.device:
            raise ValueError(f"codes on {codes.device}, scales on {scales.device}")
        self.__dict__.update(codes=codes, scales=scales, n=codes.shape[0], k=k, group=group, device=codes.device, _index=codes.get_device(),
                             _descs={a: bytes(capi.W4Desc(codes.shape[0], k, group, a)) for a in (capi.LINEAR, capi.LEAKY)})


def quantize_weights4(weights: torch.Tensor, group: int) -> Matrix4:
    """Packs a matrix [n][k] (rows contiguous) to four bits: xnor_b200_w4_quantize."""
    if weights.dim() != 2 or weights.numel() == 0 or (weights.stride(1) != 1 and weights.shape[1] != 1):
        raise ValueError("weights must be a matrix [n][k] with contiguous rows")
    if group not in _GROUPS:
        raise ValueError(f"group must be one of {_GROUPS}, not {group}")
    n, k = weights.shape
    dtype = _dtype(weights, "weights")
    _on(weights.device)
    with torch.cuda.device(weights.device):
        codes = torch.empty(n, (k + 31) // 32 * 16, dtype=torch.uint8, device=weights.device)
        scales = torch.empty(n, (k + group - 1) // group, 2, dtype=torch.float16, device=weights.device)
        capi.check(capi.lib().xnor_b200_w4_quantize(C.byref(capi.W4Desc(n, k, group, capi.LINEAR)), weights.data_ptr(), dtype,
                                                   weights.stride(0) if n > 1 else k, codes.data_ptr(), scales.data_ptr(),
                                                   torch.cuda.current_stream().cuda_stream), "xnor_b200_w4_quantize")
    return Matrix4(codes, scales, k, group)


def _refuse_product(m: Matrix4, x, biases, activation, out) -> None:
    if x.dim() != 2 or x.shape[1] != m.k or (x.stride(1) != 1 and m.k != 1):
        raise ValueError(f"x must be [rows][{m.k}] with contiguous rows")
    _dtype(x, "x")
    if activation not in m._descs:
        raise ValueError("activation must be capi.LINEAR or capi.LEAKY")
    if biases is not None and (biases.dtype != torch.float32 or biases.shape != (m.n,) or not biases.is_contiguous()):
        raise ValueError(f"biases must be contiguous fp32 [{m.n}]")
    if out is not None and (out.dtype != x.dtype or out.shape != (x.shape[0], m.n) or (out.stride(1) != 1 and m.n != 1)):
        raise ValueError(f"out must be {x.dtype} [{x.shape[0]}][{m.n}] with contiguous rows")
    _on(m.device, x, m.codes, m.scales, biases, out)


def forward_connected4(m: Matrix4, x: torch.Tensor, biases: Optional[torch.Tensor] = None, activation: int = capi.LINEAR,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x @ W.T + biases) for x [rows][k] (rows contiguous, any distance apart), W the packed matrix: xnor_b200_w4_forward.
    biases: fp32 [n].  out: [rows][n] of x's type, rows contiguous; made where it is not given.  One pass over the weights serves up to
    16 rows."""
    index, shape, dtype, desc, n = m._index, x.shape, _DTYPES.get(x.dtype), m._descs.get(activation), m.n
    if (index < 0 or dtype is None or desc is None or out is not None or len(shape) != 2 or shape[1] != m.k or x.get_device() != index
            or not x.is_contiguous()
            or (biases is not None and (biases.dtype is not torch.float32 or biases.shape != (n,) or not biases.is_contiguous() or biases.get_device() != index))):
        _refuse_product(m, x, biases, activation, out)
    if _current_device() != index:
        with torch.cuda.device(index):
            return forward_connected4(m, x, biases, activation, out)
    rows = shape[0]
    if out is None:
        out = x.new_empty((rows, n))
    if rows == 0:
        return out
    nbytes, scratch = 0, None
    if rows > 8:                                              # (fewer never need any)
        nbytes = _calls.w4_scratch_bytes(desc, dtype, rows)
        if nbytes:
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    rc = _calls.w4_forward(desc, x.data_ptr(), dtype, rows, x.stride(0) if rows > 1 else m.k, m.codes.data_ptr(), m.scales.data_ptr(),
                           None if biases is None else biases.data_ptr(), out.data_ptr(), out.stride(0) if rows > 1 else n,
                           None if scratch is None else scratch.data_ptr(), nbytes, _raw_stream(index))
    if rc:
        capi.check(rc, "xnor_b200_w4_forward")
    return out


class Cache4(_Fixed):
    """Pages of four-bit keys and values (struct xnor_b200_kv4_cache): codes uint8 [pages][kv_heads][page][dim/2], scales fp16
    [pages][kv_heads][page][dim/group][2], contiguous."""

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor, group: int) -> None:
        if group not in _GROUPS:
            raise ValueError(f"group must be one of {_GROUPS}, not {group}")
        if k_codes.dim() != 4 or 0 in k_codes.shape:
            raise ValueError("codes must be [pages][kv_heads][page][dim/2]")
        pages, kv_heads, page, half = k_codes.shape
        dim = 2 * half
        if page % 16 or dim % 32 or dim % group or dim > capi.KV4_MAX_DIM:
            raise ValueError(f"page must be a multiple of 16, dim one of 32 and of the group, at most {capi.KV4_MAX_DIM}: got page {page}, dim {dim}, group {group}")
        for codes, scales in ((k_codes, k_scales), (v_codes, v_scales)):
            if codes.dtype != torch.uint8 or codes.shape != k_codes.shape or not codes.is_contiguous():
                raise ValueError(f"codes of keys and values must be contiguous uint8 {list(k_codes.shape)}")
            if scales.dtype != torch.float16 or scales.shape != (pages, kv_heads, page, dim // group, 2) or not scales.is_contiguous():
                raise ValueError(f"scales must be contiguous fp16 {[pages, kv_heads, page, dim // group, 2]}")
            if codes.device != k_codes.device or scales.device != k_codes.device:
                raise ValueError("all four buffers must be on one device")
        # _scratch: bytes of scratch memory by the sizes of a call
        self.__dict__.update(k_codes=k_codes, k_scales=k_scales, v_codes=v_codes, v_scales=v_scales, pages=pages, kv_heads=kv_heads, page=page,
                             dim=dim, group=group, device=k_codes.device, _index=k_codes.get_device(), _scale=dim ** -0.5, _scratch={})

    def _struct(self) -> bytes:
        """Packed for every call, so that it never names memory that a tensor has given up."""
        return _CACHE(self.k_codes.data_ptr(), self.k_scales.data_ptr(), self.v_codes.data_ptr(), self.v_scales.data_ptr(), self.pages,
                      self.kv_heads, self.page, self.dim, self.group)


def new_cache4(pages: int, kv_heads: int, page: int, dim: int, group: int, device="cuda:0") -> Cache4:
    """An empty cache (zeros)."""
    def buffer(*shape, dtype):
        return torch.zeros(pages, kv_heads, page, *shape, dtype=dtype, device=device)
    if group not in _GROUPS:
        raise ValueError(f"group must be one of {_GROUPS}, not {group}")
    return Cache4(buffer(dim // 2, dtype=torch.uint8), buffer(dim // group, 2, dtype=torch.float16), buffer(dim // 2, dtype=torch.uint8),
                  buffer(dim // group, 2, dtype=torch.float16), group)


def _rows(c: Cache4, batch: int, tokens: int, table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor]) -> bytes:
    """struct xnor_b200_kv4_rows of a call, checked."""
    index, shape = c._index, table.shape
    if (index < 0 or len(shape) != 2 or shape[0] != batch or shape[1] == 0 or table.dtype is not torch.int32 or not table.is_contiguous()
            or lengths.dtype is not torch.int32 or lengths.shape != (batch,) or not lengths.is_contiguous() or table.get_device() != index
            or lengths.get_device() != index
            or (counts is not None and (counts.dtype is not torch.int32 or counts.shape != (batch,) or not counts.is_contiguous() or counts.get_device() != index))):
        if len(shape) != 2 or shape[0] != batch or shape[1] == 0 or table.dtype != torch.int32 or not table.is_contiguous():
            raise ValueError(f"table must be contiguous int32 [{batch}][pages of a sequence]")
        for name, t in (("lengths", lengths), ("counts", counts)):
            if t is not None and (t.dtype != torch.int32 or t.shape != (batch,) or not t.is_contiguous()):
                raise ValueError(f"{name} must be contiguous int32 [{batch}]")
        _on(c.device, table, lengths, counts)
    return _ROWS(batch, tokens, shape[1], table.data_ptr(), lengths.data_ptr(), 0 if counts is None else counts.data_ptr())


def _tensor(t: torch.Tensor, dtype: int, index: int, what: str) -> bytes:
    """struct xnor_b200_kv4_tensor of a tensor of four dimensions on device `index`."""
    a, b, c, d = t.stride()
    if d != 1 and t.shape[3] != 1:
        raise ValueError(f"the last dimension of {what} must be contiguous")
    if t.get_device() != index or index < 0:
        raise ValueError(f"{what} on {t.device}: all of a call's tensors are on one CUDA device, the cache's")
    return _TENSOR(t.data_ptr(), dtype, a, b, c)


def append4(c: Cache4, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor] = None) -> None:
    """Packs the newest tokens' keys and values [batch][tokens][kv_heads][dim] into their pages: xnor_b200_kv4_append.  lengths: what each
    sequence holds with them; counts: how many of the rows are tokens (default: all), the first ones of each sequence.  table: int32
    [batch][pages of a sequence].  No two rows may share a place."""
    shape, dtype = k.shape, _DTYPES.get(k.dtype)
    if dtype is None or len(shape) != 4 or shape[2] != c.kv_heads or shape[3] != c.dim or v.shape != shape or v.dtype is not k.dtype:
        _dtype(k, "k")
        raise ValueError(f"k and v must be [batch][tokens][{c.kv_heads}][{c.dim}] of one type")
    index = c._index
    kt, vt, rows = _tensor(k, dtype, index, "k"), _tensor(v, dtype, index, "v"), _rows(c, shape[0], shape[1], table, lengths, counts)
    if k.numel() == 0:
        return
    if _current_device() != index:
        with torch.cuda.device(index):
            return append4(c, k, v, table, lengths, counts)
    rc = _calls.kv4_append(c._struct(), rows, kt, vt, _raw_stream(index))
    if rc:
        capi.check(rc, "xnor_b200_kv4_append")


def read4(c: Cache4, table: torch.Tensor, lengths: torch.Tensor, tokens: int, counts: Optional[torch.Tensor] = None, dtype=torch.float32):
    """What the cache holds for the last `tokens` positions (or counts[b] of them) of every sequence, as keys and values [batch][tokens][kv_heads][dim]:
    xnor_b200_kv4_read.  Rows that stand for no token are 0."""
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be fp32, fp16 or bf16, not {dtype}")
    if table.dim() != 2 or tokens < 0:
        raise ValueError("table must be int32 [batch][pages of a sequence], tokens at least 0")
    index, batch = c._index, table.shape[0]
    rows = _rows(c, batch, tokens, table, lengths, counts)
    if _current_device() != index:
        with torch.cuda.device(index):
            return read4(c, table, lengths, tokens, counts, dtype)
    k = torch.empty((batch, tokens, c.kv_heads, c.dim), dtype=dtype, device=c.device)
    v = torch.empty_like(k)
    if batch and tokens:
        head = c.dim
        strides = (_DTYPES[dtype], tokens * c.kv_heads * head, c.kv_heads * head, head)
        rc = _calls.kv4_read(c._struct(), rows, _TENSOR(k.data_ptr(), *strides), _TENSOR(v.data_ptr(), *strides), _raw_stream(index))
        if rc:
            capi.check(rc, "xnor_b200_kv4_read")
    return k, v


def attend4(c: Cache4, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor] = None,
            scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the newest tokens' queries [batch][tokens][heads][dim] over what their sequences hold, those tokens among it (append4
    comes first): xnor_b200_kv4_attend.  scale: 1/sqrt(dim) where not given.  window: positions that a token sees, itself among them
    (0: all).  Rows that see nothing are 0.  out: as q; made where it is not given.  lse: fp32 [batch][tokens][heads], contiguous, receives
    the logarithm of each row's sum of exponentials."""
    index, shape, dtype = c._index, q.shape, _DTYPES.get(q.dtype)
    if dtype is None or len(shape) != 4 or shape[3] != c.dim or shape[2] == 0 or shape[2] % c.kv_heads or window < 0:
        _dtype(q, "q")
        raise ValueError(f"q must be [batch][tokens][heads][{c.dim}], heads a multiple of {c.kv_heads}; window at least 0")
    if out is not None and (out.shape != shape or out.dtype != q.dtype):
        raise ValueError(f"out must be {q.dtype} {list(shape)}")
    if out is not None and torch._debug_has_internal_overlap(out) == 1:
        raise ValueError("out has rows that share memory")
    if lse is not None and (lse.shape != shape[:3] or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.get_device() != index):
        raise ValueError(f"lse must be contiguous fp32 {list(shape[:3])} on the cache's device")
    batch, tokens, heads = shape[0], shape[1], shape[2]
    rows, qt = _rows(c, batch, tokens, table, lengths, counts), _tensor(q, dtype, index, "q")
    if _current_device() != index:
        with torch.cuda.device(index):
            return attend4(c, q, table, lengths, counts, scale, window, out, lse)
    if out is None:
        out = torch.empty_like(q)
    if batch == 0 or tokens == 0:
        return out
    ot = _tensor(out, dtype, index, "out")
    cache, sizes = c._struct(), (batch, tokens, table.shape[1], heads, window)
    nbytes = c._scratch.get(sizes)
    if nbytes is None:
        if len(c._scratch) >= 1024:
            c._scratch.clear()
        nbytes = c._scratch[sizes] = _calls.kv4_attend_scratch_bytes(cache, rows, heads, window)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=c.device) if nbytes else None
    rc = _calls.kv4_attend(cache, rows, qt, heads, c._scale if scale is None else scale, window, ot, None if lse is None else lse.data_ptr(),
                           None if scratch is None else scratch.data_ptr(), nbytes, _raw_stream(index))
    if rc:
        capi.check(rc, "xnor_b200_kv4_attend")
    return out
