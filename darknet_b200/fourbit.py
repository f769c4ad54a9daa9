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
from typing import Optional

import torch

from . import capi

_DTYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_GROUPS = (32, 64, 128)


class _Calls:
    """bindings/fourbit_calls.cpp, loaded at the first call: a decoding step is a few small kernels, so what a call costs on the host counts.
    Its functions read the tensors, make what is not given and call the library.  They return None where an argument is not what it has to
    be: _refuse_* then look for the fault and name it."""

    def __getattr__(self, name: str):
        capi.lib()
        try:
            from . import _fourbit
        except ImportError as e:
            raise FileNotFoundError(f"_fourbit.so is missing or does not load ({e}): it has not been built (python -m darknet_b200.build). "
                                    "There is no CPU or PyTorch fallback for this path.") from e
        if _fourbit.built_for != torch.__version__:
            raise FileNotFoundError(f"_fourbit.so has been built for torch {_fourbit.built_for}, this is {torch.__version__}: build it again (python -m darknet_b200.build)")
        for f in ("product", "append", "read", "attend"):
            setattr(self, f, getattr(_fourbit, f))
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


def _fits(n: int, k: int) -> None:
    if n > capi.W4_MAX_N or k > capi.W4_MAX_K:
        raise ValueError(f"a matrix has at most {capi.W4_MAX_N} rows of at most {capi.W4_MAX_K} values: got [{n}][{k}]")


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
        _fits(codes.shape[0], k)
        self.__dict__.update(codes=codes, scales=scales, n=codes.shape[0], k=k, group=group, device=codes.device, _native=(codes, scales, k, group))


def quantize_weights4(weights: torch.Tensor, group: int) -> Matrix4:
    """Packs a matrix [n][k] (rows contiguous) to four bits: xnor_b200_w4_quantize."""
    if weights.dim() != 2 or weights.numel() == 0 or (weights.stride(1) != 1 and weights.shape[1] != 1):
        raise ValueError("weights must be a matrix [n][k] with contiguous rows")
    if group not in _GROUPS:
        raise ValueError(f"group must be one of {_GROUPS}, not {group}")
    n, k = weights.shape
    _fits(n, k)
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
    _on(m.device, x, biases, out)
    if x.dim() != 2 or x.shape[1] != m.k or (x.stride(1) != 1 and m.k != 1):
        raise ValueError(f"x must be [rows][{m.k}] with contiguous rows")
    _dtype(x, "x")
    if biases is not None and (biases.dtype != torch.float32 or biases.shape != (m.n,) or not biases.is_contiguous()):
        raise ValueError(f"biases must be contiguous fp32 [{m.n}]")
    if out is not None and (out.dtype != x.dtype or out.shape != (x.shape[0], m.n) or (out.stride(1) != 1 and m.n != 1)):
        raise ValueError(f"out must be {x.dtype} [{x.shape[0]}][{m.n}] with contiguous rows")
    raise ValueError("activation must be capi.LINEAR or capi.LEAKY, x of fewer than 2^31 rows")


def forward_connected4(m: Matrix4, x: torch.Tensor, biases: Optional[torch.Tensor] = None, activation: int = capi.LINEAR,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x @ W.T + biases) for x [rows][k] (rows contiguous, any distance apart), W the packed matrix: xnor_b200_w4_forward.
    biases: fp32 [n].  out: [rows][n] of x's type, rows contiguous, no memory in common with any input; made where it is not given.  One pass over the weights serves up to
    16 rows."""
    y = _calls.product(m._native, x, biases, activation, out)
    if y is None:
        _refuse_product(m, x, biases, activation, out)
    if type(y) is int:
        capi.check(y, "xnor_b200_w4_forward")
    return y


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
        if pages >= 2 ** 31 or kv_heads >= 2 ** 31 or page >= 2 ** 31:
            raise ValueError(f"pages, heads and tokens of a page are below 2^31: got {list(k_codes.shape)}")
        if page % 16 or dim % 32 or dim % group or dim > capi.KV4_MAX_DIM:
            raise ValueError(f"page must be a multiple of 16, dim one of 32 and of the group, at most {capi.KV4_MAX_DIM}: got page {page}, dim {dim}, group {group}")
        for codes, scales in ((k_codes, k_scales), (v_codes, v_scales)):
            if codes.dtype != torch.uint8 or codes.shape != k_codes.shape or not codes.is_contiguous():
                raise ValueError(f"codes of keys and values must be contiguous uint8 {list(k_codes.shape)}")
            if scales.dtype != torch.float16 or scales.shape != (pages, kv_heads, page, dim // group, 2) or not scales.is_contiguous():
                raise ValueError(f"scales must be contiguous fp16 {[pages, kv_heads, page, dim // group, 2]}")
            if codes.device != k_codes.device or scales.device != k_codes.device:
                raise ValueError("all four buffers must be on one device")
        self.__dict__.update(k_codes=k_codes, k_scales=k_scales, v_codes=v_codes, v_scales=v_scales, pages=pages, kv_heads=kv_heads, page=page,
                             dim=dim, group=group, device=k_codes.device, _native=(k_codes, k_scales, v_codes, v_scales, group))


def new_cache4(pages: int, kv_heads: int, page: int, dim: int, group: int, device="cuda:0") -> Cache4:
    """An empty cache (zeros)."""
    def buffer(*shape, dtype):
        return torch.zeros(pages, kv_heads, page, *shape, dtype=dtype, device=device)
    if group not in _GROUPS:
        raise ValueError(f"group must be one of {_GROUPS}, not {group}")
    return Cache4(buffer(dim // 2, dtype=torch.uint8), buffer(dim // group, 2, dtype=torch.float16), buffer(dim // 2, dtype=torch.uint8),
                  buffer(dim // group, 2, dtype=torch.float16), group)


def _refuse_rows(c: Cache4, batch: int, table, lengths, counts) -> None:
    _on(c.device, table, lengths, counts)
    if table.dim() != 2 or table.shape[0] != batch or table.shape[1] == 0 or table.dtype != torch.int32 or not table.is_contiguous():
        raise ValueError(f"table must be contiguous int32 [{batch}][pages of a sequence]")
    for name, t in (("lengths", lengths), ("counts", counts)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (batch,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous int32 [{batch}]")


def append4(c: Cache4, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor] = None) -> None:
    """Packs the newest tokens' keys and values [batch][tokens][kv_heads][dim] into their pages: xnor_b200_kv4_append.  lengths: what each
    sequence holds with them; counts: how many of the rows are tokens (default: all), the first ones of each sequence.  table: int32
    [batch][pages of a sequence].  No two rows may share a place."""
    done = _calls.append(c._native, k, v, table, lengths, counts)
    if done is None:
        _on(c.device, k, v)
        _dtype(k, "k")
        if k.dim() != 4 or k.shape[2:] != (c.kv_heads, c.dim) or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError(f"k and v must be [batch][tokens][{c.kv_heads}][{c.dim}] of one type")
        _refuse_rows(c, k.shape[0], table, lengths, counts)
        raise ValueError("the last dimension of k and v must be contiguous")
    if type(done) is int:
        capi.check(done, "xnor_b200_kv4_append")


def read4(c: Cache4, table: torch.Tensor, lengths: torch.Tensor, tokens: int, counts: Optional[torch.Tensor] = None, dtype=torch.float32):
    """What the cache holds for the last `tokens` positions (or counts[b] of them) of every sequence, as keys and values [batch][tokens][kv_heads][dim]:
    xnor_b200_kv4_read.  Rows that stand for no token are 0."""
    both = _calls.read(c._native, table, lengths, tokens, counts, _DTYPES.get(dtype, -1))
    if both is None:
        if dtype not in _DTYPES:
            raise ValueError(f"dtype must be fp32, fp16 or bf16, not {dtype}")
        _refuse_rows(c, table.shape[0], table, lengths, counts)
        raise ValueError("tokens must be a number, at least 0")
    if type(both) is int:
        capi.check(both, "xnor_b200_kv4_read")
    return both


def attend4(c: Cache4, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor] = None,
            scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the newest tokens' queries [batch][tokens][heads][dim] over what their sequences hold, those tokens among it (append4
    comes first): xnor_b200_kv4_attend.  scale: 1/sqrt(dim) where not given.  window: positions that a token sees, itself among them
    (0: all).  Rows that see nothing are 0.  out: as q, and may be q itself, but have no other memory in common with it; made where it is not
    given.  lse: fp32 [batch][tokens][heads], contiguous, receives
    the logarithm of each row's sum of exponentials.  tokens * heads: up to half a million a call, up to dim 128 three times as many."""
    y = _calls.attend(c._native, q, table, lengths, counts, scale, window, out, lse)
    if y is None:
        _on(c.device, q, out, lse)
        _dtype(q, "q")
        if q.dim() != 4 or q.shape[3] != c.dim or q.shape[2] == 0 or q.shape[2] % c.kv_heads or q.stride(3) != 1:
            raise ValueError(f"q must be [batch][tokens][heads][{c.dim}], heads a multiple of {c.kv_heads}, the last dimension contiguous")
        _refuse_rows(c, q.shape[0], table, lengths, counts)
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(3) != 1):
            raise ValueError(f"out must be {q.dtype} {list(q.shape)}, the last dimension contiguous")
        if lse is not None and (lse.shape != q.shape[:3] or lse.dtype != torch.float32 or not lse.is_contiguous()):
            raise ValueError(f"lse must be contiguous fp32 {list(q.shape[:3])}")
        raise ValueError("window must be a number, at least 0")
    if type(y) is int:
        capi.check(y, "xnor_b200_kv4_attend")
    return y
