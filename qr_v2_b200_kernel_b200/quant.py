"""Operators on data held in 8 and 4 bits, for what a user of ``householder_product`` builds next.

An orthogonal ``Q`` mixes channels without changing norms or inner products, so activations,
weights, keys and values that were rotated by one have no outlying channels and can be held in few
bits. These are the operators that make and consume such data:

* :func:`rms_norm_int8`, :func:`quantize_int8`, :func:`dequantize_int8`: rows into 8 bits and back;
* :func:`int8_linear`: the product of 8-bit activations and weights;
* :func:`kv4_cache`, :func:`kv4_write`, :func:`kv4_read`: a paged key/value cache in 4 bits;
* :func:`kv4_attention`: attention of new tokens over that cache.

All run on CUDA tensors only, on the current stream of the operands' device with no host
synchronisation, and never modify an input (``kv4_write`` writes its cache). Wrong arguments raise
``TypeError``/``ValueError``, host tensors ``RuntimeError``, and a failing C-ABI call, or one that an
earlier kernel on the device has reported (an index outside a cache), ``QRB200Error``. Rounding to integers
has no derivative, so a call that autograd would record raises ``RuntimeError``: use
``torch.no_grad()``. None of them has a counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

__all__ = ["rms_norm_int8", "quantize_int8", "dequantize_int8", "int8_linear",
           "KV4Cache", "kv4_cache", "kv4_write", "kv4_read", "kv4_attention"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # QRB200_F32, _BF16, _F16
_MAX_COLS = 32768
_MAX_DEPTH = 131071


def _operand(t, name: str, dtypes, like: torch.Tensor | None = None) -> None:
    """Type, device and autograd checks that every tensor operand gets."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (qrb200 has no CPU path)")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires grad, and quantised operators have no backward pass; use torch.no_grad()")


def _call(what: str, like: torch.Tensor, fn, *args) -> None:
    """``fn(*args, stream)`` on the current stream of ``like``'s device."""
    device = like.get_device()
    if torch.cuda.current_device() == device:
        status = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if status:
        raise _lib.QRB200Error(status, what)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as (rows, cols) with unit column stride, copied only where its strides need it."""
    r = t if t.dim() == 2 else t.reshape(t.shape[:-1].numel(), t.shape[-1])
    if (r.stride(1) != 1 and r.shape[1] > 1) or (r.stride(0) < r.shape[1] and r.shape[0] > 1):
        r = r.contiguous()
    return r


def _loadable(t: torch.Tensor) -> torch.Tensor:
    """8-bit rows as the tensor-core product loads them: from 16-byte boundaries, copied only where they are not."""
    if t.data_ptr() % 16 == 0 and (t.stride(0) % 16 == 0 or t.shape[0] == 1):
        return t
    return _codes(t.shape[0], t.shape[1], t).copy_(t)


def _codes(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    """An int8 (rows, cols) tensor whose rows start on 16-byte boundaries, as the tensor-core product loads them."""
    padded = -(-cols // 16) * 16
    q = torch.empty((rows, padded), dtype=torch.int8, device=like.device)
    return q if padded == cols else q[:, :cols]


def _shaped(q: torch.Tensor, shape) -> torch.Tensor:
    if q.shape == shape:
        return q
    return q[0] if len(shape) == 1 else q.unflatten(0, shape[:-1])


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                  eps: float = 1e-6):
    """Root-mean-square norm of ``x + residual`` into 8 bits: ``(codes, scale, h)``.

    ``h = x + residual`` (``x`` itself without a residual), in ``x``'s type; ``codes`` int8 of ``x``'s
    shape and ``scale`` float32 of its leading shape, with ``codes * scale[..., None]`` the values of
    ``weight * h / sqrt(mean(h^2) + eps)`` to within half a step of the row's largest / 127. The sums run in 32 bits
    on ``h`` before its rounding.

    ``x`` (..., cols), cols <= 32768, and ``residual``: bfloat16, float16 or float32, any strides;
    ``weight`` (cols,) of ``x``'s type or float32. A row with a NaN or an infinity gets a NaN scale. Rows of ``codes`` are
    16-byte aligned, so ``codes`` is contiguous only where cols is a multiple of 16.
    """
    _operand(x, "x", tuple(_TYPES))
    if x.dim() == 0 or x.shape[-1] > _MAX_COLS:
        raise ValueError(f"x must be (..., cols) with cols <= {_MAX_COLS}, got {tuple(x.shape)}")
    cols = x.shape[-1]
    if residual is not None:
        _operand(residual, "residual", (x.dtype,), x)
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {tuple(x.shape)}, got {tuple(residual.shape)}")
    if weight is not None:
        _operand(weight, "weight", (x.dtype, torch.float32), x)
        if weight.dim() != 1 or weight.shape[0] != cols:
            raise ValueError(f"weight must be ({cols},), got {tuple(weight.shape)}")
        weight = weight.contiguous()
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    xr = _rows(x)
    rows = xr.shape[0]
    rr = _rows(residual) if residual is not None else None
    q = _codes(rows, cols, x)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else x
    if rows == 0 or cols == 0:
        return _shaped(q, x.shape), scale.zero_(), h
    _call("rms_norm_int8", x, _lib.load().qrb200_rms_norm_int8, xr.data_ptr(), xr.stride(0),
          rr.data_ptr() if rr is not None else None, rr.stride(0) if rr is not None else 0,
          weight.data_ptr() if weight is not None else None, _TYPES[weight.dtype] if weight is not None else 0,
          q.data_ptr(), q.stride(0), scale.data_ptr(), h.data_ptr() if rr is not None else None, rows, cols, eps,
          _TYPES[x.dtype])
    return _shaped(q, x.shape), scale, h


def quantize_int8(x: torch.Tensor):
    """``(codes, scale)``: each row of ``x`` (..., cols) in 8 bits, ``codes * scale[..., None]`` within half a step
    of its largest / 127. For weights (a scale for each output channel) and for activations that no norm precedes.
    Types, strides and odd rows as :func:`rms_norm_int8`."""
    _operand(x, "x", tuple(_TYPES))
    if x.dim() == 0 or x.shape[-1] > _MAX_COLS:
        raise ValueError(f"x must be (..., cols) with cols <= {_MAX_COLS}, got {tuple(x.shape)}")
    xr = _rows(x)
    rows, cols = xr.shape
    q = _codes(rows, cols, x)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if rows == 0 or cols == 0:
        return _shaped(q, x.shape), scale.zero_()
    _call("quantize_int8", x, _lib.load().qrb200_quantize_int8, xr.data_ptr(), xr.stride(0), q.data_ptr(),
          q.stride(0), scale.data_ptr(), rows, cols, _TYPES[x.dtype])
    return _shaped(q, x.shape), scale


def dequantize_int8(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``codes * scale[..., None]`` rounded once to ``dtype``: the values that 8-bit rows stand for."""
    _operand(codes, "codes", (torch.int8,))
    _operand(scale, "scale", (torch.float32,), codes)
    if dtype not in _TYPES:
        raise TypeError(f"dtype must be one of {list(_TYPES)}, got {dtype}")
    if codes.dim() == 0 or codes.shape[-1] > _MAX_COLS:
        raise ValueError(f"codes must be (..., cols) with cols <= {_MAX_COLS}, got {tuple(codes.shape)}")
    if scale.shape != codes.shape[:-1]:
        raise ValueError(f"scale must be {tuple(codes.shape[:-1])}, got {tuple(scale.shape)}")
    q = _rows(codes)
    rows, cols = q.shape
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    if rows == 0 or cols == 0:
        return out
    scale = scale.contiguous()
    _call("dequantize_int8", codes, _lib.load().qrb200_dequantize_int8, q.data_ptr(), q.stride(0), scale.data_ptr(),
          out.data_ptr(), rows, cols, _TYPES[dtype])
    return out


def int8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(x x_scale[..., None]) (weight weight_scale[:, None])^T + bias`` of 8-bit operands, in ``dtype``.

    ``x`` int8 (..., depth) with a float32 scale for each row (token), ``weight`` int8 (outs, depth) with a
    float32 scale for each output channel, as :func:`rms_norm_int8` and :func:`quantize_int8` make them;
    ``bias`` (outs,) of ``dtype``. 1 <= depth <= 131071. The products are summed exactly, in 32-bit integers, and the
    result is rounded once. Operands whose rows do not start on 16-byte boundaries are copied first.
    """
    _operand(x, "x", (torch.int8,))
    _operand(weight, "weight", (torch.int8,), x)
    _operand(x_scale, "x_scale", (torch.float32,), x)
    _operand(weight_scale, "weight_scale", (torch.float32,), x)
    if dtype not in _TYPES:
        raise TypeError(f"dtype must be one of {list(_TYPES)}, got {dtype}")
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be (..., depth) and weight (outs, depth), got {tuple(x.shape)} and {tuple(weight.shape)}")
    outs, depth = weight.shape
    if not 1 <= depth <= _MAX_DEPTH:
        raise ValueError(f"depth must be from 1 to {_MAX_DEPTH}, got {depth}")
    if x_scale.shape != x.shape[:-1]:
        raise ValueError(f"x_scale must be {tuple(x.shape[:-1])}, got {tuple(x_scale.shape)}")
    if weight_scale.dim() != 1 or weight_scale.shape[0] != outs:
        raise ValueError(f"weight_scale must be ({outs},), got {tuple(weight_scale.shape)}")
    if bias is not None:
        _operand(bias, "bias", (dtype,), x)
        if bias.dim() != 1 or bias.shape[0] != outs:
            raise ValueError(f"bias must be ({outs},), got {tuple(bias.shape)}")
        bias = bias.contiguous()
    xr, wr = _rows(x), _rows(weight)
    rows = xr.shape[0]
    y = torch.empty((*x.shape[:-1], outs), dtype=dtype, device=x.device)
    if rows == 0 or outs == 0:
        return y
    xr, wr = _loadable(xr), _loadable(wr)
    x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()
    _call("int8_linear", x, _lib.load().qrb200_int8_linear, xr.data_ptr(), xr.stride(0), x_scale.data_ptr(),
          wr.data_ptr(), wr.stride(0), weight_scale.data_ptr(), bias.data_ptr() if bias is not None else None,
          y.data_ptr(), rows, outs, depth, _TYPES[dtype])
    return y


class KV4Cache:
    """A paged key/value cache in 4 bits (see :func:`kv4_cache`).

    ``data``: uint8 (pages, kv_heads, bytes of a block), the whole state; a copy of it, made by any means, is a
    copy of the cache. A token occupies head_dim + 8 head_dim / group_size bytes a head for its key and value.
    """

    __slots__ = ("data", "pages", "page_size", "kv_heads", "head_dim", "group_size", "dtype", "_shape")

    def __init__(self, data: torch.Tensor, page_size: int, head_dim: int, group_size: int, dtype: torch.dtype):
        self.data, self.page_size, self.head_dim, self.group_size, self.dtype = data, page_size, head_dim, group_size, dtype
        self.pages, self.kv_heads = int(data.shape[0]), int(data.shape[1])
        self._shape = _lib.KV4Shape(self.pages, self.kv_heads, page_size, head_dim, head_dim // group_size, _TYPES[dtype])

    @property
    def shape_ref(self):
        return ctypes.byref(self._shape)


def kv4_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, group_size: int | None = None,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> KV4Cache:
    """An empty 4-bit cache of ``pages`` pages of ``page_size`` tokens (a power of two from 16 to 1024).

    ``head_dim`` 64 or 128; ``group_size`` channels share a step and a minimum: 32, 64 or 128, at most and by default
    head_dim. ``dtype``: bfloat16 or float16, of the keys and values written and the queries that read. Fresh slots
    hold zeros.
    """
    group_size = head_dim if group_size is None else group_size
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"dtype must be torch.bfloat16 or torch.float16, got {dtype}")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    if group_size not in (32, 64, 128) or group_size > head_dim:
        raise ValueError(f"group_size must be 32, 64 or 128, and at most head_dim, got {group_size}")
    if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
    if not 0 <= pages < 2**31 or not 1 <= kv_heads <= 65535:
        raise ValueError(f"need 0 <= pages < 2^31 and 1 <= kv_heads <= 65535, got {pages} and {kv_heads}")
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("qrb200 runs on CUDA devices only (no CPU fallback)")
    size = int(_lib.load().qrb200_kv4_block_bytes(page_size, head_dim, group_size))
    return KV4Cache(torch.zeros((pages, kv_heads, size), dtype=torch.uint8, device=device), page_size, head_dim,
                    group_size, dtype)


def _cache_operand(cache) -> None:
    if not isinstance(cache, KV4Cache):
        raise TypeError("cache must be a KV4Cache")


def _slots_operand(slots, cache: KV4Cache) -> torch.Tensor:
    _operand(slots, "slots", (torch.int64,), cache.data)
    if slots.dim() != 1:
        raise ValueError(f"slots must be (tokens,), got {tuple(slots.shape)}")
    return slots.contiguous()


def kv4_write(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises ``k`` and ``v`` (tokens, kv_heads, head_dim) of the cache's type into its ``slots``.

    ``slots`` int64 (tokens,): page * page_size + offset, each at most once; negative ones are skipped (padding). Channels
    must be contiguous, the other strides are free. Each group's least entry is kept in the cache's type, its range in fifteen
    steps; a group with a NaN or an infinity reads back as NaN. A slot past the cache is skipped and reported by the
    next call as ``QRB200Error``.
    """
    _cache_operand(cache)
    _operand(k, "k", (cache.dtype,), cache.data)
    _operand(v, "v", (cache.dtype,), cache.data)
    slots = _slots_operand(slots, cache)
    want = (slots.shape[0], cache.kv_heads, cache.head_dim)
    if k.shape != want or v.shape != want:
        raise ValueError(f"k and v must be {want}, got {tuple(k.shape)} and {tuple(v.shape)}")
    if want[0] == 0:
        return
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    _call("kv4_write", cache.data, _lib.load().qrb200_kv4_write, cache.data.data_ptr(), cache.shape_ref, k.data_ptr(),
          k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(), want[0])


def kv4_read(cache: KV4Cache, slots: torch.Tensor):
    """``(k, v)``, each (tokens, kv_heads, head_dim): the values that the cache holds at ``slots`` (int64), rounded
    once to its type; zeros for a negative slot. A slot past the cache reads as zeros and is reported by the next call."""
    _cache_operand(cache)
    slots = _slots_operand(slots, cache)
    n = slots.shape[0]
    k = torch.empty((n, cache.kv_heads, cache.head_dim), dtype=cache.dtype, device=cache.data.device)
    v = torch.empty_like(k)
    if n:
        _call("kv4_read", cache.data, _lib.load().qrb200_kv4_read, cache.data.data_ptr(), cache.shape_ref,
              k.data_ptr(), v.data_ptr(), slots.data_ptr(), n)
    return k, v


def kv4_attention(q: torch.Tensor, cache: KV4Cache, block_table: torch.Tensor, lengths: torch.Tensor,
                  scale: float | None = None, causal: bool = True, window: int | None = None) -> torch.Tensor:
    """Softmax attention of each sequence's newest tokens over its 4-bit cache.

    ``q`` (batch, queries, heads, head_dim) of the cache's type, heads a multiple of kv_heads (head h reads key head
    h // (heads // kv_heads)). ``block_table`` int32 (batch, max_pages): the pages of each sequence in order; entries past its length are
    not read. ``lengths`` int32 (batch,): tokens in the cache, the queries' own included, so
    query i stands at position lengths - queries + i. It sees every token up to its position (all tokens with
    ``causal=False``), or the last ``window`` of those up to its position. ``scale`` multiplies the scores (default head_dim ** -0.5). Rows that see
    nothing (an empty sequence, a position before its start) are zero. Returns (batch, queries, heads, head_dim);
    the scores, the softmax and the sums are in 32 bits, the result is rounded once. A length or page outside
    the table or the cache is left out and reported by the next call as ``QRB200Error``.
    """
    _cache_operand(cache)
    _operand(q, "q", (cache.dtype,), cache.data)
    _operand(block_table, "block_table", (torch.int32,), cache.data)
    _operand(lengths, "lengths", (torch.int32,), cache.data)
    if q.dim() != 4 or q.shape[3] != cache.head_dim or q.shape[2] % cache.kv_heads:
        raise ValueError(f"q must be (batch, queries, heads, {cache.head_dim}) with heads a multiple of {cache.kv_heads}, "
                         f"got {tuple(q.shape)}")
    batch, queries, heads, _ = q.shape
    if block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError(f"block_table must be ({batch}, max_pages), got {tuple(block_table.shape)}")
    if lengths.dim() != 1 or lengths.shape[0] != batch:
        raise ValueError(f"lengths must be ({batch},), got {tuple(lengths.shape)}")
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if scale is not None and not 0 <= scale < 3e38:
        raise ValueError(f"scale must be finite and not negative, got {scale}")
    if q.stride(3) != 1:
        q = q.contiguous()
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        block_table = block_table.contiguous()
    lengths = lengths.contiguous()
    out = torch.empty((batch, queries, heads, cache.head_dim), dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    lib = _lib.load()
    pages = block_table.shape[1]
    need = lib.qrb200_kv4_attention_workspace_bytes(cache.shape_ref, batch, queries, heads, pages)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    strides = (ctypes.c_int64 * 3)(q.stride(0), q.stride(1), q.stride(2))
    _call("kv4_attention", q, lib.qrb200_kv4_attention, q.data_ptr(), strides, cache.data.data_ptr(), cache.shape_ref,
          block_table.data_ptr(), block_table.stride(0), lengths.data_ptr(), out.data_ptr(), batch, queries, heads, pages,
          window or 0, int(causal), 1 / math.sqrt(cache.head_dim) if scale is None else scale,
          ws.data_ptr() if need else None, need)
    return out
