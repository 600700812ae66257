"""Operators on data held in 8 and 4 bits, for what a user of ``householder_product`` builds next.

An orthogonal ``Q`` mixes channels without changing norms or inner products, so activations,
weights, keys and values that were rotated by one have no outlying channels and can be held in few
bits. These are the operators that make and consume such data:

* :func:`rms_norm_int8`, :func:`quantize_int8`, :func:`dequantize_int8`: rows into 8 bits and back;
* :func:`int8_linear`: the product of 8-bit activations and weights;
* :func:`kv4_cache`, :func:`kv4_write`, :func:`kv4_read`: a paged key/value cache in 4 bits;
* :func:`kv4_attention`: attention of new tokens over that cache;
* :func:`kv8_cache`, :func:`kv8_write`, :func:`kv8_read`, :func:`kv8_attention`: the same in 8 bits, with a
  range for each page and head;
* :func:`quantize_fp8`, :func:`dequantize_fp8`, :func:`fp8_linear`: 8-bit floating point with a scale for
  each block of 128, for what is not rotated, and the product of such operands.

All run on CUDA tensors only, on the current stream of the operands' device with no host
synchronisation, and never modify an input (``kv4_write`` and ``kv8_write`` write their cache). Wrong arguments raise
``TypeError``/``ValueError``, host tensors ``RuntimeError``, and a failing C-ABI call, or one that
an earlier kernel on the device has reported (an index outside a cache), ``QRB200Error``. Rounding
to integers has no derivative, so a call that autograd would record raises ``RuntimeError``: use
``torch.no_grad()``. None of them has a counterpart in the reference.
"""

from __future__ import annotations

import os

import torch

from . import _lib
from .build import NATIVE_PATH

__all__ = ["rms_norm_int8", "quantize_int8", "dequantize_int8", "int8_linear",
           "KV4Cache", "kv4_cache", "kv4_write", "kv4_read", "kv4_attention",
           "quantize_fp8", "dequantize_fp8", "fp8_linear",
           "KV8Cache", "kv8_cache", "kv8_write", "kv8_read", "kv8_attention"]

_module = None


def _native():
    """The native binding; like the library it binds, it is loaded from this package's directory only, on first use."""
    global _module
    if _module is None:
        _lib.load()
        if not os.path.exists(NATIVE_PATH):
            raise ImportError(f"qrb200 binding not found at {NATIVE_PATH}; build it with "
                              "`python -m qr_v2_b200_kernel_b200.build` (no CPU fallback exists)")
        from . import _native as module

        _module = module
    return _module


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                  eps: float = 1e-6):
    """Root-mean-square norm of ``x + residual`` into 8 bits: ``(codes, scale, h)``.

    ``h = x + residual`` (``x`` itself without a residual), in ``x``'s type; ``codes`` int8 of
    ``x``'s shape and ``scale`` float32 of its leading shape, with ``codes * scale[..., None]`` the
    values of ``weight * h / sqrt(mean(h^2) + eps)`` to within half a step of the row's largest /
    127. The sums run in 32 bits on ``h`` before its rounding.

    ``x`` (..., cols), cols <= 32768, and ``residual``: bfloat16, float16 or float32, any strides;
    ``weight`` (cols,) of ``x``'s type or float32. A row with a NaN or an infinity gets a NaN scale.
    Rows of ``codes`` are 16-byte aligned, so ``codes`` is contiguous only where cols is a multiple
    of 16.
    """
    return (_module or _native()).rms_norm_int8(x, weight, residual, eps)


def quantize_int8(x: torch.Tensor):
    """``(codes, scale)``: each row of ``x`` (..., cols) in 8 bits, ``codes * scale[..., None]`` within
    half a step of its largest / 127. For weights (a scale for each output channel) and for
    activations that no norm precedes. Types, strides and odd rows as :func:`rms_norm_int8`."""
    return (_module or _native()).quantize_int8(x)


def dequantize_int8(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``codes * scale[..., None]`` rounded once to ``dtype``: the values that 8-bit rows stand for."""
    return (_module or _native()).dequantize_int8(codes, scale, dtype)


def int8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(x x_scale[..., None]) (weight weight_scale[:, None])^T + bias`` of 8-bit operands, in ``dtype``.

    ``x`` int8 (..., depth) with a float32 scale for each row (token), ``weight`` int8 (outs, depth)
    with a float32 scale for each output channel, as :func:`rms_norm_int8` and :func:`quantize_int8`
    make them; ``bias`` (outs,) of ``dtype``. 1 <= depth <= 131071. The products are summed exactly,
    in 32-bit integers; the sum is converted, scaled and given the bias in 32-bit floating point, and the result
    rounded once to ``dtype``. Beyond two rows, operands whose rows do not
    start on 16-byte boundaries are laid out anew first; those that the quantising functions return
    do.
    """
    return (_module or _native()).int8_linear(x, x_scale, weight, weight_scale, bias, dtype)


class KV4Cache:
    """A paged key/value cache in 4 bits (see :func:`kv4_cache`).

    ``data``: uint8 (pages, kv_heads, bytes of a block), the whole state, written in place;
    ``KV4Cache(data.clone(), ...)`` is a copy of the cache. Its attributes cannot be assigned: another
    tensor's bytes are another cache, or are copied into ``data``. A token occupies head_dim + 8
    head_dim / group_size bytes a head for its key and value.
    """

    __slots__ = ("data", "pages", "page_size", "kv_heads", "head_dim", "group_size", "dtype", "_handle")

    def __init__(self, data: torch.Tensor, page_size: int, head_dim: int, group_size: int, dtype: torch.dtype):
        if group_size < 1 or head_dim % group_size:
            raise ValueError(f"group_size must divide head_dim, got {group_size} and {head_dim}")
        handle = _native().Cache(data, page_size, head_dim, head_dim // group_size, dtype)
        for name, value in (("data", data), ("pages", int(data.shape[0])), ("page_size", page_size), ("kv_heads", int(data.shape[1])),
                            ("head_dim", head_dim), ("group_size", group_size), ("dtype", dtype), ("_handle", handle)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):  # the handle would go on with what it was made of
        raise AttributeError(f"a KV4Cache's {name} cannot be assigned")

    def __reduce__(self):  # copy.copy shares the bytes, copy.deepcopy and pickle copy them
        return KV4Cache, (self.data, self.page_size, self.head_dim, self.group_size, self.dtype)


def kv4_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, group_size: int | None = None,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> KV4Cache:
    """An empty 4-bit cache of ``pages`` pages of ``page_size`` tokens (a power of two from 16 to 1024).

    ``head_dim`` 64 or 128; ``group_size`` channels share a step and a minimum: 32, 64 or 128, at
    most and by default head_dim. ``dtype``: bfloat16 or float16, of the keys and values written and
    the queries that read. Fresh slots hold zeros.
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


def _handle(cache, kind=KV4Cache):
    if not isinstance(cache, kind):
        raise TypeError(f"cache must be a {kind.__name__}")
    return cache._handle


def kv4_write(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises ``k`` and ``v`` (tokens, kv_heads, head_dim) of the cache's type into its ``slots``.

    ``slots`` int64 (tokens,): page * page_size + offset, each at most once; negative ones are
    skipped (padding). Any strides (copied where channels are not contiguous). Each group's least
    entry is kept in the cache's type, its range in fifteen steps; a group with a NaN or an infinity
    reads back as NaN. A slot past the cache is skipped and reported by the next call as
    ``QRB200Error``.
    """
    (_module or _native()).kv4_write(_handle(cache), k, v, slots)


def kv4_read(cache: KV4Cache, slots: torch.Tensor):
    """``(k, v)``, each (tokens, kv_heads, head_dim): the values that the cache holds at ``slots``
    (int64), rounded once to its type; zeros for a negative slot. A slot past the cache reads as
    zeros and is reported by the next call."""
    return (_module or _native()).kv4_read(_handle(cache), slots)


def kv4_attention(q: torch.Tensor, cache: KV4Cache, block_table: torch.Tensor, lengths: torch.Tensor,
                  scale: float | None = None, causal: bool = True, window: int | None = None) -> torch.Tensor:
    """Softmax attention of each sequence's newest tokens over its 4-bit cache.

    ``q`` (batch, queries, heads, head_dim) of the cache's type, heads a multiple of kv_heads (head
    h reads key head h // (heads // kv_heads)). ``block_table`` int32 (batch, max_pages): the pages
    of each sequence in order; entries past its length, or behind every query's window, are not
    read. ``lengths`` int32 (batch,): tokens in the cache, the queries' own included, so query i
    stands at position lengths - queries + i. It sees every token up to its position (to the end with
    ``causal=False``), with ``window`` only those from position - window + 1 on. ``scale`` multiplies
    the scores (default head_dim ** -0.5). Rows that see nothing (an empty sequence, a position before
    its start) are zero. Returns (batch, queries, heads, head_dim), rounded once. Scores, softmax and sums
    are in 32 bits at any length, the weights of the values in 22; the matrix instruction's cut-offs make
    the error some units of 2^-24 of the values' size, a few times that of 32-bit operations
    throughout. A length or page outside the table or the cache is left out and reported by the next
    call as ``QRB200Error``; heads <= 65535, queries * heads / kv_heads <= 2^24.
    """
    return (_module or _native()).kv4_attention(q, _handle(cache), block_table, lengths, scale, causal, window)


def quantize_fp8(x: torch.Tensor, tile_rows: int = 1):
    """``(codes, scale)``: ``x`` in 8-bit floating point (``torch.float8_e4m3fn``), a scale for each block of 128.

    With ``tile_rows=1`` a block is 128 entries of a row: ``scale`` float32 (..., ceil(cols / 128)), for
    activations. With ``tile_rows=128`` it is 128 rows and 128 columns of ``x`` (rows, cols): ``scale``
    (ceil(rows / 128), ceil(cols / 128)), for weights. Blocks at the ends may be smaller. A block's largest
    magnitude a becomes 448, the largest code: ``scale = a / 448``, and a code is the number nearest to ``448 x / a``, ties to
    even. ``x``: bfloat16, float16 or float32, any strides, cols <= 1048576. A block with a NaN or an infinity gets a NaN
    scale. Rows of ``codes`` are 16-byte aligned, so ``codes`` is contiguous only where cols is a
    multiple of 16.
    """
    return (_module or _native()).quantize_fp8(x, tile_rows)


def dequantize_fp8(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                   tile_rows: int = 1) -> torch.Tensor:
    """``codes`` times the scale of their block (``tile_rows`` as in :func:`quantize_fp8`), rounded once to ``dtype``."""
    return (_module or _native()).dequantize_fp8(codes, scale, dtype, tile_rows)


def fp8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The product of operands in 8-bit floating point, ``x weight^T + bias`` of the values they stand for, in ``dtype``.

    ``x`` (..., depth) with ``x_scale`` (..., ceil(depth / 128)) and ``weight`` (outs, depth) with
    ``weight_scale`` (ceil(outs / 128), ceil(depth / 128)), as :func:`quantize_fp8` makes them with ``tile_rows`` 1 and
    128; ``bias`` (outs,) of ``dtype``. 1 <= depth <= 1048576. A block's products are summed, then multiplied by the
    product of its two scales and added, all in 32-bit floating point; the result is rounded once to ``dtype``. Operands whose
    rows do not start on 16-byte boundaries may be laid out anew first; those that :func:`quantize_fp8` returns
    do.
    """
    return (_module or _native()).fp8_linear(x, x_scale, weight, weight_scale, bias, dtype)


class KV8Cache:
    """A paged key/value cache in 8 bits (see :func:`kv8_cache`).

    ``data``: uint8 (pages, kv_heads, bytes of a block), the codes; ``range``: float32 (pages, kv_heads, 2), what a page's
    keys and values reach. Both are the state, written in place; ``KV8Cache(data.clone(),
    range.clone(), ...)`` is a copy of the cache. Its attributes cannot be assigned. A token
    occupies 2 head_dim bytes a head for its key and value.
    """

    __slots__ = ("data", "range", "pages", "page_size", "kv_heads", "head_dim", "dtype", "_handle")

    def __init__(self, data: torch.Tensor, range: torch.Tensor, page_size: int, head_dim: int, dtype: torch.dtype):
        handle = _native().Cache8(data, range, page_size, head_dim, dtype)
        for name, value in (("data", data), ("range", range), ("pages", int(data.shape[0])), ("page_size", page_size),
                            ("kv_heads", int(data.shape[1])), ("head_dim", head_dim), ("dtype", dtype), ("_handle", handle)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):  # the handle would go on with what it was made of
        raise AttributeError(f"a KV8Cache's {name} cannot be assigned")

    def __reduce__(self):  # copy.copy shares the bytes, copy.deepcopy and pickle copy them
        return KV8Cache, (self.data, self.range, self.page_size, self.head_dim, self.dtype)


def kv8_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> KV8Cache:
    """An empty 8-bit cache of ``pages`` pages of ``page_size`` tokens (a power of two from 16 to 1024).

    ``head_dim`` 64 or 128. Each page and head has a range for its keys and one for its values, in 127
    steps either way. ``dtype``: bfloat16 or float16, of the keys and values written and the queries that read.
    """
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"dtype must be torch.bfloat16 or torch.float16, got {dtype}")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
    if not 0 <= pages < 2**31 or not 1 <= kv_heads <= 65535:
        raise ValueError(f"need 0 <= pages < 2^31 and 1 <= kv_heads <= 65535, got {pages} and {kv_heads}")
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("qrb200 runs on CUDA devices only (no CPU fallback)")
    size = int(_lib.load().qrb200_kv8_block_bytes(page_size, head_dim))
    return KV8Cache(torch.full((pages, kv_heads, size), 128, dtype=torch.uint8, device=device),
                    torch.zeros((pages, kv_heads, 2), dtype=torch.float32, device=device), page_size, head_dim, dtype)


def kv8_write(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises ``k`` and ``v`` (tokens, kv_heads, head_dim) of the cache's type into its ``slots``.

    ``slots`` int64 (tokens,): page * page_size + offset, in any order, each at most once; negative ones are
    skipped (padding). Any strides (copied where channels are not contiguous). A page's range for a head
    grows to the largest magnitude written, rounded up to three significant bits; a code is the nearest of
    127 steps either way, and where the range grew the page's older codes are rounded to the new
    steps. A call that writes a page's first token begins the page anew: the rest of it reads as zeros. A
    NaN or an infinity makes what the page holds of its head NaN, until the page begins anew. Calls that
    run at the same time may not write the same page. More than 1024 tokens take a workspace of 4 bytes a slot of the
    cache. A slot past the cache is skipped and reported by the next call as ``QRB200Error``.
    """
    (_module or _native()).kv8_write(_handle(cache, KV8Cache), k, v, slots)


def kv8_read(cache: KV8Cache, slots: torch.Tensor):
    """``(k, v)``, each (tokens, kv_heads, head_dim): the values that the cache holds at ``slots``
    (int64), rounded once to its type; zeros for a negative slot. A slot past the cache reads as
    zeros and is reported by the next call."""
    return (_module or _native()).kv8_read(_handle(cache, KV8Cache), slots)


def kv8_attention(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, lengths: torch.Tensor,
                  scale: float | None = None, causal: bool = True, window: int | None = None) -> torch.Tensor:
    """Softmax attention of each sequence's newest tokens over its 8-bit cache.

    Operands, masks, limits and failures as in :func:`kv4_attention`; single tokens, drafts and long prompts alike. Weights
    are held in 22 bits; in prompts over more than some 2000 tokens (float16 1000) the matrix instruction's cut-offs make
    the error some 2^-16 (2^-17) of the values' size. What a row does not see does not enter its result.
    """
    return (_module or _native()).kv8_attention(q, _handle(cache, KV8Cache), block_table, lengths, scale, causal, window)
