"""Host-side checks of 8-bit floating point and the 8-bit cache: refusals before any device work (CPU)."""

import ctypes

import pytest
import torch

import qr_v2_b200_kernel_b200 as qr
from qr_v2_b200_kernel_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


P = ctypes.c_void_p(256)
ARG, OK = _lib.QRB200_ERR_ARG, _lib.QRB200_OK


def test_fp8_rows_entries_check_their_arguments(lib):
    def quantise(x=P, xs=8, q=P, qs=16, scale=P, rows=2, cols=8, tile=1, dtype=1):
        return lib.qrb200_quantize_fp8(x, xs, q, qs, scale, rows, cols, tile, dtype, None)

    def values(q=P, qs=16, scale=P, out=P, rows=2, cols=8, tile=1, dtype=1):
        return lib.qrb200_dequantize_fp8(q, qs, scale, out, rows, cols, tile, dtype, None)

    for f in (quantise, values):
        assert f(rows=0) == OK and f(cols=0) == OK
        assert f(rows=-1) == ARG and f(cols=(1 << 20) + 1) == ARG and f(tile=2) == ARG and f(tile=0) == ARG and f(dtype=3) == ARG
        assert f(q=None) == ARG and f(scale=None) == ARG and f(qs=7) == ARG
    assert quantise(x=None) == ARG and quantise(xs=7) == ARG and values(out=None) == ARG


def test_fp8_linear_entry_checks_its_arguments(lib):
    def linear(x=P, xs=16, sx=P, w=P, ws=16, sw=P, b=None, y=P, rows=2, outs=3, depth=16, dtype=1):
        return lib.qrb200_fp8_linear(x, xs, sx, w, ws, sw, b, y, rows, outs, depth, dtype, None, 0, None)

    assert linear(rows=0) == OK and linear(outs=0) == OK
    assert linear(depth=0) == ARG and linear(depth=(1 << 20) + 1) == ARG and linear(dtype=7) == ARG
    assert linear(x=None) == ARG and linear(sw=None) == ARG and linear(y=None) == ARG and linear(y=ctypes.c_void_p(264)) == ARG
    assert linear(xs=15) == ARG and linear(ws=15) == ARG and linear(rows=-1) == ARG


def test_kv8_entries_check_their_arguments(lib):
    assert lib.qrb200_kv8_block_bytes(64, 128) == 2 * 64 * 128 and lib.qrb200_kv8_block_bytes(16, 64) == 2048
    for bad in ((24, 128), (8, 128), (2048, 128), (64, 96), (0, 64), (64, -64)):
        assert lib.qrb200_kv8_block_bytes(*bad) == 0
    good = _lib.KV8Shape(4, 2, 16, 64, 1)
    w, r = lib.qrb200_kv8_write, lib.qrb200_kv8_read

    def write(shape=good, codes=P, rng=P, k=P, slots=P, tokens=3):
        return w(codes, rng, ctypes.byref(shape), k, 128, 64, P, 128, 64, slots, tokens, None, 0, None)

    assert write(tokens=0) == OK and write(tokens=-1) == ARG
    assert write(codes=None) == ARG and write(rng=None) == ARG and write(k=None) == ARG and write(slots=None) == ARG
    assert write(codes=ctypes.c_void_p(264)) == ARG  # not 16-byte aligned
    odd = ctypes.c_void_p(260)  # not 8-byte aligned, as pairs of ranges are read
    assert write(rng=odd) == ARG and r(P, odd, ctypes.byref(good), P, P, P, 3, None) == ARG
    for shape in (_lib.KV8Shape(4, 2, 16, 64, 0), _lib.KV8Shape(4, 0, 16, 64, 1), _lib.KV8Shape(4, 2, 24, 64, 1),
                  _lib.KV8Shape(4, 2, 16, 96, 1), _lib.KV8Shape(-1, 2, 16, 64, 1)):
        assert write(shape=shape) == ARG
        assert r(P, P, ctypes.byref(shape), P, P, P, 3, None) == ARG
    assert r(P, P, ctypes.byref(good), P, None, P, 3, None) == ARG and r(P, P, ctypes.byref(good), P, P, P, 0, None) == OK
    assert w(P, P, None, P, 0, 0, P, 0, 0, P, 3, None, 0, None) == ARG
    need = lib.qrb200_kv8_write_workspace_bytes
    assert need(ctypes.byref(good), 1) == 0 and need(ctypes.byref(good), 1 << 20) >= 4 * 16 * 4
    strides = (ctypes.c_int64 * 3)(256, 256, 64)

    def attend(q=P, batch=2, queries=1, heads=4, pages=2, window=0, table=P, lengths=P, st=strides, codes=P, rng=P, scale=0.125):
        return lib.qrb200_kv8_attention(q, st, codes, rng, ctypes.byref(good), table, 2, lengths, P, batch, queries, heads, pages, window,
                                        1, scale, None, 0, None)

    assert attend(batch=0) == OK and attend(queries=0) == OK and attend(heads=0) == OK
    assert attend(heads=3) == ARG and attend(batch=-1) == ARG and attend(window=-1) == ARG and attend(pages=-1) == ARG
    assert attend(q=None) == ARG and attend(table=None) == ARG and attend(lengths=None) == ARG and attend(st=None) == ARG
    assert attend(codes=None) == ARG and attend(rng=None) == ARG and attend(scale=-1.0) == ARG and attend(scale=float("nan")) == ARG
    assert attend(rng=odd) == ARG
    assert attend(queries=1 << 25) == ARG and attend(pages=1 << 30) == ARG


def test_operators_refuse_host_tensors_and_wrong_types():
    x, codes, s = torch.zeros(2, 8), torch.zeros(2, 8).to(torch.float8_e4m3fn), torch.zeros(2, 1)
    with pytest.raises(TypeError):
        qr.quantize_fp8([[1.0]])
    with pytest.raises(TypeError):
        qr.quantize_fp8(x.double())
    for call in (lambda: qr.quantize_fp8(x), lambda: qr.dequantize_fp8(codes, s), lambda: qr.fp8_linear(codes, s, codes, s)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        qr.fp8_linear(x, s, codes, s)
    with pytest.raises(TypeError):
        qr.kv8_write(None, x, x, s)


@pytest.mark.parametrize("change, error", [
    (dict(dtype=torch.float32), TypeError), (dict(head_dim=96), ValueError), (dict(page_size=24), ValueError), (dict(page_size=8), ValueError),
    (dict(pages=-1), ValueError), (dict(kv_heads=0), ValueError), (dict(device="cpu"), RuntimeError)])
def test_cache_refuses_unsupported_shapes(change, error):
    with pytest.raises(error):
        qr.kv8_cache(**{**dict(pages=2, page_size=16, kv_heads=2, head_dim=128), **change})
