"""Host-side checks of the operators on 8- and 4-bit data: refusals before any device work (CPU)."""

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


def test_rows_entries_check_their_arguments(lib):
    def norm(x=P, xs=8, r=None, rs=0, w=None, wt=0, q=P, qs=16, scale=P, h=None, rows=2, cols=8, eps=1e-6, dtype=1):
        return lib.qrb200_rms_norm_int8(x, xs, r, rs, w, wt, q, qs, scale, h, rows, cols, eps, dtype, None)

    assert norm(rows=0) == OK and norm(cols=0) == OK  # empty: no-op
    assert norm(rows=-1) == ARG and norm(cols=32769) == ARG and norm(dtype=3) == ARG
    assert norm(x=None) == ARG and norm(q=None) == ARG and norm(scale=None) == ARG
    assert norm(r=P, rs=8) == ARG and norm(h=P) == ARG  # the residual and its sum come together
    assert norm(xs=7) == ARG and norm(qs=7) == ARG and norm(r=P, rs=7, h=P) == ARG
    assert norm(w=P, wt=2) == ARG  # a weight of another 16-bit type
    assert norm(eps=-1.0) == ARG and norm(eps=float("nan")) == ARG
    f = lib.qrb200_quantize_int8
    assert f(P, 8, P, 16, P, 0, 8, 1, None) == OK
    assert f(P, 7, P, 16, P, 2, 8, 1, None) == ARG and f(None, 8, P, 16, P, 2, 8, 1, None) == ARG
    f = lib.qrb200_dequantize_int8
    assert f(P, 8, P, P, 0, 8, 1, None) == OK
    assert f(P, 7, P, P, 2, 8, 1, None) == ARG and f(P, 8, P, None, 2, 8, 1, None) == ARG


def test_linear_entry_checks_its_arguments(lib):
    def linear(x=P, xs=16, sx=P, w=P, ws=16, sw=P, b=None, y=P, rows=2, outs=3, depth=16, dtype=1):
        return lib.qrb200_int8_linear(x, xs, sx, w, ws, sw, b, y, rows, outs, depth, dtype, None, 0, None)

    assert linear(rows=0) == OK and linear(outs=0) == OK
    assert linear(depth=0) == ARG and linear(depth=131072) == ARG and linear(dtype=7) == ARG
    assert linear(x=None) == ARG and linear(sw=None) == ARG and linear(y=None) == ARG
    assert linear(xs=15) == ARG and linear(ws=15) == ARG and linear(rows=-1) == ARG
    need = lib.qrb200_int8_linear_workspace_bytes
    assert need(P, 112, P, 112, 50, 70, 100) == 0  # rows on 16-byte boundaries
    assert need(P, 100, P, 112, 50, 70, 100) == 50 * 112 and need(ctypes.c_void_p(257), 112, P, 100, 50, 70, 100) == 120 * 112
    assert need(P, 100, P, 100, 2, 70, 100) == 0 and need(P, 100, P, 112, 0, 70, 100) == 0  # few rows are read as they lie


def test_cache_entries_check_their_arguments(lib):
    assert lib.qrb200_kv4_block_bytes(64, 128, 128) == 64 * (128 + 8)
    assert lib.qrb200_kv4_block_bytes(16, 64, 32) == 16 * (64 + 16)
    for bad in ((24, 128, 128), (8, 128, 128), (2048, 128, 128), (64, 96, 32), (64, 64, 128), (64, 128, 48), (64, 128, 0), (64, -64, 32)):
        assert lib.qrb200_kv4_block_bytes(*bad) == 0
    good = _lib.KV4Shape(4, 2, 16, 64, 1, 1)
    w, r = lib.qrb200_kv4_write, lib.qrb200_kv4_read

    def write(shape=good, cache=P, k=P, slots=P, tokens=3):
        return w(cache, ctypes.byref(shape), k, 128, 64, P, 128, 64, slots, tokens, None)

    assert write(tokens=0) == OK and write(tokens=-1) == ARG
    assert write(cache=None) == ARG and write(k=None) == ARG and write(slots=None) == ARG
    assert write(cache=ctypes.c_void_p(264)) == ARG  # not 16-byte aligned
    for shape in (_lib.KV4Shape(4, 2, 16, 64, 1, 0), _lib.KV4Shape(4, 0, 16, 64, 1, 1), _lib.KV4Shape(4, 2, 24, 64, 1, 1),
                  _lib.KV4Shape(4, 2, 16, 96, 1, 1), _lib.KV4Shape(4, 2, 16, 64, 4, 1), _lib.KV4Shape(-1, 2, 16, 64, 1, 1)):
        assert write(shape=shape) == ARG
        assert r(P, ctypes.byref(shape), P, P, P, 3, None) == ARG
    assert w(P, None, P, 0, 0, P, 0, 0, P, 3, None) == ARG
    strides = (ctypes.c_int64 * 3)(256, 256, 64)

    def attend(q=P, batch=2, queries=1, heads=4, pages=2, window=0, table=P, lengths=P, st=strides):
        return lib.qrb200_kv4_attention(q, st, P, ctypes.byref(good), table, 2, lengths, P, batch, queries, heads, pages, window, 1,
                                        0.125, None, 0, None)

    assert attend(batch=0) == OK and attend(queries=0) == OK and attend(heads=0) == OK
    assert attend(heads=3) == ARG and attend(batch=-1) == ARG and attend(window=-1) == ARG and attend(pages=-1) == ARG
    assert attend(q=None) == ARG and attend(table=None) == ARG and attend(lengths=None) == ARG and attend(st=None) == ARG


def test_status_string_of_an_index_error(lib):
    assert b"outside the cache" in lib.qrb200_status_string(_lib.QRB200_ERR_INDEX)


def test_operators_refuse_host_tensors_and_wrong_types():
    x, codes, s = torch.zeros(2, 8), torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)
    with pytest.raises(TypeError):
        qr.rms_norm_int8([[1.0]])
    with pytest.raises(TypeError):
        qr.rms_norm_int8(x.double())
    for call in (lambda: qr.rms_norm_int8(x), lambda: qr.quantize_int8(x), lambda: qr.dequantize_int8(codes, s),
                 lambda: qr.int8_linear(codes, s, codes, s)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        qr.int8_linear(x, s, codes, s)
    with pytest.raises(TypeError):
        qr.kv4_write(None, x, x, s)


@pytest.mark.parametrize("change, error", [
    (dict(dtype=torch.float32), TypeError), (dict(head_dim=96), ValueError), (dict(group_size=48), ValueError),
    (dict(head_dim=64, group_size=128), ValueError), (dict(page_size=24), ValueError), (dict(page_size=8), ValueError),
    (dict(pages=-1), ValueError), (dict(kv_heads=0), ValueError), (dict(device="cpu"), RuntimeError)])
def test_cache_refuses_unsupported_shapes(change, error):
    with pytest.raises(error):
        qr.kv4_cache(**{**dict(pages=2, page_size=16, kv_heads=2, head_dim=128), **change})
