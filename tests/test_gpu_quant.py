"""Operators on 8- and 4-bit data against 64-bit restatements of their formulas.

Tolerances follow from the formulas: u is the unit roundoff of the result's type (one rounding),
a code is within half a step of its value, and sums in 32 bits are off by a few units of 2^-24 of
the sum of absolute values. Each check states its own.
"""

import math

import pytest
import torch

import qr_v2_b200_kernel_b200 as qr
from qr_v2_b200_kernel_b200._lib import QRB200Error

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed=0, dtype=SF, size=1.0):
    return (size * torch.randn(*shape, generator=_gen(seed), device="cuda")).to(dtype)


# ---- rows into 8 bits -----------------------------------------------------------------------


def _check_rows(codes, scale, y64):
    """y64: the values in 64 bits. Codes: half a step, and the few units of 2^-24 by which 32-bit
    factors of the code differ from exact ones (code <= 127: 2^-15). Scale: 2^-24 per factor and the
    sum's own error, cols 2^-24 at the very worst, far less for a tree of partial sums."""
    cols = y64.shape[-1]
    a = y64.abs().amax(-1)
    rel = (16 + cols / 64) * 2.0**-24
    assert torch.all((scale.double() - a / 127).abs() <= rel * a / 127)
    steps = y64 / (a / 127).clamp_min(1e-300).unsqueeze(-1)
    assert torch.all((codes.double() - steps).abs() <= 0.5 + 2.0**-14)
    assert codes.abs().max() <= 127 if codes.numel() else True


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (2, 128), (5, 130), (1, 1000), (7, 1024), (4, 1025), (3, 2048),
                                        (2, 4096), (2, 4104), (1, 8191), (3, 16384), (2, 32768), (2, 32767)])
def test_rms_norm_int8(rows, cols, dtype):
    x, r = _randn(rows, cols, seed=1, dtype=dtype), _randn(rows, cols, seed=2, dtype=dtype, size=3)
    w = _randn(cols, seed=3, dtype=dtype)
    for residual, weight in ((r, w), (r, None), (None, w), (None, w.float())):
        codes, scale, h = qr.rms_norm_int8(x, weight, residual, eps=1e-5)
        h64 = x.double() + residual.double() if residual is not None else x.double()
        y64 = h64 / (h64.square().mean(-1, keepdim=True) + 1e-5).sqrt() * (weight.double() if weight is not None else 1)
        _check_rows(codes, scale, y64)
        assert codes.dtype == torch.int8 and codes.shape == x.shape and scale.shape == (rows,)
        assert h.dtype == dtype and torch.all((h.double() - h64).abs() <= U[dtype] * h64.abs() + 1e-30)
        assert (h is x) == (residual is None)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows, cols", [(1, 1), (9, 33), (300, 176), (2, 4096)])
def test_quantize_and_dequantize_int8(rows, cols, dtype):
    x = _randn(rows, cols, seed=4, dtype=dtype)
    codes, scale = qr.quantize_int8(x)
    _check_rows(codes, scale, x.double())
    for out in (BF, HF, SF):
        v = qr.dequantize_int8(codes, scale, out)
        v64 = codes.double() * scale.double().unsqueeze(-1)
        assert v.dtype == out and torch.all((v.double() - v64).abs() <= U[out] * v64.abs() * 1.01 + 2.0**-25)


def test_rows_of_any_shape_and_stride():
    x = _randn(2, 3, 5, 40, seed=5, dtype=BF)
    codes, scale, h = qr.rms_norm_int8(x, residual=x)
    assert codes.shape == x.shape and scale.shape == (2, 3, 5) and h.shape == x.shape
    c2, s2, _ = qr.rms_norm_int8(x.reshape(30, 40), residual=x.reshape(30, 40))
    assert torch.equal(codes.reshape(30, 40), c2) and torch.equal(scale.reshape(30), s2)
    wide = _randn(6, 100, seed=6, dtype=HF)
    for view in (wide[:, 3:67], wide[:, 8:72], wide[::2, :64], wide.T[:96], wide[0].expand(4, 100), wide[0], wide[:, :1]):
        want = qr.rms_norm_int8(view.contiguous(), residual=view.contiguous())
        got = qr.rms_norm_int8(view, residual=view)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        cq, sq = qr.quantize_int8(view)
        assert torch.equal(qr.dequantize_int8(cq, sq, SF), cq.float() * sq.unsqueeze(-1))
    for shape in ((0, 8), (3, 0), (0,), (2, 0, 4)):
        e = torch.empty(shape, device="cuda", dtype=BF)
        codes, scale, h = qr.rms_norm_int8(e, residual=e)
        assert codes.shape == shape and scale.shape == shape[:-1] and h.shape == shape
        assert qr.dequantize_int8(*qr.quantize_int8(e)).shape == shape


@pytest.mark.parametrize("cols", [50, 4096, 5000])
def test_rows_that_are_zero_tiny_huge_or_not_finite(cols):
    x = _randn(7, cols, seed=7)
    x[1] = 0
    x[2] *= 1e-35
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    x[5] *= 1e15
    x[6, 0] = -float("inf")
    codes, scale, _ = qr.rms_norm_int8(x, eps=0.0)
    _check_rows(codes[[0, 5]], scale[[0, 5]], x[[0, 5]].double() / x[[0, 5]].double().square().mean(-1, keepdim=True).sqrt())
    assert not codes[1:5].any() and not codes[6].any()
    assert scale[1] == 0 and scale[2] == 0 and torch.isnan(scale[[3, 4, 6]]).all()
    values = qr.dequantize_int8(codes, scale, SF)
    assert torch.isnan(values[[3, 4, 6]]).all() and not values[1].any()
    codes, scale = qr.quantize_int8(x)
    _check_rows(codes[[0, 5]], scale[[0, 5]], x[[0, 5]].double())
    assert torch.isnan(scale[[3, 4, 6]]).all() and scale[1] == 0


def test_rows_past_32_bit_offsets():
    rows, cols = 65600, 32768  # 2.15e9 elements
    x = torch.zeros(rows, cols, dtype=BF, device="cuda")
    x[-3:] = _randn(3, cols, seed=8, dtype=BF)
    codes, scale, h = qr.rms_norm_int8(x, residual=x)
    h64 = 2 * x[-3:].double()
    _check_rows(codes[-3:], scale[-3:], h64 / (h64.square().mean(-1, keepdim=True) + 1e-6).sqrt())
    assert torch.equal(h[-3:], 2 * x[-3:]) and not codes[:-3].any()
    del x, h
    v = qr.dequantize_int8(codes, scale, BF)
    assert torch.equal(v[-3:], (codes[-3:].float() * scale[-3:, None]).to(BF))


# ---- the 8-bit product ----------------------------------------------------------------------


def _codes(rows, cols, seed, lo=-127, hi=127):
    return torch.randint(lo, hi + 1, (rows, cols), generator=_gen(seed), device="cuda").to(torch.int8)


def _check_linear(x, sx, w, sw, b, dtype):
    """The sum is exact up to its conversion to 32-bit floating point (2^-24); two products and an
    addition follow, each 2^-24 of their own, then one rounding u."""
    y = qr.int8_linear(x, sx, w, sw, b, dtype=dtype)
    p64 = (x.double() @ w.double().T) * sx.double().unsqueeze(-1) * sw.double()
    y64 = p64 + (b.double() if b is not None else 0)
    slack = 4 * 2.0**-24 * (p64.abs() + (b.double().abs() if b is not None else 0))
    assert y.dtype == dtype and y.shape == y64.shape
    assert torch.all((y.double() - y64).abs() <= U[dtype] * y64.abs() + 2 * slack + 2.0**-25)


@pytest.mark.parametrize("rows, outs, depth", [
    (1, 1, 1), (1, 128, 128), (2, 3, 5), (1, 4096, 4096), (3, 1000, 176), (16, 129, 512), (17, 127, 100), (32, 64, 2047),
    (33, 500, 48), (64, 256, 1024), (100, 260, 130), (128, 128, 16), (129, 384, 96), (255, 513, 640), (300, 130, 4096),
    (1025, 257, 352), (2048, 2048, 512), (700, 4100, 65)])
def test_int8_linear(rows, outs, depth):
    x, w = _codes(rows, depth, 10), _codes(outs, depth, 11)
    sx = torch.rand(rows, generator=_gen(12), device="cuda") * 0.05 + 0.001
    sw = torch.rand(outs, generator=_gen(13), device="cuda") * 0.01 + 0.0001
    for dtype in (BF, HF, SF):
        b = _randn(outs, seed=14, dtype=dtype)
        _check_linear(x, sx, w, sw, b if dtype != HF else None, dtype)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_int8_linear_largest_sums(rows):
    """Every product at its largest, -128 x -128, over the greatest depth: the sum reaches 2^31 - 2^14."""
    depth, outs = 131071, 3
    x = torch.full((rows, depth), -128, dtype=torch.int8, device="cuda")
    w = torch.full((outs, depth), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one = torch.ones(rows, device="cuda")
    y = qr.int8_linear(x, one, w, torch.ones(outs, device="cuda"), dtype=SF)
    want = torch.tensor([128 * 128 * depth, -128 * 127 * depth, 128 * 128 * depth], dtype=torch.float64, device="cuda")
    assert torch.equal(y, want.float().expand(rows, outs))


def test_int8_linear_strides_shapes_and_scales():
    x, w = _codes(24, 300, 15), _codes(50, 300, 16)
    sx, sw = torch.rand(24, device="cuda") + 0.5, torch.rand(50, device="cuda") + 0.5
    for lo, hi in ((0, 256), (16, 272), (1, 300), (3, 4), (7, 263)):  # bases and widths off 16 bytes
        _check_linear(x[:, lo:hi], sx, w[:, lo:hi], sw, None, SF)
    _check_linear(x[::2, :64], sx[::2], w[::3, :64], sw[::3], None, BF)
    _check_linear(x.T.contiguous().T, sx, w.T.contiguous().T, sw, None, BF)
    y = qr.int8_linear(x.reshape(2, 3, 4, 300), sx.reshape(2, 3, 4), w, sw)
    assert y.shape == (2, 3, 4, 50) and torch.equal(y.reshape(24, 50), qr.int8_linear(x, sx, w, sw))
    assert torch.equal(qr.int8_linear(x[0], sx[0], w, sw), y[0, 0, 0])
    assert qr.int8_linear(x[:0], sx[:0], w, sw).shape == (0, 50) and qr.int8_linear(x, sx, w[:0], sw[:0]).shape == (24, 0)
    sx[3], sw[4] = float("nan"), float("inf")
    y = qr.int8_linear(x, sx, w, sw, dtype=SF)
    assert torch.isnan(y[3]).all() and torch.isfinite(y).sum() == 23 * 49 and not torch.isfinite(y[:, 4]).any()


def test_int8_linear_offsets_past_32_bits():
    x, w = _codes(70000, 64, 17), _codes(32000, 64, 18)
    sx, sw = torch.ones(70000, device="cuda"), torch.ones(32000, device="cuda")
    y = qr.int8_linear(x, sx, w, sw)  # 2.24e9 outputs
    for i in (0, 33333, 69999):
        assert torch.equal(y[i], (x[i].double() @ w.double().T).to(BF))


# ---- the 4-bit cache ------------------------------------------------------------------------


def _decode(cache):
    """(codes, steps, minima) of keys and of values, from the bytes, by the documented layout."""
    P, D, NG = cache.page_size, cache.head_dim, cache.head_dim // cache.group_size
    runs = cache.data.reshape(*cache.data.shape[:2], P // 16, 16 * D + 128 * NG)
    tok, d = torch.meshgrid(torch.arange(16), torch.arange(D), indexing="ij")
    j, t, e = d // 16, d // 4 % 4, d % 4
    nib = 2 * (j % 2) + e // 2 + 4 * (e % 2)
    k_at = (tok * (D // 2) + t * (D // 8) + j // 2 * 4 + nib // 2, nib % 2)
    lane, byte, r = (d % 8) * 4 + tok % 8 // 2, 2 * (tok % 2) + tok // 8, d % 16
    v_at = (8 * D + d // 64 * 512 + lane * 16 + d // 16 % 4 * 4 + byte, r // 8)
    out = []
    for (at, nibble), pairs in ((k_at, 16 * D), (v_at, 16 * D + 64 * NG)):
        codes = runs[..., at.cuda()].int() >> (4 * nibble.cuda()) & 15  # pages, heads, runs, 16, D
        raw = runs[..., pairs : pairs + 64 * NG].contiguous().view(cache.dtype).double()
        raw = raw.reshape(*runs.shape[:2], P, NG, 2)
        out.append((codes.flatten(2, 3).double(), raw[..., 0], raw[..., 1]))
    return out


def _values(cache):
    """Keys and values in 64 bits, (slots, heads, dim)."""
    G = cache.group_size
    both = []
    for codes, s, m in _decode(cache):
        x = (m.unsqueeze(-1) + s.unsqueeze(-1) * codes.unflatten(-1, (-1, G))).flatten(-2)
        both.append(x.transpose(1, 2).flatten(0, 1))
    return both


def _fresh(pages, page, heads, dim, group, dtype, junk=True):
    cache = qr.kv4_cache(pages, page, heads, dim, group, dtype)
    if junk:  # bytes of all ones: NaN steps and minima wherever nothing was written
        cache.data.fill_(255)
    return cache


LAYOUTS = [(16, 64, 32), (64, 64, 64), (16, 128, 128), (64, 128, 32), (256, 128, 64)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page, dim, group", LAYOUTS)
@pytest.mark.parametrize("tokens, start, heads", [(1, 0, 1), (1, 15, 3), (16, 0, 2), (50, 9, 3), (131, 30, 2)])
def test_cache_write_and_read(tokens, start, heads, page, dim, group, dtype):
    """A value is within half a step of what was written, plus what rounding the step by u moves the
    top of the range (15 u steps), and u of the value once more when it is read."""
    cache = _fresh(-(-(tokens + start) // page) + 1, page, heads, dim, group, dtype)
    before = cache.data.clone()
    k, v = _randn(tokens, heads, dim, seed=20, dtype=dtype, size=2), _randn(tokens, heads, dim, seed=21, dtype=dtype)
    k[..., 3] += 20
    slots = torch.arange(start, start + tokens, device="cuda")
    qr.kv4_write(cache, k, v, slots)
    got, u = qr.kv4_read(cache, slots), U[dtype]
    for x, y, exact in zip((k, v), got, _values(cache)):
        g = x.double().unflatten(-1, (-1, group))
        step = (g.amax(-1) - g.amin(-1)) / 15
        assert torch.all((exact[slots].unflatten(-1, (-1, group)) - g).abs() <= (step * (0.5 + 16 * u)).unsqueeze(-1) + 1e-7)
        assert torch.all((y.double() - exact[slots]).abs() <= u * exact[slots].abs() + 2.0**-25)
    # nothing but the written slots changed
    other = qr.kv4_cache(cache.pages, page, heads, dim, group, dtype)
    other.data.copy_(before)
    keep = torch.ones(cache.pages * page, dtype=torch.bool, device="cuda")
    keep[slots] = False
    for a, b in zip(_decode(cache), _decode(other)):
        for p, q in zip(a, b):
            p, q = (z.transpose(1, 2).flatten(0, 1)[keep] for z in (p, q))
            assert torch.equal(torch.nan_to_num(p, nan=-1.0), torch.nan_to_num(q, nan=-1.0))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim, group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
def test_cache_codes_are_the_formulas_bit_for_bit(dim, group, dtype):
    """Steps, minima and codes as elementary 32-bit operations give them, each rounded, ties to even: a 16-bit number often
    lies midway between two codes."""
    cache = qr.kv4_cache(8, 64, 3, dim, group, dtype)
    for at, slots in ((0, torch.arange(500, device="cuda")), (1, torch.arange(7, 507, device="cuda"))):  # whole runs, and not
        k, v = (_randn(500, 3, dim, seed=60 + at + c, dtype=dtype) * (1 + c) for c in (0, 2))
        qr.kv4_write(cache, k, v, slots)
        for x, (codes, s, m) in zip((k, v), _decode(cache)):
            g = x.float().unflatten(-1, (-1, group))
            lo, hi = g.amin(-1), g.amax(-1)
            step = (hi * (1 / 15) - lo * (1 / 15)).to(dtype).float()
            want = torch.round((g - lo.unsqueeze(-1)) * (1 / step).unsqueeze(-1)).clamp(0, 15).flatten(-2)
            pick = lambda t: t.transpose(1, 2).flatten(0, 1)[slots].float()  # noqa: E731
            assert torch.equal(pick(s), step) and torch.equal(pick(m), lo) and torch.equal(pick(codes), want)


def test_cache_groups_wider_than_32_bits_reach():
    """bf16 ends whose difference overflows 32 bits: the codes are the formula's in 64 bits; ends at 0 and 15."""
    x = _randn(40, 2, 128, seed=64).mul(2.0**127).clamp(-3.2e38, 3.2e38).to(BF)
    x[:, :, 0], x[:, :, 64] = -3e38, 3e38  # each group wider than 3.4e38
    x[:, :, 1], x[:, :, 65] = 2.5e38, -2.5e38
    cache = qr.kv4_cache(4, 16, 2, 128, 64)
    slots = torch.arange(3, 43, device="cuda")
    qr.kv4_write(cache, x, -x, slots)
    for x, (codes, s, m) in zip((x, -x), _decode(cache)):
        g = x.double().unflatten(-1, (-1, 64))
        lo, hi = g.amin(-1), g.amax(-1)
        pick = lambda t: t.transpose(1, 2).flatten(0, 1)[slots].double()  # noqa: E731
        step = pick(s)
        assert torch.equal(pick(m), lo) and bool(((step - (hi - lo) / 15).abs() <= step * 2.0**-8).all())
        want = (g - lo.unsqueeze(-1)) / step.unsqueeze(-1)
        # The nearest code; near halfway (within 16 roundings of 2^-24) either.
        assert bool(((pick(codes).unflatten(-1, (-1, 64)) - want.clamp(0, 15)).abs() <= 0.5 + 15 * 2.0**-20).all())


def test_cache_codes_do_not_depend_on_how_slots_arrive():
    """The same tokens in one call, in a shuffled one, and one by one: the same bytes."""
    k, v = _randn(77, 2, 128, seed=22, dtype=BF), _randn(77, 2, 128, seed=23, dtype=BF)
    slots = torch.arange(5, 82, device="cuda")
    caches = [qr.kv4_cache(4, 32, 2, 128, 64) for _ in range(3)]
    qr.kv4_write(caches[0], k, v, slots)
    p = torch.randperm(77, generator=_gen(1), device="cuda")
    qr.kv4_write(caches[1], k[p], v[p], slots[p])
    for i in range(77):
        qr.kv4_write(caches[2], k[i : i + 1], v[i : i + 1], slots[i : i + 1])
    assert torch.equal(caches[0].data, caches[1].data) and torch.equal(caches[0].data, caches[2].data)


def test_cache_strides_padding_and_special_groups():
    cache = _fresh(3, 16, 2, 64, 32, HF)
    kv = _randn(20, 2, 2, 64, seed=24, dtype=HF)  # token, key or value, head, channel
    kv[0, :, :, :32] = 1.5  # a constant group: step 0
    kv[1, :, :, 32:] = 0
    kv[2, 0, 0, 5] = float("nan")
    kv[3, 1, 1, 40] = float("inf")
    kv[4, 0, 0] = torch.linspace(-65504, 65504, 64, device="cuda").to(HF)  # the widest range of the type
    slots = torch.arange(20, device="cuda")
    slots[[6, 19]] = -1
    kt = kv[:, 0].transpose(1, 2).contiguous().transpose(1, 2)  # channels not contiguous
    qr.kv4_write(cache, kt, kv[:, 1], slots)
    k, v = qr.kv4_read(cache, slots)
    assert torch.equal(k[0, :, :32], kv[0, 0, :, :32]) and torch.equal(v[1, :, 32:], kv[1, 1, :, 32:])
    assert torch.isnan(k[2, 0, :32]).all() and torch.isfinite(k[2, 0, 32:]).all() and torch.isfinite(k[2, 1]).all()
    assert torch.isnan(v[3, 1, 32:]).all() and torch.isfinite(v[3, 1, :32]).all()
    assert torch.isfinite(k[4]).all() and not k[6].any() and not v[19].any()
    assert all(torch.isnan(x).all() for x in qr.kv4_read(cache, torch.tensor([6], device="cuda")))  # never written
    a, b = qr.kv4_read(cache, slots[:0])
    assert a.shape == (0, 2, 64) and b.shape == (0, 2, 64)
    qr.kv4_write(cache, kv[:0, 0], kv[:0, 1], slots[:0])


def test_cache_past_32_bit_offsets():
    cache = qr.kv4_cache(520000, 64, 1, 128)  # 4.5 GB
    k, v = _randn(70, 1, 128, seed=25, dtype=BF), _randn(70, 1, 128, seed=26, dtype=BF)
    slots = 520000 * 64 - 70 + torch.arange(70, device="cuda")
    qr.kv4_write(cache, k, v, slots)
    small = qr.kv4_cache(2, 64, 1, 128)
    qr.kv4_write(small, k, v, torch.arange(58, 128, device="cuda"))
    assert torch.equal(small.data, cache.data[-2:])
    assert all(torch.equal(a, b) for a, b in zip(qr.kv4_read(cache, slots), qr.kv4_read(small, torch.arange(58, 128, device="cuda"))))
    q = _randn(1, 1, 2, 128, seed=27, dtype=BF)
    n = torch.tensor([128], dtype=torch.int32, device="cuda")
    table = torch.tensor([[519998, 519999]], dtype=torch.int32, device="cuda")
    assert torch.equal(qr.kv4_attention(q, cache, table, n), qr.kv4_attention(q, small, table - 519998, n))


def test_index_out_of_range_is_skipped_and_raised_by_the_next_call():
    cache = qr.kv4_cache(2, 16, 1, 64)
    k = _randn(3, 1, 64, seed=28, dtype=BF)
    n = torch.tensor([8], dtype=torch.int32, device="cuda")
    q = _randn(1, 1, 1, 64, seed=29, dtype=BF)
    table = torch.tensor([[0]], dtype=torch.int32, device="cuda")
    bad = torch.tensor([0, 32, 1 << 40], device="cuda")
    for call in (lambda: qr.kv4_write(cache, k, k, bad), lambda: qr.kv4_read(cache, bad),
                 lambda: qr.kv4_attention(q, cache, table + 2, n), lambda: qr.kv4_attention(q, cache, table - 1, n),
                 lambda: qr.kv4_attention(q, cache, table, n + 100), lambda: qr.kv4_attention(q, cache, table, n - 100)):
        call()
        torch.cuda.synchronize()
        with pytest.raises(QRB200Error):
            qr.kv4_read(cache, bad[:1])
        qr.kv4_read(cache, bad[:1])  # reported once


# ---- attention over the 4-bit cache ---------------------------------------------------------


def _attend64(q, cache, table, lengths, scale=None, causal=True, window=None):
    k, v = _values(cache)
    B, Q, H, D = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    top = torch.zeros((), dtype=torch.float64, device="cuda")
    share, P = H // cache.kv_heads, cache.page_size
    for b, n in enumerate(lengths.tolist()):
        at = torch.arange(n, device="cuda")
        slots = table[b].long()[at // P] * P + at % P
        kb, vb = (x[slots].repeat_interleave(share, 1) for x in (k, v))
        for i in range(Q):
            pos = n - Q + i
            lo = max(0, pos - window + 1) if window else 0
            hi = pos + 1 if causal else n
            if hi <= lo:
                continue
            s = torch.einsum("hd,thd->ht", q[b, i].double(), kb[lo:hi]) * (D**-0.5 if scale is None else scale)
            top = torch.maximum(top, s.abs().max())
            out[b, i] = torch.einsum("ht,thd->hd", s.softmax(-1), vb[lo:hi])
    return out, top.item()


def _case(lengths, queries, heads, share, page, dim, group, dtype, seed=30):
    """A cache with scattered pages, NaN wherever nothing was written, and queries."""
    per = max(1, -(-max(lengths) // page))
    cache = _fresh(len(lengths) * per + 2, page, heads, dim, group, dtype)
    table = torch.randperm(cache.pages, generator=_gen(seed), device="cuda")[: len(lengths) * per]
    table = table.reshape(len(lengths), per).int()
    for b, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        k, v = (_randn(n, heads, dim, seed=seed + 2 * b + c, dtype=dtype) for c in (1, 2))
        k[..., 7] *= 4
        qr.kv4_write(cache, k, v + 0.3, table[b].long()[at // page] * page + at % page)
    q = _randn(len(lengths), queries, heads * share, dim, seed=seed + 99, dtype=dtype)
    return q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _check_attention(q, cache, table, lengths, **options):
    """One rounding u; the scores, of size up to S, are off by a few units of 2^-24 (1 + S) times the
    spread of their terms (2^-19 in all), and weights held in two 16-bit halves by 2^-16."""
    got = qr.kv4_attention(q, cache, table, lengths, **options)
    want, top = _attend64(q, cache, table, lengths, **options)
    size = torch.nan_to_num(_values(cache)[1]).abs().max().item()
    tol = U[q.dtype] * want.abs() + (2.0**-16 + (1 + top) * 2.0**-19) * size
    assert got.shape == q.shape and got.dtype == q.dtype
    assert torch.all((got.double() - want).abs() <= tol)
    return got


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page, dim, group", LAYOUTS)
@pytest.mark.parametrize("lengths, queries, heads, share", [
    ([1], 1, 1, 1), ([17, 0, 1, 300], 1, 2, 4), ([64, 63, 65], 1, 1, 8), ([130, 5, 2], 4, 2, 3), ([700], 1, 3, 13), ([90, 33], 33, 1, 2)])
def test_attention(lengths, queries, heads, share, page, dim, group, dtype):
    _check_attention(*_case(lengths, queries, heads, share, page, dim, group, dtype))


@pytest.mark.parametrize("options", [dict(window=1), dict(window=20), dict(window=64), dict(window=1000), dict(causal=False),
                                     dict(causal=False, window=30), dict(scale=0.02), dict(scale=0.9)])
def test_attention_options(options):
    _check_attention(*_case([200, 77, 3, 0, 128], 6, 2, 2, 16, 64, 32, BF), **options)
    _check_attention(*_case([500, 0, 1], 1, 1, 4, 64, 128, 128, HF), **options)


def test_attention_window_beyond_every_position():
    args = _case([3, 40], 6, 1, 2, 16, 64, 32, BF)
    for causal in (True, False):
        want = _check_attention(*args, causal=causal)
        for window in (54, 1 << 30, (1 << 31) - 1):
            assert torch.equal(want, qr.kv4_attention(*args, causal=causal, window=window))


@pytest.mark.parametrize("lengths, heads, share, dim", [([20000], 1, 8, 128), ([9001, 12345], 2, 1, 64), ([5000] * 3, 8, 8, 128)])
def test_attention_over_long_contexts(lengths, heads, share, dim):
    args = _case(lengths, 1, heads, share, 64, dim, 64, BF)
    got = _check_attention(*args)
    for _ in range(3):  # the same bits on every call
        assert torch.equal(got, qr.kv4_attention(*args))


def test_attention_empty_rows_and_tables():
    q, cache, table, lengths = _case([3, 0], 5, 1, 2, 16, 64, 64, BF)
    out = _check_attention(q, cache, table, lengths)
    assert not out[1].any() and not out[0, :2].any() and out[0, 2:].any()
    assert not qr.kv4_attention(q, cache, table[:, :0], lengths * 0).any()
    assert qr.kv4_attention(q[:0], cache, table[:0], lengths[:0]).shape == (0, 5, 2, 64)
    assert qr.kv4_attention(q[:, :0], cache, table, lengths).shape == (2, 0, 2, 64)


def test_attention_strides_streams_and_a_poisoned_neighbour():
    q, cache, table, lengths = _case([100, 40], 3, 2, 2, 16, 128, 64, BF)
    want = _check_attention(q, cache, table, lengths)
    wide = torch.cat([table, table], 1).repeat_interleave(2, 1)[:, ::2]  # table rows and columns apart
    for other in (q.transpose(1, 2).contiguous().transpose(1, 2), q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(want, qr.kv4_attention(other, cache, wide, lengths))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qr.kv4_attention(q, cache, table, lengths)
    side.synchronize()
    assert torch.equal(want, got)
    q2 = q.clone()
    q2[0, 1, 2] = float("nan")  # one query row does not touch the others
    got = qr.kv4_attention(q2, cache, table, lengths)
    assert torch.isnan(got[0, 1, 2]).all()
    got[0, 1, 2] = want[0, 1, 2]
    assert torch.equal(want, got)


def test_attention_weights_that_underflow_and_dominate():
    """Scores far apart: one token takes everything, the others' weights are exactly zero."""
    cache = qr.kv4_cache(8, 16, 1, 64, 64, BF)
    k, v = torch.zeros(100, 1, 64, dtype=BF, device="cuda"), _randn(100, 1, 64, seed=40, dtype=BF)
    k[:, 0, 0] = torch.linspace(-300, 300, 100, device="cuda").to(BF)
    qr.kv4_write(cache, k, v, torch.arange(100, device="cuda"))
    q = torch.zeros(1, 1, 2, 64, dtype=BF, device="cuda")
    q[..., 0, 0], q[..., 1, 0] = 100, -100
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    n = torch.tensor([100], dtype=torch.int32, device="cuda")
    got = _check_attention(q, cache, table, n, scale=1.0)
    _, values = qr.kv4_read(cache, torch.tensor([99, 0], device="cuda"))
    assert torch.equal(got[0, 0], values[:, 0])


@pytest.mark.parametrize("dtype, size", [(HF, 2.0**-13), (HF, 2.0**10), (BF, 2.0**-100), (BF, 2.0**90)])
def test_attention_queries_of_any_size(dtype, size):
    """Small and large queries keep their bits: the scores only scale (a power of two, exactly)."""
    q, cache, table, lengths = _case([150, 40], 2, 2, 3, 16, 128, 64, dtype)
    q = q * 0.9  # an odd significand
    wide = q * size
    if dtype == HF:
        wide[..., 5] = 0.75 * size  # small entries beside large ones
        q = (wide.double() / size).to(HF)
        assert torch.equal(q.double() * size, wide.double())
    # the scale takes the size back, as far as 32 bits go
    a = _check_attention(q, cache, table, lengths, scale=0.1)
    if size < 2.0**40 and size > 2.0**-40:
        _check_attention(wide, cache, table, lengths, scale=0.1 / size)
    b = qr.kv4_attention(wide, cache, table, lengths, scale=0.1 / size)
    assert torch.all((a.double() - b.double()).abs() <= 2 * U[dtype] * a.double().abs() + 2.0**-14)


@pytest.mark.parametrize("power", [-90, -60, 60, 100, 110])
def test_attention_of_large_queries_and_small_keys_is_the_same_and_the_reverse(power):
    """Queries times 2^p on keys divided by it: every number only changes its exponent, so every bit of the result stays.
    (Where queries shrink the smallest partial products may leave the normal range: then to its rounding.)"""
    q, plain, table, lengths = _case([70, 33], 2, 2, 3, 16, 128, 64, BF)
    k, v = _randn(128, 2, 128, seed=66, dtype=BF), _randn(128, 2, 128, seed=67, dtype=BF)
    slots = torch.arange(128, device="cuda")
    shifted = qr.kv4_cache(plain.pages, 16, 2, 128, 64, BF)
    qr.kv4_write(plain, k, v, slots)
    qr.kv4_write(shifted, k * 2.0**-power, v, slots)
    a = qr.kv4_attention(q, plain, table % 8, lengths)
    b = qr.kv4_attention(q * 2.0**power, shifted, table % 8, lengths)
    if power > 0:
        assert torch.equal(a, b)
    else:
        assert torch.all((a.double() - b.double()).abs() <= 2 * U[BF] * a.double().abs() + 2.0**-14)


@pytest.mark.parametrize("scale", [0.7, 1.0, 5.0])
def test_attention_of_large_queries_with_a_scale_above_one(scale):
    """As above, every bit of the result stays; the scale comes in where the queries' size is taken back."""
    q, plain, table, lengths = _case([70, 33], 2, 2, 3, 16, 128, 64, BF)
    k, v = _randn(128, 2, 128, seed=68, dtype=BF), _randn(128, 2, 128, seed=69, dtype=BF)
    slots = torch.arange(128, device="cuda")
    shifted = qr.kv4_cache(plain.pages, 16, 2, 128, 64, BF)
    qr.kv4_write(plain, k, v, slots)
    qr.kv4_write(shifted, k * 2.0**-100, v, slots)
    a = qr.kv4_attention(q, plain, table % 8, lengths, scale=scale)
    assert torch.equal(a, qr.kv4_attention(q * 2.0**100, shifted, table % 8, lengths, scale=scale))


# ---- refusals -------------------------------------------------------------------------------


def test_refusals():
    x, w = _randn(4, 32, seed=50, dtype=BF), _randn(32, seed=51, dtype=BF)
    codes, s = qr.quantize_int8(x)
    for call in (lambda: qr.rms_norm_int8(x, w[:31]), lambda: qr.rms_norm_int8(x, w, x[:3]), lambda: qr.rms_norm_int8(x, eps=-1.0),
                 lambda: qr.rms_norm_int8(torch.empty(1, 32769, device="cuda")), lambda: qr.rms_norm_int8(x.sum()),
                 lambda: qr.dequantize_int8(codes, s[:3]), lambda: qr.int8_linear(codes, s, codes[:, :16], s),
                 lambda: qr.int8_linear(codes, s[:2], codes, s), lambda: qr.int8_linear(codes, s, codes, s[:2]),
                 lambda: qr.int8_linear(codes, s, codes, s, w[:3]), lambda: qr.int8_linear(codes[:, :0], s, codes[:, :0], s),
                 lambda: qr.int8_linear(codes, s, codes[0], s)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: qr.rms_norm_int8(x, w.half()), lambda: qr.rms_norm_int8(x, None, x.float()), lambda: qr.quantize_int8(codes),
                 lambda: qr.dequantize_int8(codes, s, torch.float64), lambda: qr.int8_linear(codes, s.half(), codes, s),
                 lambda: qr.int8_linear(codes, s, codes, s, w[:4].float())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: qr.rms_norm_int8(x.cpu()), lambda: qr.rms_norm_int8(x, w.cpu()), lambda: qr.int8_linear(codes, s, codes.cpu(), s)):
        with pytest.raises(RuntimeError):
            call()
    g = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no_grad"):
        qr.rms_norm_int8(g)
    with torch.no_grad():
        qr.rms_norm_int8(g)


def test_cache_from_bytes():
    """A cache's bytes are its whole state; bytes that do not fit the layout are refused."""
    q, cache, table, n = _case([20, 30], 1, 2, 2, 16, 64, 32, BF)
    copy = qr.KV4Cache(cache.data.clone(), 16, 64, 32, BF)
    assert torch.equal(qr.kv4_attention(q, cache, table, n), qr.kv4_attention(q, copy, table, n))
    for bad in (lambda: qr.KV4Cache(cache.data[..., :-16], 16, 64, 32, BF), lambda: qr.KV4Cache(cache.data, 32, 64, 32, BF),
                lambda: qr.KV4Cache(cache.data[0], 16, 64, 32, BF), lambda: qr.KV4Cache(cache.data, 16, 64, 24, BF)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        qr.KV4Cache(cache.data.int(), 16, 64, 32, BF)


def test_cache_refusals():
    q, cache, table, n = _case([20, 30], 1, 2, 2, 16, 64, 64, BF)
    k, slots = _randn(3, 2, 64, seed=52, dtype=BF), torch.arange(3, device="cuda")
    for call in (lambda: qr.kv4_write(cache, k[:2], k, slots), lambda: qr.kv4_write(cache, k, k[..., :32], slots),
                 lambda: qr.kv4_write(cache, k, k, slots[None]), lambda: qr.kv4_attention(q[..., :32], cache, table, n),
                 lambda: qr.kv4_attention(q[:, :, :3], cache, table, n), lambda: qr.kv4_attention(q[0], cache, table, n),
                 lambda: qr.kv4_attention(q, cache, table[:1], n), lambda: qr.kv4_attention(q, cache, table, n[:1]),
                 lambda: qr.kv4_attention(q, cache, table, n, window=0),
                 lambda: qr.kv4_attention(q, cache, table, n, scale=-1.0), lambda: qr.kv4_attention(q, cache, table, n, scale=float("nan"))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: qr.kv4_write(cache, k.half(), k, slots), lambda: qr.kv4_write(cache, k, k, slots.int()),
                 lambda: qr.kv4_attention(q.half(), cache, table, n), lambda: qr.kv4_attention(q, cache, table.long(), n),
                 lambda: qr.kv4_attention(q, cache, table, n.long()), lambda: qr.kv4_read(cache.data, slots)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: qr.kv4_write(cache, k.cpu(), k, slots), lambda: qr.kv4_attention(q.cpu(), cache, table, n),
                 lambda: qr.kv4_attention(q.clone().requires_grad_(), cache, table, n)):
        with pytest.raises(RuntimeError):
            call()
