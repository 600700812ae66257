"""The operators on 8- and 4-bit data at the ends of their ranges: how near long sums are to the 64-bit result,
numbers at either end of a type, indexes that no query needs, captured calls.

Each check derives its own tolerance; U is the unit roundoff of a type.
"""

import copy
import pickle

import pytest
import torch
from test_gpu_quant import BF, HF, SF, U, _attend64, _case, _check_rows, _randn, _values

import qr_v2_b200_kernel_b200 as qr
from qr_v2_b200_kernel_b200 import _lib

pytestmark = pytest.mark.gpu


def _half_step(x):
    """The spacing of fp16 numbers at x."""
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0**-14))) - 10)


@pytest.mark.parametrize("batch, heads, share, tokens, dim, group", [
    (4, 2, 8, 8192, 128, 128), (64, 8, 8, 8192, 128, 128), (64, 8, 8, 8192, 128, 32), (64, 8, 4, 8192, 64, 64), (20, 2, 13, 8192, 128, 64),
    (2, 8, 8, 65536, 128, 128), (64, 8, 8, 65536, 128, 128), (64, 8, 1, 65536, 64, 32)])
def test_attention_sums_hold_32_bits_at_any_length(batch, heads, share, tokens, dim, group):
    """An output that is off by e before its rounding misses the nearest fp16 number with the probability e / step. One
    unit of 2^-24 of the values' weighted mean size is allowed for e, what a handful of roundings of 32-bit sums come to."""
    pages = -(-tokens // 64)
    cache = qr.kv4_cache(pages, 64, heads, dim, group, HF)
    k, v = _randn(tokens, heads, dim, seed=80, dtype=HF), _randn(tokens, heads, dim, seed=81, dtype=HF)
    qr.kv4_write(cache, k, v, torch.arange(tokens, device="cuda"))
    q = _randn(batch, 1, heads * share, dim, seed=82, dtype=HF)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, pages)  # one context, many questions
    got = qr.kv4_attention(q, cache, table, torch.full((batch,), tokens, dtype=torch.int32, device="cuda"))
    k, v = _values(cache)
    missed, allowed, of = 0, 0.0, 0
    for b in range(0, batch, max(1, batch // 4)):
        p = (torch.einsum("hgd,thd->hgt", q[b, 0].double().unflatten(0, (heads, share)), k) * dim**-0.5).softmax(-1)
        want = torch.einsum("hgt,thd->hgd", p, v).flatten(0, 1)
        size = torch.einsum("hgt,thd->hgd", p, v.abs()).flatten(0, 1)
        missed += (got[b, 0] != want.to(HF)).sum().item()
        allowed += (size * 2.0**-24 / _half_step(want)).clamp_max(1).sum().item()
        of += want.numel()
    assert missed <= allowed, f"{missed} of {of} outputs are not the nearest, {allowed:.0f} allowed"


@pytest.mark.parametrize("base, dtype", [(b, t) for b in (0, 24, 26, 27, 28) for t in (BF, HF) if b < 28 or t is BF])
@pytest.mark.parametrize("batch, tokens", [(1, 640), (150, 640), (1, 9000)])
def test_attention_of_scores_a_rounding_apart(base, batch, tokens, dtype):
    """Scores 2^base + c 2^(base - 23) in the exponent's units, neighbours in 32 bits from 2^26 on eight or more apart:
    the weights are powers of two, the sums exact, so an output has its own rounding and no more than 2^-20 of the
    values' size beside it."""
    page = 64
    pages = -(-tokens // page)
    cache = qr.kv4_cache(pages, page, 1, 64, 32, dtype)
    unit = max(1.0, 2.0 ** (base - 23))
    k, v = torch.zeros(tokens, 1, 64, dtype=dtype, device="cuda"), _randn(tokens, 1, 64, seed=83, dtype=dtype)
    k[..., :32] = 2.0**12 if base else 0.0  # a constant group: q . k = 2^base
    at = torch.arange(tokens, device="cuda")
    climb = at * 4 // tokens + (at * 37 % 11 == 0).int()  # rises along the tokens, with single ones ahead
    k[:, 0, 32], k[:, 0, 33], k[:, 0, 34] = climb.to(dtype) + 1, 0, 15  # codes 1 to 6 of steps of one
    qr.kv4_write(cache, k, v, at)
    q = torch.zeros(batch, 1, 3, 64, dtype=dtype, device="cuda")
    q[..., 0] = 2.0 ** (base - 12) if base else 0.0
    q[..., 32] = unit
    q[:, :, 2, 32] = -unit
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, pages)
    lengths = torch.full((batch,), tokens, dtype=torch.int32, device="cuda")
    scale = 0.6931472  # times log2(e), in 32 bits, is 1
    assert float(torch.tensor(scale) * torch.tensor(1.4426950408889634)) == 1.0
    got = qr.kv4_attention(q, cache, table, lengths, scale=scale)
    keys, values = _values(cache)
    s = torch.einsum("gd,td->gt", q[0, 0].double(), keys[:tokens, 0])
    p = torch.exp2(s - s.amax(-1, keepdim=True))
    want = (p / p.sum(-1, keepdim=True)) @ values[:tokens, 0]
    assert bool(((got[:, 0].double() - want).abs() <= U[dtype] * want.abs() + 2.0**-20 * values.abs().max()).all())


# Entries' size (a power of two), eps, and the gain's size: squares or products with the gain that 32 bits cannot hold,
# and, in the last two, ordinary ones.
ROWS = [(66, 0.0, 0), (66, 1e-6, 0), (100, 1e-6, 0), (120, 1e-6, 6), (124, 0.0, -60), (-83, 0.0, 0), (-83, 1e-40, 0),
        (-60, 1e-36, 0), (-70, 0.0, 90), (-95, 0.0, 20), (60, 1e-6, 80), (100, 1e6, 100), (0, 0.0, 0), (3, 1e-6, 3)]


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("rows, cols", [(3, 50), (700, 256), (2, 1000), (2, 4096), (2, 4099), (1, 32768)])
@pytest.mark.parametrize("power, eps, gain", ROWS)
def test_norm_over_the_whole_range(power, eps, gain, rows, cols, dtype):
    """Finite rows of any size are normalised as ordinary ones are: the same bounds, and h as it was. (Where the scale
    itself is below the normal range, to its spacing.)"""
    x = _randn(rows, cols, seed=90).clamp(-4, 4).mul(2.0**power).to(dtype)
    r = _randn(rows, cols, seed=91).clamp(-4, 4).mul(2.0**power).to(dtype)
    w = _randn(cols, seed=92).clamp(-4, 4).mul(2.0**gain)
    w = w.to(dtype) if cols != 4096 else w
    for residual, weight in ((r, w), (None, w), (r, None)):
        if weight is None and gain:
            continue
        codes, scale, h = qr.rms_norm_int8(x, weight, residual, eps=eps)
        h64 = x.double() + residual.double() if residual is not None else x.double()
        e64 = torch.tensor(eps, dtype=torch.float32, device="cuda").double()
        y64 = h64 / (h64.square().mean(-1, keepdim=True) + e64).sqrt() * (weight.double() if weight is not None else 1)
        _check_rows(codes, scale, y64)
        assert bool(((h.double() - h64).abs() <= U[dtype] * h64.abs()).all())


@pytest.mark.parametrize("cols", [200, 4096, 5001])
def test_norm_of_large_rows_that_are_not_finite(cols):
    x = _randn(6, cols, seed=93, size=1e20).to(BF)
    w = _randn(cols, seed=94)
    x[1, 3], x[2, -1], x[3, 0] = float("inf"), float("nan"), -float("inf")
    codes, scale, _ = qr.rms_norm_int8(x, w)
    assert torch.isnan(scale[1:4]).all() and not codes[1:4].any() and torch.isfinite(scale[[0, 4, 5]]).all()
    for bad in (float("inf"), float("nan")):
        w[7] = bad
        codes, scale, _ = qr.rms_norm_int8(x, w)
        assert torch.isnan(scale).all() and not codes.any()


@pytest.mark.parametrize("cols", [48, 4096])
def test_norm_in_place_of_the_residual(cols):
    """The C entry may store h where the residual was (rows on 16-byte boundaries), in rows of any size."""
    lib = _lib.load()
    for dtype, code in ((BF, 1), (SF, 0)):
        for size in (1.0, 1e20):
            x, r = _randn(5, cols, seed=95, size=size).to(dtype), _randn(5, cols, seed=96, size=size).to(dtype)
            want = qr.rms_norm_int8(x, None, r)
            q, s = torch.empty(5, cols, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
            assert lib.qrb200_rms_norm_int8(x.data_ptr(), cols, r.data_ptr(), cols, None, 0, q.data_ptr(), cols, s.data_ptr(), r.data_ptr(),
                                            5, cols, 1e-6, code, torch.cuda.current_stream().cuda_stream) == 0
            assert all(torch.equal(a, b) for a, b in zip((q, s, r), want))


def test_attention_of_a_prompt_past_65535_row_tiles():
    """8200 queries, 128 heads on 8: 65600 tiles of 16 rows. Some of them against 64 bits."""
    queries, heads, share, window = 8200, 8, 16, 40
    cache = qr.kv4_cache(130, 64, heads, 64, 64, BF)
    k, v = _randn(queries, heads, 64, seed=100, dtype=BF), _randn(queries, heads, 64, seed=101, dtype=BF)
    qr.kv4_write(cache, k, v, torch.arange(queries, device="cuda"))
    q = _randn(1, queries, heads * share, 64, seed=102, dtype=BF)
    table = torch.arange(130, dtype=torch.int32, device="cuda")[None]
    got = qr.kv4_attention(q, cache, table, torch.tensor([queries], dtype=torch.int32, device="cuda"), window=window)
    k, v = _values(cache)
    for i in (0, 1, 15, 39, 40, 4000, 8190, 8191, 8192, 8199):
        lo = max(0, i - window + 1)
        p = (torch.einsum("hgd,thd->hgt", q[0, i].double().unflatten(0, (heads, share)), k[lo : i + 1]) / 8).softmax(-1)
        want = torch.einsum("hgt,thd->hgd", p, v[lo : i + 1]).flatten(0, 1)
        assert bool(((got[0, i].double() - want).abs() <= U[BF] * want.abs() + 2.0**-16 * v.abs().max()).all())


def test_attention_of_more_sequences_than_a_launch_holds():
    batch = 70000
    cache = qr.kv4_cache(500, 16, 1, 64, 64, HF)
    k, v = _randn(8000, 1, 64, seed=103, dtype=HF), _randn(8000, 1, 64, seed=104, dtype=HF)
    qr.kv4_write(cache, k, v, torch.arange(8000, device="cuda"))
    gen = torch.Generator(device="cuda").manual_seed(105)
    table = torch.randint(0, 500, (batch, 2), generator=gen, device="cuda").int()
    lengths = torch.randint(0, 33, (batch,), generator=gen, device="cuda").int()
    q = _randn(batch, 2, 2, 64, seed=106, dtype=HF)
    got = qr.kv4_attention(q.transpose(0, 1).contiguous().transpose(0, 1), cache, table, lengths)
    for lo, hi in ((0, 5), (30000, 30005), (65530, 65540), (69995, 70000)):
        assert torch.equal(got[lo:hi], qr.kv4_attention(q[lo:hi], cache, table[lo:hi], lengths[lo:hi]))


def test_sizes_beyond_the_library_are_value_errors():
    cache = qr.kv4_cache(2, 16, 1, 64, 64, BF)
    one = torch.zeros(1, 1, 1, 64, dtype=BF, device="cuda")
    table, n = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        qr.kv4_attention(one.expand(1, (1 << 24) + 1, 1, 64), cache, table, n)
    with pytest.raises(ValueError):
        qr.kv4_attention(one.expand(1, 1, 65536, 64), cache, table, n)


@pytest.mark.parametrize("page, dim", [(16, 64), (16, 128), (32, 64), (64, 128)])
@pytest.mark.parametrize("queries, window, causal", [(1, 20, True), (3, 1, True), (5, 70, True), (4, 33, False)])
def test_attention_reads_no_page_behind_the_window(queries, window, causal, page, dim):
    """Pages that the window has left may be gone from the table, wherever its start falls."""
    lengths = list(range(queries, 230, 3))
    q, cache, table, n = _case(lengths, queries, 1, 2, page, dim, 64, BF, seed=110)
    want = qr.kv4_attention(q, cache, table, n, window=window, causal=causal)
    freed = table.clone()
    for b, length in enumerate(lengths):
        freed[b, : max(0, length - queries - window + 1) // page] = -1
    assert torch.equal(want, qr.kv4_attention(q, cache, freed, n, window=window, causal=causal))
    torch.cuda.synchronize()
    qr.kv4_read(cache, torch.zeros(1, dtype=torch.int64, device="cuda"))  # nothing was reported


@pytest.mark.parametrize("scale", [0.09, 1.0, 30.0])
@pytest.mark.parametrize("power", [-100, -20, 112, 118, 125])
def test_attention_of_keys_as_small_as_queries_are_large(power, scale):
    """Queries times 2^p on keys divided by it: scores of ordinary size. Products at the bottom of 32 bits' range
    lose up to 2^-18 of a score's terms. (Where a step falls below the normal range the cache holds minima alone.)"""
    q, plain, table, lengths = _case([70, 33], 2, 2, 3, 16, 128, 64, BF, seed=120)
    k, v = _randn(128, 2, 128, seed=121).clamp(-3, 3).to(BF), _randn(128, 2, 128, seed=122, dtype=BF)
    q = q.clamp(-3.5, 3.5)
    shifted = qr.kv4_cache(plain.pages, 16, 2, 128, 64, BF)
    qr.kv4_write(shifted, k * 2.0**-power, v, torch.arange(128, device="cuda"))
    got = qr.kv4_attention(q * 2.0**power, shifted, table % 8, lengths, scale=scale)
    want, _ = _attend64(q * 2.0**power, shifted, table % 8, lengths, scale=scale)
    size = v.double().abs().max() * (scale * q.double().abs().sum(-1).max() * 3)
    assert bool(((got.double() - want).abs() <= U[BF] * 2 * want.abs() + 2.0**-18 * size).all())


@pytest.mark.parametrize("power", [95, 105, 118, 125])
def test_attention_of_large_queries_with_scales_as_small(power):
    """Queries times 2^p, the scale divided by it: every bit stays."""
    q, cache, table, lengths = _case([150, 40], 2, 2, 3, 16, 128, 64, BF, seed=123)
    q = q.clamp(-3.5, 3.5)
    a = qr.kv4_attention(q, cache, table, lengths, scale=0.1)
    assert torch.equal(a, qr.kv4_attention(q * 2.0**power, cache, table, lengths, scale=0.1 * 2.0**-power))


def test_attention_with_a_scale_of_zero_is_the_mean():
    q, cache, table, lengths = _case([150, 0, 41], 1, 2, 3, 16, 128, 64, BF, seed=124)
    for size in (1.0, 2.0**120):
        got = qr.kv4_attention(q.clamp(-3.5, 3.5) * size, cache, table, lengths, scale=0.0)
        _, v = _values(cache)
        for b, n in enumerate((150, 0, 41)):
            slots = table[b].long()[torch.arange(n, device="cuda") // 16] * 16 + torch.arange(n, device="cuda") % 16
            want = v[slots].mean(0).repeat_interleave(3, 0) if n else torch.zeros(6, 128, device="cuda", dtype=torch.float64)
            assert bool(((got[b, 0].double() - want).abs() <= U[BF] * want.abs() + 2.0**-18).all())


def test_attention_of_keys_at_the_top_of_the_type():
    """Keys of 2^120 with queries of 2^-118: scores of ordinary size."""
    q, cache, table, lengths = _case([100], 1, 1, 4, 16, 64, 64, BF, seed=125)
    k, v = _randn(112, 1, 64, seed=126).clamp(-3, 3).to(BF), _randn(112, 1, 64, seed=127, dtype=BF)
    slots, plain = torch.arange(112, device="cuda"), qr.kv4_cache(cache.pages, 16, 1, 64, 64, BF)
    qr.kv4_write(plain, k, v, slots)
    qr.kv4_write(cache, k * 2.0**120, v, slots)
    table = table % 7
    for down, scale in ((2.0**-118, 0.1), (1.0, 0.1 * 2.0**-118)):
        a = qr.kv4_attention(q, plain, table, lengths, scale=0.4)
        b = qr.kv4_attention(q * down, cache, table, lengths, scale=scale)
        assert bool(((a.double() - b.double()).abs() <= 2 * U[BF] * a.double().abs() + 2.0**-14).all())


def test_a_caches_attributes_cannot_be_assigned():
    """The kernels work on the tensor that the cache was made of; another one in its place would be ignored."""
    cache = qr.kv4_cache(2, 16, 1, 64, 64, BF)
    other = cache.data.clone()
    for name, value in (("data", other), ("pages", 1), ("page_size", 32), ("dtype", HF), ("group_size", 32)):
        with pytest.raises(AttributeError):
            setattr(cache, name, value)
    assert cache.pages == 2 and cache.page_size == 16 and cache.kv_heads == 1 and cache.head_dim == 64 and cache.dtype is BF
    block = cache.data.numel()
    unaligned = torch.zeros(block + 16, dtype=torch.uint8, device="cuda")[8 : block + 8].view(cache.data.shape)
    with pytest.raises(ValueError):
        qr.KV4Cache(unaligned, 16, 64, 64, BF)
    with pytest.raises(ValueError):
        qr.KV4Cache(cache.data.flatten(), 16, 64, 64, BF)


@pytest.mark.parametrize("dtype, largest", [(HF, 65504.0), (BF, 3.3895313892515355e38)])
@pytest.mark.parametrize("dim, group", [(64, 32), (128, 128)])
def test_cache_of_groups_that_reach_the_types_largest_number(dim, group, dtype, largest):
    """They read back finite, within half a step and what the step's rounding, here by up to its last place, moves the
    top of the range (30 u steps), rounded by u."""
    x = _randn(300, 2, dim, seed=130).mul(largest / 6).clamp(-largest, largest)
    low = torch.linspace(-1, 0.9, 300, device="cuda")[:, None] * largest
    x[:, 0, ::32], x[:, 0, 1::32] = largest, low
    x[:, 1, ::32], x[:, 1, 1::32] = -largest, -low
    x = x.to(dtype)
    slots = torch.arange(3, 303, device="cuda")
    cache = qr.kv4_cache(5, 64, 2, dim, group, dtype)
    qr.kv4_write(cache, x, -x, slots)
    for got, want in zip(qr.kv4_read(cache, slots), (x, -x)):
        g = want.double().unflatten(-1, (-1, group))
        step = (g.amax(-1) - g.amin(-1)) / 15
        assert torch.isfinite(got).all()
        off = (got.double().unflatten(-1, (-1, group)) - g).abs()
        assert bool((off <= (step * (0.5 + 30 * U[dtype])).unsqueeze(-1) + U[dtype] * largest).all())


@pytest.mark.parametrize("tokens, batch", [(60, 1), (600, 1), (700, 100), (5000, 1), (60000, 1)])
def test_attention_keeps_a_nan_value_however_little_it_weighs(tokens, batch):
    """The first token takes everything; a group of a later one's values is NaN, in whichever part of the tokens."""
    pages = -(-tokens // 64)
    cache = qr.kv4_cache(pages, 64, 1, 64, 32, BF)
    k, v = torch.zeros(tokens, 1, 64, dtype=BF, device="cuda"), _randn(tokens, 1, 64, seed=140, dtype=BF)
    k[0, 0, 0], k[1:, 0, 0] = 300, -300
    q = torch.zeros(batch, 1, 2, 64, dtype=BF, device="cuda")
    q[..., 0] = 4
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, pages)
    n = torch.full((batch,), tokens, dtype=torch.int32, device="cuda")
    for at in (1, tokens // 2, tokens - 1):
        w = v.clone()
        w[at, 0, 40] = float("nan")
        qr.kv4_write(cache, k, w, torch.arange(tokens, device="cuda"))
        got = qr.kv4_attention(q, cache, table, n)
        assert torch.isnan(got[..., 32:]).all()
        first = qr.kv4_read(cache, torch.zeros(1, dtype=torch.int64, device="cuda"))[1][0, 0, :32]
        assert torch.equal(got[..., :32], first.expand(batch, 1, 2, 32))


@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 31, 10**12, (1 << 63) - 1])
def test_attention_window_of_any_size(window):
    q, cache, table, n = _case([30, 5000, 0], 2, 1, 2, 64, 64, 64, BF, seed=150)
    for causal in (True, False):
        want = qr.kv4_attention(q, cache, table, n, causal=causal)
        assert torch.equal(want, qr.kv4_attention(q, cache, table, n, causal=causal, window=window))


# ---- captured calls -------------------------------------------------------------------------


def _replayed(call, refill):
    """`call`'s outputs when it is captured with one content of its operands and replayed with another."""
    call()  # set-up that a capture cannot hold
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    refill()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    return out


def _same(a, b):
    a, b = ((x,) if isinstance(x, torch.Tensor) else x for x in (a, b))
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("rows, cols", [(1, 4096), (33, 130), (700, 2048)])
def test_captured_rows(rows, cols):
    x, r, w = _randn(rows, cols, seed=160, dtype=BF), _randn(rows, cols, seed=161, dtype=BF), _randn(cols, seed=162, dtype=BF)
    for call in (lambda: qr.rms_norm_int8(x, w, r), lambda: qr.quantize_int8(x), lambda: qr.dequantize_int8(*qr.quantize_int8(x), BF)):
        got = _replayed(call, lambda: x.copy_(_randn(rows, cols, seed=163, size=5)))
        assert _same(got, call())


@pytest.mark.parametrize("rows, outs, depth", [(1, 512, 1024), (4, 300, 512), (16, 512, 4096), (3, 130, 1001), (64, 130, 1001), (333, 1000, 2048),
                                               (2048, 2048, 512)])
def test_captured_product(rows, outs, depth):
    x, w = (torch.randint(-127, 128, s, device="cuda").to(torch.int8) for s in ((rows, depth), (outs, depth)))
    sx, sw = torch.rand(rows, device="cuda"), torch.rand(outs, device="cuda")
    call = lambda: qr.int8_linear(x, sx, w, sw)  # noqa: E731
    got = _replayed(call, lambda: (x.neg_(), sw.mul_(2), w[0].zero_()))
    assert _same(got, call())


@pytest.mark.parametrize("lengths, queries, heads, share, dim", [([100, 0, 7], 1, 1, 2, 64), ([700], 5, 2, 8, 128), ([3000] * 3, 1, 2, 4, 128),
                                                                 ([50000], 1, 1, 8, 128), ([600] * 40, 2, 8, 2, 64)])
def test_captured_cache_and_attention(lengths, queries, heads, share, dim):
    """A decode step: the new tokens' keys and values go into the cache, and the attention reads them; replayed with other
    tokens, lengths and pages."""
    q, cache, table, n = _case([max(lengths)] * len(lengths), queries, heads, share, 64, dim, 64, HF, seed=170)
    n.copy_(torch.tensor(lengths))
    k, v = _randn(16, heads, dim, seed=171, dtype=HF), _randn(16, heads, dim, seed=172, dtype=HF)
    slots = table[0, 0].long() * 64 + torch.arange(16, device="cuda")

    def call():
        qr.kv4_write(cache, k, v, slots)
        return (qr.kv4_attention(q, cache, table, n), *qr.kv4_read(cache, slots))

    def refill():
        q.mul_(0.5), k.neg_(), v.mul_(3)
        n.copy_(n.clamp_min(1) - 1)
        full = table[:, : max(lengths) // 64]  # (the last page's unwritten slots hold NaN)
        full.copy_(full.flip(1))

    got = _replayed(call, refill)
    assert _same(got, call())


def test_operators_take_the_tensors_stream():
    """On a side stream each operator waits for nothing but that stream's work, and its results are the same."""
    x, r = _randn(300, 512, seed=180, dtype=BF), _randn(300, 512, seed=181, dtype=BF)
    q, cache, table, n = _case([300, 40], 2, 2, 2, 16, 64, 64, BF, seed=182)

    def step():
        codes, scale, h = qr.rms_norm_int8(x, None, r)
        y = qr.int8_linear(codes, scale, codes[:256], scale[:256])
        kv = y[:64].unflatten(1, (2, 2, 64))
        qr.kv4_write(cache, kv[:, 0], kv[:, 1], torch.arange(64, device="cuda"))
        return (codes, scale, h, y, qr.dequantize_int8(codes, scale, BF), qr.kv4_attention(q, cache, table, n))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert _same(got, want)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("large", [1.0, 256.0, 4096.0])
def test_attention_with_one_large_channel(large, dtype):
    """One channel of the queries far above the others, over keys that hold the same there: it takes no part in the softmax,
    but the small channels' products must keep their bits beside it. A score is off by 16 units of 2^-24 of its terms'
    sum at the most (128 products, each cut or rounded: the root of that, and some more), and an output by so
    much of its size, beside its own rounding; as root mean squares."""
    tokens, dim = 400, 128
    cache = qr.kv4_cache(7, 64, 1, dim, 128, dtype)
    k, v = _randn(tokens, 1, dim, seed=190, dtype=dtype).clamp(-3, 3), _randn(tokens, 1, dim, seed=191, dtype=dtype)
    k[..., 5], k[..., 7] = 3, -3
    qr.kv4_write(cache, k, v, torch.arange(tokens, device="cuda"))
    q = _randn(1, 1, 32, dim, seed=192, dtype=dtype)
    q[..., 5] = large
    table = torch.arange(7, dtype=torch.int32, device="cuda")[None]
    got = qr.kv4_attention(q, cache, table, torch.tensor([tokens], dtype=torch.int32, device="cuda"))[0, 0].double()
    keys, values = (x[:tokens, 0] for x in _values(cache))
    want = ((q[0, 0].double() @ keys.T) * dim**-0.5).softmax(-1) @ values
    terms = ((q[0, 0].double().abs() @ keys.abs().T) * dim**-0.5).max()
    rms = lambda x: x.square().mean().sqrt()  # noqa: E731
    assert rms(got - want) <= (rms(want.to(dtype).double() - want).square() + (16 * 2.0**-24 * terms * rms(want)).square()).sqrt() * 1.02


def test_copies_of_a_cache():
    """copy.copy is another handle on the same bytes; copy.deepcopy and pickle have their own."""
    q, cache, table, n = _case([20, 30], 1, 2, 2, 16, 64, 32, BF, seed=200)
    want = qr.kv4_attention(q, cache, table, n)
    shared, own, stored = copy.copy(cache), copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))
    for other in (shared, own, stored):
        assert torch.equal(want, qr.kv4_attention(q, other, table, n))
        assert (other.group_size, other.kv_heads, other.dtype) == (32, 2, BF)
    cache.data.zero_()
    assert not qr.kv4_attention(q, shared, table, n).any()
    assert torch.equal(want, qr.kv4_attention(q, own, table, n)) and torch.equal(want, qr.kv4_attention(q, stored, table, n))
