"""The 8-bit cache and attention over it, against 64-bit restatements.

The cache: ranges are exact (the largest magnitude rounded up to three significant bits), codes are compared
for equality with those of the exact quotients, values are one product of 32 bits, rounded once. Attention, over the
values that the cache holds: see ``_check_attention``.
"""

import copy
import math

import pytest
import torch

import qr_v2_b200_kernel_b200 as qr
from qr_v2_b200_kernel_b200._lib import QRB200Error

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed=0, dtype=BF, size=1.0):
    return (size * torch.randn(*shape, generator=_gen(seed), device="cuda")).to(dtype)


# ---- the cache ------------------------------------------------------------------------------


def _range(a, most):
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(1e-300))) - 2)
    up = torch.ceil(a / step) * step
    up = torch.where(up <= most, up, a)  # no value reads back as infinity
    return torch.where(a >= 2.0**-100, up, 0.0)


class Model:
    """The cache in 64 bits: codes and ranges, as their definition has them."""

    def __init__(self, pages, page, heads, dim):
        self.page = page
        self.codes = torch.zeros(2, pages, page, heads, dim, dtype=torch.float64, device="cuda")
        self.range = torch.zeros(2, pages, heads, dtype=torch.float64, device="cuda")

    def write(self, k, v, slots):
        slots = slots.tolist()
        for page in sorted({s // self.page for s in slots if s >= 0}):
            rows = [i for i, s in enumerate(slots) if s >= 0 and s // self.page == page]
            at = [slots[i] % self.page for i in rows]
            for part, x in enumerate((k, v)):
                most, x = torch.finfo(x.dtype).max, x[rows].double()
                old = torch.zeros_like(self.range[part, page]) if 0 in at else self.range[part, page].clone()
                new = torch.maximum(old, _range(x.abs().amax((0, 2)), most))
                safe = torch.where(new > 0, new, 1.0)[None, :, None]
                self.codes[part, page] = (self.codes[part, page] * old[None, :, None] / safe).round()
                self.codes[part, page, at] = torch.where(new[None, :, None] > 0, (127 * x / safe).round(), 0.0)
                self.range[part, page] = new

    def check(self, cache, slots):
        assert torch.equal(cache.range.double().permute(2, 0, 1), self.range)
        for part, got in enumerate(qr.kv8_read(cache, slots)):
            page, at = slots // self.page, slots % self.page
            step = self.range[part, page] / 127
            want = self.codes[part, page, at] * step.unsqueeze(-1)
            assert got.dtype == cache.dtype
            # which code it is shows through one rounding: 127 half steps are less than half a code
            assert torch.equal((got.double() / step.clamp_min(1e-300).unsqueeze(-1)).round(), torch.where(step.unsqueeze(-1) > 0, self.codes[part, page, at], 0.0))
            assert torch.all((got.double() - want).abs() <= (U[cache.dtype] + 2.0**-22) * want.abs() + (2.0**-25 if cache.dtype == HF else 0))


def _all(cache):
    return torch.arange(cache.pages * cache.page_size, device="cuda")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page, heads", [(16, 1), (64, 3), (256, 2), (1024, 1)])
def test_writes_in_any_order_and_number(page, heads, dim, dtype):
    pages = 7
    cache, model = qr.kv8_cache(pages, page, heads, dim, dtype=dtype), Model(pages, page, heads, dim)
    model.check(cache, _all(cache))
    order = torch.randperm(pages * page, generator=_gen(1), device="cuda")
    for i, n in enumerate((1, 2, 17, 100, 3, 400, 1, 64)):  # scattered tokens, their sizes growing
        slots = order[i * n % 50 : i * n % 50 + n] if n < 64 else torch.randperm(pages * page, generator=_gen(i), device="cuda")[:n]
        k, v = _randn(len(slots), heads, dim, seed=i, dtype=dtype, size=1 + i), _randn(len(slots), heads, dim, seed=50 + i, dtype=dtype)
        qr.kv8_write(cache, k, v, slots)
        model.write(k, v, slots)
        model.check(cache, _all(cache))


@pytest.mark.parametrize("dtype, dim", [(BF, 128), (HF, 64)])
def test_token_by_token_and_begun_anew(dtype, dim):
    cache, model = qr.kv8_cache(3, 16, 2, dim, dtype=dtype), Model(3, 16, 2, dim)
    for turn in range(2):  # the second sequence takes over the first one's page
        for j in range(16 - 5 * turn):
            k, v = _randn(1, 2, dim, seed=j, dtype=dtype, size=1 + 0.3 * j), _randn(1, 2, dim, seed=90 + j, dtype=dtype, size=2.0 ** -j)
            slots = torch.tensor([16 + j], device="cuda")
            qr.kv8_write(cache, k, v, slots)
            model.write(k, v, slots)
            model.check(cache, _all(cache))


@pytest.mark.parametrize("tokens", [255, 256, 257, 1024, 1025, 5000])
def test_many_tokens_as_few(tokens):
    # the same rows in one call, whichever way their pages are looked up, and in the order of time
    heads, dim, page, batch = 2, 64, 64, 5
    per = -(-tokens // batch)
    k, v = _randn(batch * per, heads, dim, seed=1), _randn(batch * per, heads, dim, seed=2)
    at = torch.arange(3, 3 + per, device="cuda")
    pages = -(-(per + 3) // page)
    table = torch.randperm(batch * pages, generator=_gen(3), device="cuda").reshape(batch, pages)
    slots = (table[:, at // page] * page + at % page).reshape(-1)
    caches = [qr.kv8_cache(batch * pages, page, heads, dim) for _ in range(3)]
    qr.kv8_write(caches[0], k, v, slots)
    order = torch.arange(batch * per, device="cuda").reshape(batch, per).T.reshape(-1)
    qr.kv8_write(caches[1], k[order], v[order], slots[order])
    model = Model(batch * pages, page, heads, dim)
    model.write(k, v, slots)
    for c in caches[:2]:
        model.check(c, slots)
    assert torch.equal(caches[0].data, caches[1].data)
    holes = slots.clone()
    holes[::7] = -1
    kept = holes >= 0
    qr.kv8_write(caches[2], k, v, holes)
    short = Model(batch * pages, page, heads, dim)
    short.write(k[kept], v[kept], holes[kept])
    short.check(caches[2], slots)


@pytest.mark.parametrize("dtype, dim, page, pages", [(BF, 128, 64, 300), (HF, 64, 16, 400), (BF, 64, 256, 120), (HF, 128, 1024, 12)])
def test_pages_that_get_few_tokens_and_pages_that_get_many(dtype, dim, page, pages):
    # many rows in a call, from one to all of a page's; a second call over the first, larger, so that codes move
    heads = 3
    cache, model = qr.kv8_cache(pages, page, heads, dim, dtype=dtype), Model(pages, page, heads, dim)
    for turn in range(2):
        counts = [1, 8, 9, 2, page, 7, 10][turn:]
        slots = torch.cat([p * page + torch.randperm(page, generator=_gen(100 * turn + p), device="cuda")[: min(page, counts[p % len(counts)])] for p in range(pages)])
        slots = slots[torch.randperm(len(slots), generator=_gen(turn), device="cuda")]
        assert len(slots) > 1024
        k, v = _randn(len(slots), heads, dim, seed=turn, dtype=dtype, size=1 + 2 * turn), _randn(len(slots), heads, dim, seed=7 + turn, dtype=dtype, size=4 - 3 * turn)
        qr.kv8_write(cache, k, v, slots)
        model.write(k, v, slots)
        model.check(cache, _all(cache))


def test_rest_of_a_page_begun_anew_reads_as_zeros():
    cache = qr.kv8_cache(2, 32, 1, 64)
    qr.kv8_write(cache, _randn(64, 1, 64, seed=1), _randn(64, 1, 64, seed=2), torch.arange(64, device="cuda"))
    before = [x.clone() for x in qr.kv8_read(cache, torch.arange(32, 64, device="cuda"))]
    qr.kv8_write(cache, _randn(2, 1, 64, seed=3), _randn(2, 1, 64, seed=4), torch.tensor([5, 0], device="cuda"))
    k, v = qr.kv8_read(cache, _all(cache))
    rest = torch.ones(32, dtype=torch.bool, device="cuda")
    rest[[0, 5]] = False
    assert torch.all(k[:32][rest] == 0) and torch.all(v[:32][rest] == 0) and torch.all(k[0] != 0)
    assert torch.equal(k[32:], before[0]) and torch.equal(v[32:], before[1])


def test_ends_of_the_types_ranges():
    for dtype, sizes in ((BF, (2.0**-99, 2.0**-60, 1.0, 2.0**60, 3.3e38)), (HF, (2.0**-14, 1.0, 65504.0))):
        for size in sizes:
            x = _randn(40, 2, 64, seed=7, dtype=torch.float32)
            k = (x / x.abs().max() * size).to(dtype)
            cache, model = qr.kv8_cache(2, 32, 2, 64, dtype=dtype), Model(2, 32, 2, 64)
            for slots in (torch.arange(0, 40, 2, device="cuda"), torch.arange(1, 41, 2, device="cuda")):
                qr.kv8_write(cache, k[slots], -k[slots], slots)
                model.write(k[slots], -k[slots], slots)
                model.check(cache, torch.arange(41, device="cuda"))
    cache = qr.kv8_cache(1, 16, 1, 64)
    qr.kv8_write(cache, _randn(16, 1, 64, size=2.0**-120), _randn(16, 1, 64), torch.arange(16, device="cuda"))
    k, v = qr.kv8_read(cache, torch.arange(16, device="cuda"))
    assert torch.all(k == 0) and cache.range[0, 0, 0] == 0 and torch.all(v.isfinite())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_not_finite_until_begun_anew(bad):
    cache = qr.kv8_cache(3, 16, 2, 64)
    every = torch.arange(48, device="cuda")
    k, v = _randn(48, 2, 64, seed=1), _randn(48, 2, 64, seed=2)
    qr.kv8_write(cache, k, v, every)
    was = qr.kv8_read(cache, every)
    k2 = k.clone()
    k2[20, 1, 5] = bad
    qr.kv8_write(cache, k2[20:21], v[20:21], every[20:21])
    for step in range(2):
        got = qr.kv8_read(cache, every)
        assert got[0][16:32, 1].isnan().all() and got[0].isnan().sum() == 16 * 64
        assert torch.equal(got[1], was[1]) and torch.equal(got[0][:16], was[0][:16]) and torch.equal(got[0][16:32, 0], was[0][16:32, 0])
        qr.kv8_write(cache, k[21:22], v[21:22], every[21:22])  # a good one changes nothing yet
    qr.kv8_write(cache, k[16:32], v[16:32], every[16:32])
    assert all(torch.equal(a, b) for a, b in zip(qr.kv8_read(cache, every), was))


def test_strides_padding_and_slots_outside():
    cache, model = qr.kv8_cache(4, 16, 2, 64), Model(4, 16, 2, 64)
    base = _randn(30, 2 + 2 * 2, 65, seed=3)
    slots = torch.randperm(64, generator=_gen(2), device="cuda")[:30]
    for k, v in ((base[:, 2:4, :64], base[:, 4:6, 1:]), (base[:, 0:2, 1:], base.flip(0)[:, 2:4, :64]),
                 (base.transpose(1, 2)[:, :64, :2].transpose(1, 2), base[:, :2, ::1][:, :, 1:])):
        qr.kv8_write(cache, k, v, slots)
        model.write(k, v, slots)
        model.check(cache, _all(cache))
    odd = base[:, :2, :64].transpose(0, 2).contiguous().transpose(0, 2)  # channels not contiguous
    qr.kv8_write(cache, odd, odd, slots)
    model.write(odd, odd, slots)
    model.check(cache, _all(cache))
    before = cache.data.clone()
    qr.kv8_write(cache, odd, odd, torch.full_like(slots, -1))
    assert torch.equal(cache.data, before)
    k, v = qr.kv8_read(cache, torch.tensor([-1, 3], device="cuda"))
    assert torch.all(k[0] == 0) and torch.all(v[0] == 0)
    qr.kv8_write(cache, odd[:2], odd[:2], torch.tensor([64, 2**40], device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(QRB200Error):
        qr.kv8_read(cache, slots)
    assert torch.equal(cache.data, before)
    k, _ = qr.kv8_read(cache, torch.tensor([64], device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(QRB200Error):
        qr.kv8_read(cache, slots)
    assert torch.all(k == 0)
    qr.kv8_write(cache, odd[:0], odd[:0], slots[:0])


def test_a_slot_given_twice_spoils_nothing_else():
    cache, other = qr.kv8_cache(2, 16, 1, 64), qr.kv8_cache(2, 16, 1, 64)
    k = _randn(20, 1, 64, seed=1)
    slots = torch.arange(20, device="cuda")
    slots[7] = 3
    for tokens in (20, 1100):
        s = torch.cat([slots, torch.full((tokens - 20,), -1, device="cuda")])
        kk = torch.cat([k, k[:1].expand(tokens - 20, -1, -1)])
        qr.kv8_write(cache, kk, kk, s)
        got, _ = qr.kv8_read(cache, torch.arange(32, device="cuda"))
        step = cache.range[:, 0, 0].double() / 127
        keep = [i for i in range(20) if i not in (3, 7)]
        assert torch.all((got[keep].double() - k[keep].double()).abs() <= (0.5 + 127 * U[BF]) * step[torch.tensor(keep, device="cuda") // 16, None, None])


def test_copies_and_refusals():
    cache = qr.kv8_cache(2, 16, 2, 64)
    qr.kv8_write(cache, _randn(32, 2, 64), _randn(32, 2, 64, seed=1), torch.arange(32, device="cuda"))
    deep, shallow = copy.deepcopy(cache), copy.copy(cache)
    assert deep.data.data_ptr() != cache.data.data_ptr() and shallow.range.data_ptr() == cache.range.data_ptr()
    assert torch.equal(deep.data, cache.data) and torch.equal(deep.range, cache.range)
    with pytest.raises(AttributeError):
        cache.range = deep.range
    k, slots = _randn(3, 2, 64), torch.arange(3, device="cuda")
    table, lengths, q = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"), _randn(1, 1, 4, 64)
    for call, error in (
            (lambda: qr.kv8_write(None, k, k, slots), TypeError), (lambda: qr.kv8_write(cache, k.half(), k, slots), TypeError),
            (lambda: qr.kv8_write(cache, k, k[:2], slots), ValueError), (lambda: qr.kv8_write(cache, k, k, slots.int()), TypeError),
            (lambda: qr.kv8_write(cache, k, k, slots[:2]), ValueError), (lambda: qr.kv8_write(cache, k.cpu(), k, slots), RuntimeError),
            (lambda: qr.kv8_write(cache, k.clone().requires_grad_(), k, slots), RuntimeError),
            (lambda: qr.kv8_read(cache, slots.cpu()), RuntimeError), (lambda: qr.kv8_read(qr.kv4_cache(2, 16, 2, 64), slots), TypeError),
            (lambda: qr.KV8Cache(cache.data, cache.range[:1], 16, 64, BF), ValueError), (lambda: qr.KV8Cache(cache.data, cache.range, 32, 64, BF), ValueError),
            (lambda: qr.KV8Cache(cache.data, cache.range, 16, 64, torch.float32), TypeError),
            (lambda: qr.KV8Cache(cache.data, torch.zeros(9, device="cuda")[1:].view(2, 2, 2), 16, 64, BF), ValueError),  # off 8 bytes
            (lambda: qr.kv8_attention(q.half(), cache, table, lengths), TypeError), (lambda: qr.kv8_attention(q[:, :, :3], cache, table, lengths), ValueError),
            (lambda: qr.kv8_attention(q, cache, table.long(), lengths), TypeError), (lambda: qr.kv8_attention(q, cache, table[0], lengths), ValueError),
            (lambda: qr.kv8_attention(q, cache, table, lengths, window=0), ValueError), (lambda: qr.kv8_attention(q, cache, table, lengths, scale=-1.0), ValueError),
            (lambda: qr.kv8_attention(q, cache, table, lengths, scale=float("nan")), ValueError)):
        with pytest.raises(error):
            call()


# ---- attention ------------------------------------------------------------------------------


def _filled(batch, capacity, heads, dim, page, dtype, seed=0, spare=2):
    """A cache of full sequences in scattered pages, its table, and its values in 64 bits (batch, capacity, heads, dim)."""
    per = -(-capacity // page)
    table = torch.randperm(batch * per + spare, generator=_gen(seed), device="cuda")[: batch * per].reshape(batch, per).int()
    cache = qr.kv8_cache(batch * per + spare, page, heads, dim, dtype=dtype)
    at = torch.arange(per * page, device="cuda")
    slots = table.long()[:, at // page] * page + at % page
    size = torch.exp(0.5 * torch.randn(batch * per * page, 1, 1, generator=_gen(seed + 1), device="cuda"))
    k = (_randn(batch * per * page, heads, dim, seed=seed + 2, dtype=torch.float32) * size + 0.5).to(dtype)
    v = (_randn(batch * per * page, heads, dim, seed=seed + 3, dtype=torch.float32) * size).to(dtype)
    qr.kv8_write(cache, k, v, slots.reshape(-1))
    return cache, table, _values(cache, slots)


def _values(cache, slots):
    out = []
    for part, x in enumerate(qr.kv8_read(cache, slots.reshape(-1))):
        step = cache.range[..., part].double()[slots.reshape(-1) // cache.page_size].unsqueeze(-1) / 127
        code = (x.double() / step.clamp_min(1e-300)).round()
        out.append((code * step).unflatten(0, slots.shape))
    return out


def _check_attention(q, cache, table, lengths, values, scale=None, causal=True, window=None):
    """Scores are sums of 32 bits: off by at most dim + 4 steps of 2^-23 of their terms' magnitudes (d below); weights by
    twice that (theirs and the largest one's), 2^-20 for the exponential, and, where there are more than 16 query rows a key
    head, 2^-11, half a step of the 16 bits that then hold them; sums of weights and values by 2^-20 of the magnitudes (splits of 32-bit sums).
    One rounding on top.

    And a floor: a weight is two fp16 numbers, high and low, of p w 2^10 / cap with w a value's step and cap < 2 w the power of two
    above the largest; fp16 numbers are 2^-24 apart at least, so the low one leaves up to 2^-25, which a code (at most 127)
    turns into 127 2^-35 cap <= 2^-34 times the largest 127 w, the largest range R of the values. Weights are taken against the
    largest score or one below it, so their sum is at least 1, and each of the n tokens adds no more than that: n 2^-34 R.
    (Found with one weight of 0.9999998 whose value's code is 0, and a result of 1e-8 from weights of 2^-25.)"""
    out = qr.kv8_attention(q, cache, table, lengths, scale=scale, causal=causal, window=window)
    batch, queries, heads, dim = q.shape
    k64, v64 = values
    share = heads // k64.shape[2]
    factor = dim**-0.5 if scale is None else scale
    for b in range(batch):
        n = int(lengths[b])
        k, v = (x[b, :n].repeat_interleave(share, 1) for x in (k64, v64))  # tokens, heads, dim
        pos = n - queries + torch.arange(queries, device="cuda")
        at = torch.arange(n, device="cuda")
        seen = (at <= pos[:, None]) if causal else torch.ones(queries, n, dtype=torch.bool, device="cuda")
        if window:
            seen = seen & (at > pos[:, None] - window)
        s = torch.einsum("qhd,thd->hqt", q[b].double(), k) * factor
        terms = torch.einsum("qhd,thd->hqt", q[b].double().abs(), k.abs()) * factor
        s = s.masked_fill(~seen, -math.inf)
        some = seen.any(-1)
        p = torch.where(some[:, None], torch.softmax(s, -1), 0.0).nan_to_num(0.0)
        want = torch.einsum("hqt,thd->qhd", p, v)
        size = torch.einsum("hqt,thd->qhd", p, v.abs()) if n else torch.zeros_like(want)
        d = (torch.where(seen, terms, 0.0).amax(-1) if n else torch.zeros(heads, queries, device="cuda")) * (dim + 4) * 2.0**-23
        weights = (2 * d).exp() - 1 + 2.0**-19 + (2.0**-11 if queries * share > 16 else 0.0)
        floor = n * 2.0**-34 * cache.range[table[b, : -(-n // cache.page_size)].long(), :, 1].double().nan_to_num(0.0).amax() if n else 0.0
        bound = U[q.dtype] * want.abs() + 2 * weights.T[..., None] * size + (2.0**-24 if q.dtype == HF else 0) + floor
        err = (out[b].double() - want).abs()
        odd = ~q[b].isfinite().all(-1, keepdim=True) & some[:, None, None]  # such a query has no scores
        assert torch.all((err <= bound) | odd), (b, (err / bound.clamp_min(1e-300)).max().item())
        assert torch.all(out[b].isnan() | ~odd)
        assert torch.all(out[b][~some] == 0)
    return out


def _lengths(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads, share, page, queries, window", [
    (1, 1, 16, 1, None), (2, 4, 64, 1, None), (2, 8, 32, 1, 100), (1, 3, 64, 5, None), (2, 3, 16, 5, 37), (1, 16, 128, 1, None), (1, 5, 1024, 7, 7),
    (2, 2, 64, 16, None), (1, 4, 64, 40, 64), (2, 1, 16, 130, None)])
def test_attention(heads, share, page, queries, window, dim, dtype):
    cache, table, values = _filled(5, 517, heads, dim, page, dtype, seed=share + page)
    q = _randn(5, queries, heads * share, dim, seed=9, dtype=dtype)
    for lengths in (_lengths(517, 0, 1, 300, 64), _lengths(queries, max(0, queries - 1), 33, 16, 511)):
        _check_attention(q, cache, table, lengths, values, window=window)
        _check_attention(q, cache, table, lengths, values, window=window, causal=False, scale=0.3)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads, share, queries, length, window, causal", [
    (2, 1, 127, 127, None, True), (1, 4, 33, 400, None, True), (1, 1, 129, 1000, 50, True), (2, 3, 200, 203, None, True), (1, 8, 100, 640, 129, True),
    (1, 2, 300, 300, None, False), (1, 16, 17, 1025, 400, False), (2, 1, 1000, 1000, 1, True), (1, 4, 640, 1200, None, True)])
def test_prompts(heads, share, queries, length, window, causal, dim, dtype):
    cache, table, values = _filled(2, length, heads, dim, 64, dtype, seed=queries)
    q = _randn(2, queries, heads * share, dim, seed=9, dtype=dtype)
    for lengths in (_lengths(length, length - length // 3), _lengths(queries // 2, 0)):
        _check_attention(q, cache, table, lengths, values, window=window, causal=causal)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, heads, share, page, queries, capacity, window, causal", [
    (40, 8, 4, 16, 40, 200, None, True), (40, 8, 4, 64, 33, 130, 50, True), (48, 4, 8, 32, 40, 190, None, False), (30, 8, 1, 64, 200, 260, 70, False),
    (70, 3, 5, 128, 52, 100, 1, True), (4, 8, 2, 64, 500, 1000, None, True), (3, 8, 4, 16, 300, 1100, 333, True), (1, 4, 16, 1024, 700, 1300, None, True)])
def test_many_prompts(batch, heads, share, page, queries, capacity, window, causal, dim, dtype):
    # enough of them for tiles of 256 rows, whose rows begin and end anywhere, before the sequence's start too
    cache, table, values = _filled(batch, capacity, heads, dim, page, dtype, seed=queries)
    q = _randn(batch, queries, heads * share, dim, seed=9, dtype=dtype)
    lengths = torch.randint(0, capacity + 1, (batch,), generator=_gen(7), device="cuda").int()
    if batch >= 4:
        lengths[:4] = torch.tensor([capacity, 0, 1, min(capacity, queries - 1)])
    _check_attention(q, cache, table, lengths, values, window=window, causal=causal)


def test_many_prompts_over_pages_that_are_wrong_or_not_finite():
    batch, heads, dim, queries, n = 40, 8, 64, 40, 200
    cache, table, values = _filled(batch, n, heads, dim, 16, BF, seed=5)
    q = _randn(batch, queries, heads * 4, dim, seed=6)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    want = qr.kv8_attention(q, cache, table, lengths)
    seen = qr.kv8_attention(q, cache, table, lengths, window=30)
    for part in (0, 1):  # a page shows in the queries that see it
        spoiled = copy.deepcopy(cache)
        spoiled.range[table[:, 11].long(), :, part] = float("nan")  # tokens 176 to 191
        got = qr.kv8_attention(q, spoiled, table, lengths)
        pos = n - queries + torch.arange(queries, device="cuda")
        assert got[:, pos >= 176].isnan().all() and torch.equal(got[:, pos < 176], want[:, pos < 176])
    # behind the window anything goes
    spoiled = copy.deepcopy(cache)
    spoiled.range[table[:, :8].long()] = float("nan")
    gone = table.clone()
    gone[:, :8] = 2**31 - 1
    assert torch.equal(qr.kv8_attention(q, spoiled, table, lengths, window=30), seen)
    assert torch.equal(qr.kv8_attention(q, spoiled, gone, lengths, window=30), seen)
    # a page that the table has wrong is left out, and reported
    gone = table.clone()
    gone[:, 3] = -1
    got = qr.kv8_attention(q, cache, gone, lengths, causal=False)
    torch.cuda.synchronize()
    with pytest.raises(QRB200Error):
        qr.kv8_attention(q, cache, table, lengths)
    without = [torch.cat([v[:, :48], v[:, 64:n]], 1) for v in values]
    for b in (0, 39):
        k, v = (x[b].repeat_interleave(4, 1) for x in without)
        p = torch.softmax(torch.einsum("qhd,thd->hqt", q[b].double(), k) * dim**-0.5, -1)
        exact = torch.einsum("hqt,thd->qhd", p, v)
        size = torch.einsum("hqt,thd->qhd", p, v.abs())
        assert torch.all((got[b].double() - exact).abs() <= U[BF] * exact.abs() + 2.0**-9 * size)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_many_prompts_with_large_scores_and_ranges(dtype):
    batch, heads, dim, queries, n = 40, 8, 128, 40, 160
    for size in (2.0**30, 2.0**-30) if dtype == BF else (2.0**5, 2.0**-9):
        cache, table, _ = _filled(batch, n, heads, dim, 32, dtype, seed=8)
        grow = torch.exp2(torch.randint(-6, 6, cache.range.shape, generator=_gen(1), device="cuda").float())
        cache.range.mul_(grow)
        cache.range[..., 0] *= size
        cache.range[table[:, 1].long(), :, 1] = 0.0
        values = _values_of_codes(cache, table, n)
        q = (_randn(batch, queries, heads * 4, dim, seed=6, dtype=torch.float32, size=0.3) / (size if dtype == BF or size < 1 else 1)).to(dtype)
        q[..., 5] *= 64
        q[3, 7] = 0
        _check_attention(q, cache, table, torch.full((batch,), n, dtype=torch.int32, device="cuda"), values)


@pytest.mark.parametrize("queries, share", [(1, 4), (3, 8), (150, 2)])
def test_long_context_and_wide_table(queries, share):
    cache, table, values = _filled(2, 20000, 1, 128, 64, BF, seed=3)
    q = _randn(2, queries, share, 128, seed=4)
    wide = torch.full((2, 3 * table.shape[1]), 2**31 - 1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    for lengths in (_lengths(20000, 12345), _lengths(700, 19999)):
        _check_attention(q, cache, wide, lengths, values)
        _check_attention(q, cache, wide[:, : table.shape[1]], lengths, values, window=3000)


@pytest.mark.parametrize("queries", [1, 40])
def test_what_is_not_seen_may_be_anything(queries):
    heads, dim, page = 2, 64, 16
    cache, table, values = _filled(2, 160, heads, dim, page, BF, seed=5)
    q = _randn(2, queries, heads * 2, dim, seed=6)
    lengths = _lengths(150, 90)
    want = qr.kv8_attention(q, cache, table, lengths, window=30)
    # pages behind the window or past the length: not finite, gone from the table, or wild
    gone = table.clone()
    for b, n in enumerate((150, 90)):
        first = max(0, n - queries + 1 - 30) // page
        keep = torch.zeros(table.shape[1], dtype=torch.bool, device="cuda")
        keep[first : -(-n // page)] = True
        cache.range[table[b][~keep].long()] = float("nan")
        cache.data[table[b][~keep].long()] = 255
        gone[b][~keep] = 2**31 - 1
    assert torch.equal(qr.kv8_attention(q, cache, table, lengths, window=30), want)
    assert torch.equal(qr.kv8_attention(q, cache, gone, lengths, window=30), want)
    torch.cuda.synchronize()
    qr.kv8_read(cache, torch.zeros(1, dtype=torch.int64, device="cuda"))  # nothing was reported


@pytest.mark.parametrize("queries", [1, 60])
def test_a_page_that_is_not_finite_shows_where_it_is_seen(queries):
    cache, table, values = _filled(1, 128, 1, 64, 16, BF, seed=5)
    q = _randn(1, queries, 2, 64, seed=6)
    lengths = _lengths(128)
    want = qr.kv8_attention(q, cache, table, lengths)
    for part in (0, 1):
        spoiled = copy.deepcopy(cache)
        spoiled.range[table[0, 5].long(), :, part] = float("nan")  # tokens 80 to 95
        got = qr.kv8_attention(q, spoiled, table, lengths)
        pos = 128 - queries + torch.arange(queries, device="cuda")
        assert got[0, pos >= 80].isnan().all() and torch.equal(got[0, pos < 80], want[0, pos < 80])


@pytest.mark.parametrize("queries", [1, 50])
def test_large_scores_and_ranges(queries):
    for dtype, size in ((BF, 2.0**40), (BF, 2.0**-40), (HF, 2.0**6), (HF, 2.0**-10), (BF, 30.0)):
        cache, table, _ = _filled(1, 200, 1, 64, 32, dtype, seed=8)
        cache.range[..., 0] *= size
        cache.range[..., 1] /= size if dtype == BF else 1
        values = _values_of_codes(cache, table, 200)
        for up in (1.0, 20.0):
            q = _randn(1, queries, 2, 64, seed=6, dtype=torch.float32, size=up)
            q = (q / size).to(dtype) if dtype == BF or size < 1 else q.to(dtype)
            _check_attention(q, cache, table, _lengths(200), values)


def _values_of_codes(cache, table, n):
    """From a copy whose ranges are 127, so that what it reads are codes."""
    plain = copy.deepcopy(cache)
    plain.range.fill_(127.0)
    at = torch.arange(n, device="cuda")
    slots = table.long()[:, at // cache.page_size] * cache.page_size + at % cache.page_size
    return [x.double().unflatten(0, slots.shape) * cache.range[..., part].double()[slots // cache.page_size].unsqueeze(-1) / 127
            for part, x in enumerate(qr.kv8_read(plain, slots.reshape(-1)))]


@pytest.mark.parametrize("queries", [1, 50])
def test_pages_of_very_different_ranges(queries):
    cache, table, _ = _filled(1, 320, 2, 128, 16, BF, seed=8)
    grow = torch.exp2(torch.randint(-12, 12, cache.range.shape, generator=_gen(1), device="cuda").float())
    cache.range.mul_(grow)
    cache.range[table[0, 3].long(), 0] = 0.0
    values = _values_of_codes(cache, table, 320)
    q = _randn(1, queries, 4, 128, seed=6, size=2.0**-6)
    _check_attention(q, cache, table, _lengths(320), values)


def test_queries_with_a_large_channel():
    cache, table, values = _filled(1, 300, 1, 128, 64, HF, seed=2)
    for queries in (1, 40):
        q = _randn(1, queries, 4, 128, seed=3, dtype=HF, size=0.1)
        q[..., 7] *= 256
        _check_attention(q, cache, table, _lengths(300), values)


@pytest.mark.parametrize("queries", [1, 20])
def test_wrong_pages_and_lengths_are_reported(queries):
    cache, table, values = _filled(2, 64, 1, 64, 16, BF)
    q = _randn(2, queries, 1, 64)
    for t, n in ((table.clone().fill_(10**6), _lengths(64, 64)), (table.clone().fill_(-1), _lengths(64, 64)), (table, _lengths(64, 65)), (table, _lengths(-1, 3))):
        out = qr.kv8_attention(q, cache, t, n)
        torch.cuda.synchronize()
        with pytest.raises(QRB200Error):
            qr.kv8_attention(q, cache, table, _lengths(64, 64))
        assert out.isfinite().all()
    _check_attention(q, cache, table, _lengths(64, 64), values)


def test_strides_of_queries_table_and_lengths():
    cache, table, values = _filled(3, 200, 2, 64, 16, BF)
    base = _randn(3, 30, 7, 67, seed=1)
    lengths = torch.tensor([[200, 5], [100, 7], [33, 9]], dtype=torch.int32, device="cuda")[:, 0]
    wide = torch.stack([table, table + 1], -1)[..., 0]
    for queries in (1, 2, 30):
        q = base[:, :queries, 1:5, 1:65]
        want = _check_attention(q.contiguous(), cache, table, lengths.contiguous(), values)
        assert torch.equal(qr.kv8_attention(q, cache, wide, lengths), want)
        swapped = q.contiguous().transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(qr.kv8_attention(swapped, cache, table, lengths), want)
        channels = q.contiguous().transpose(1, 3).contiguous().transpose(1, 3)
        assert torch.equal(qr.kv8_attention(channels, cache, table, lengths), want)


def test_empty_calls():
    cache, table, _ = _filled(2, 32, 1, 64, 16, BF)
    lengths = _lengths(3, 3)
    for q in (_randn(2, 0, 2, 64), _randn(2, 1, 0, 64)):
        assert qr.kv8_attention(q, cache, table, lengths).shape == q.shape
    assert qr.kv8_attention(_randn(0, 1, 2, 64), cache, table[:0], lengths[:0]).shape == (0, 1, 2, 64)
    for queries in (1, 40):
        out = qr.kv8_attention(_randn(2, queries, 2, 64), cache, table[:, :0], _lengths(0, 0))
        assert torch.all(out == 0)
        none = qr.kv8_cache(0, 16, 1, 64)
        assert torch.all(qr.kv8_attention(_randn(2, queries, 2, 64), none, table, _lengths(0, 0)) == 0)


def test_a_batch_past_one_launch_grid():
    batch = 65540  # a launch's third dimension holds 65535
    cache, table, values = _filled(5, 16, 1, 64, 16, BF)
    pick = torch.arange(batch, device="cuda") % 5
    lengths = (torch.arange(batch, device="cuda") % 17).int()
    q = _randn(batch, 1, 1, 64)
    out = qr.kv8_attention(q, cache, table[pick].contiguous(), lengths)
    at = torch.cat([torch.arange(40, device="cuda"), torch.arange(batch - 40, batch, device="cuda")])
    part = _check_attention(q[at].contiguous(), cache, table[pick[at]].contiguous(), lengths[at], [x[pick[at]] for x in values])
    assert torch.equal(out[at], part)


@pytest.mark.parametrize("queries", [1, 30])
def test_windows_up_to_the_largest(queries):
    cache, table, values = _filled(2, 64, 2, 64, 16, BF)
    q, lengths = _randn(2, queries, 4, 64), _lengths(64, 5)
    whole = _check_attention(q, cache, table, lengths, values)
    for window in (63, 64, 65, 64 + queries, 2**31 - 2, 2**31 - 1):
        assert torch.equal(_check_attention(q, cache, table, lengths, values, window=window), whole) or window == 63


def test_offsets_past_two_gibibytes():
    pages, page, dim = 70000, 128, 128  # 2.3 GB of codes
    cache = qr.kv8_cache(pages, page, 1, dim)
    table = torch.tensor([[pages - 1, 69999 - 3, 5]], dtype=torch.int32, device="cuda")
    slots = (table.long()[0][:, None] * page + torch.arange(page, device="cuda")).reshape(-1)
    k, v = _randn(384, 1, dim, seed=1), _randn(384, 1, dim, seed=2)
    qr.kv8_write(cache, k, v, slots)
    values = _values(cache, slots[None])
    assert (values[0][0] - k.double()).abs().max() <= cache.range[table[0].long(), 0, 0].max() / 250
    for queries in (1, 100):
        _check_attention(_randn(1, queries, 2, dim, seed=3), cache, table, _lengths(384), values)


@pytest.mark.parametrize("queries, tokens", [(1, 4), (3, 12), (40, 160)])
def test_write_and_attend_in_a_graph_and_on_another_stream(queries, tokens):
    batch, heads, dim, page = 4, 2, 64, 16
    table = torch.randperm(batch * 8, generator=_gen(1), device="cuda").reshape(batch, 8).int()

    def inputs(seed):
        n = torch.full((batch,), 60 + seed, dtype=torch.int32, device="cuda")
        at = n.long()[:, None] - queries + torch.arange(queries, device="cuda")
        slots = (table.long().gather(1, at // page) * page + at % page).reshape(-1)
        return [_randn(batch, queries, heads * 2, dim, seed=seed), _randn(tokens, heads, dim, seed=seed + 10), _randn(tokens, heads, dim, seed=seed + 20), slots, n]

    def fill(cache):
        at = torch.arange(128, device="cuda")
        slots = (table.long()[:, at // page] * page + at % page).reshape(-1)
        qr.kv8_write(cache, _randn(batch * 128, heads, dim, seed=5), _randn(batch * 128, heads, dim, seed=6), slots)

    def step(cache, q, k, v, slots, n):
        qr.kv8_write(cache, k, v, slots)
        return qr.kv8_attention(q, cache, table, n), qr.kv8_read(cache, slots)[0]

    cache = qr.kv8_cache(batch * 8, page, heads, dim)
    want = []
    for seed in (1, 2):
        fill(cache)
        want.append([x.clone() for x in step(cache, *inputs(seed))])
    hold = inputs(1)
    fill(cache)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(cache, *hold)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, *hold)
    for seed in (2, 1, 2):
        for a, b in zip(hold, inputs(seed)):
            a.copy_(b)
        fill(cache)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[seed - 1]))


def test_repeated_calls_agree():
    cache, table, _ = _filled(3, 3000, 2, 128, 64, BF)
    for queries in (1, 4, 200):
        q = _randn(3, queries, 8, 128)
        out = qr.kv8_attention(q, cache, table, _lengths(3000, 1777, 2048))
        for _ in range(5):
            assert torch.equal(qr.kv8_attention(q, cache, table, _lengths(3000, 1777, 2048)), out)


def test_calls_at_the_same_time():
    # writes by lists of pages, attention through memory, of prompts and of single tokens, and products, each on its own
    # stream and at once, eager and from two graphs
    heads, dim, page = 2, 128, 64
    cache, table, _ = _filled(2, 8192, heads, dim, page, BF)
    one, many = _randn(1, 1, 8, dim), _randn(2, 300, 8, dim, seed=1)
    x, sx = qr.quantize_fp8(_randn(700, 512, seed=2))
    w, sw = qr.quantize_fp8(_randn(1024, 512, seed=3), tile_rows=128)
    k = _randn(1500, heads, dim, seed=4)
    order = [torch.randperm(64 * page, generator=_gen(i), device="cuda")[:1500] for i in range(2)]
    own = [qr.kv8_cache(64, page, heads, dim) for _ in range(2)]

    def write(i):
        qr.kv8_write(own[i], k, k, order[i])
        return qr.kv8_read(own[i], order[i])[0]

    calls = [lambda: write(0), lambda: write(1), lambda: qr.kv8_attention(one, cache, table[:1], _lengths_of),
             lambda: qr.kv8_attention(many, cache, table, _lengths_two), lambda: qr.fp8_linear(x, sx, w, sw), lambda: qr.fp8_linear(x[:40], sx[:40], w, sw)]
    _lengths_of, _lengths_two = _lengths(8192), _lengths(5000, 8192)
    want = [f().clone() for f in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for f, s in zip(calls, streams):
            with torch.cuda.stream(s):
                got.append([f() for _ in range(4)])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for out, b in zip(got, want) for a in out)
    graphs, outs = [], []
    for part in (0, 1):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append([f() for f in calls[part::2]])
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for part in (0, 1) for a, b in zip(outs[part], want[part::2]))
