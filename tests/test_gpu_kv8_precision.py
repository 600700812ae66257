"""How exact attention over the 8-bit cache is, against 64 bits: the weights' bits, long sums, and that a row depends on what it sees only (GPU).

Each bound is relative to `size`, the sum of |weight x value| of a row and channel: by that much may 32-bit arithmetic be off, and
no more. It holds for prompts and single tokens, and for both types, alike.
"""

import math

import pytest
import torch

import qr_v2_b200_kernel_b200 as qr

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed=0, dtype=BF, size=1.0):
    return (torch.randn(*shape, generator=_gen(seed), device="cuda") * size).to(dtype)


def _pages(batch, tokens, heads, dim, page, dtype, seed=0):
    """An empty cache, the table of its sequences and their slots (batch, tokens)."""
    per = -(-tokens // page)
    table = torch.randperm(batch * per + 1, generator=_gen(seed), device="cuda")[: batch * per].reshape(batch, per).int()
    cache = qr.kv8_cache(batch * per + 1, page, heads, dim, dtype=dtype)
    at = torch.arange(tokens, device="cuda")
    return cache, table, table.long()[:, at // page] * page + at % page


def _write(cache, slots, k, v):
    qr.kv8_write(cache, k.flatten(0, 1).to(cache.dtype), v.flatten(0, 1).to(cache.dtype), slots.reshape(-1))


def _values(cache, slots):
    """What the cache stands for at slots (tokens,), in 64 bits, and the steps of its values (tokens, heads)."""
    plain = qr.KV8Cache(cache.data, torch.full_like(cache.range, 127.0), cache.page_size, cache.head_dim, cache.dtype)
    step = cache.range.double()[slots // cache.page_size] / 127
    k, v = (x.double() * step[:, :, i, None] for i, x in enumerate(qr.kv8_read(plain, slots)))
    return k, v, step[..., 1]


def _check(out, q, cache, slots, lengths, terms, window=None, rows=None, scale=None, causal=True):
    """Of `terms` products of a score that are not zero, each is exact; their sum, and what scales it, is off by terms + 4 units of
    2^-23 of their magnitudes, and a weight by twice that (its own score's and the largest one's). A weight is held in 22 bits (half a
    unit: 2^-23) with an exponential of two units of 2^-23 and a scaling: 2^-20. Sums: up to 256 products, 128 for
    fp16, join a sum of the matrix instruction's before it is added to others in 32 bits, each cut off by up to a unit, 2^-23, of the sum so far: 2^-15 or
    2^-16, and 2^-20 for the rest.

    And weights times their steps are put, in fp16 pairs, within 2^24 / 2^10 of fp16's smallest by the largest of the row: 2^-25 2^-10 each of the
    largest weight times range; n of them, and a factor of two for the power of two above: n 2^-34 (127 w <= R).
    """
    batch, queries, heads, dim = q.shape
    share = heads // cache.kv_heads
    factor = dim**-0.5 if scale is None else scale
    for b in range(batch):
        n = int(lengths[b])
        if n == 0:
            continue
        k, v, step = _values(cache, slots[b, :n])
        k, v = (x.repeat_interleave(share, 1) for x in (k, v))
        reach = 127 * step.repeat_interleave(share, 1)  # tokens, heads
        at = torch.arange(n, device="cuda")
        for i in range(queries) if rows is None else rows:
            i = i % queries
            pos = n - queries + i
            seen = (at <= pos) if causal else torch.ones(n, dtype=torch.bool, device="cuda")
            if window:
                seen = seen & (at > pos - window)
            if not seen.any():
                assert torch.all(out[b, i] == 0)
                continue
            k_, v_, r_, qi = k[seen], v[seen], reach[seen], q[b, i].double()
            p = torch.softmax(torch.einsum("hd,thd->ht", qi, k_) * factor, -1)
            d = (torch.einsum("hd,thd->ht", qi.abs(), k_.abs()) * factor).amax(-1) * (terms + 4) * 2.0**-23
            want = torch.einsum("ht,thd->hd", p, v_)
            size = torch.einsum("ht,thd->hd", p, v_.abs())
            bound = torch.finfo(q.dtype).eps / 2 * want.abs() + ((2 * d).expm1()[:, None] + 2.0**-20 + (2.0**-16 if q.dtype == HF else 2.0**-15) + 2.0**-20) * size
            bound += len(p[0]) * 2.0**-34 * (p.T * r_).amax(0)[:, None] + (2.0**-24 if q.dtype == HF else 0.0)
            err = (out[b, i].double() - want).abs()
            assert torch.all(err <= bound), (b, i, (err / bound).max().item())


def _few_channels(batch, queries, heads, dim, dtype, size, channels=4, seed=9):
    """Queries of few channels that are not zero: their scores are sums of as many products."""
    q = _randn(batch, queries, heads, dim, seed=seed, dtype=dtype, size=size)
    q[..., channels:] = 0
    return q


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, heads, share, queries", [(40, 8, 4, 40), (2, 2, 8, 5), (2, 2, 8, 1), (1, 1, 1, 1)])
def test_weights_are_held_in_22_bits(batch, heads, share, queries, dim, dtype):
    # Values come in pairs of opposite ones under nearly the same weights: what is left of a pair is the weights' error, and no
    # rounding of the result hides it. (Held in 11 bits the larger of two weights is off by up to 2^-12.)
    n = 200
    cache, table, slots = _pages(batch, n, heads, dim, 16, dtype)
    k = torch.randn(batch, n // 2, heads, dim, generator=_gen(1), device="cuda").repeat_interleave(2, 1)
    v = torch.randn(batch, n // 2, heads, dim, generator=_gen(2), device="cuda").repeat_interleave(2, 1)
    k[:, 1::2, :, 1] += 0.02
    v[:, 1::2] *= -1
    _write(cache, slots, k, v)
    q = _few_channels(batch, queries, heads * share, dim, dtype, 1.5 * dim**0.5)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out = qr.kv8_attention(q, cache, table, lengths)
    _check(out[:2], q[:2], cache, slots, lengths, 4)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim, queries, share, n, window", [(128, 2048, 8, 32768, None), (64, 1024, 8, 40000, None), (128, 1024, 8, 20000, 16000), (128, 1, 8, 32768, None),
                                                            (64, 5, 4, 40000, None)])
def test_long_sums_keep_32_bits(dim, queries, share, n, window, dtype):
    # Positive values under nearly even weights: whatever a sum cuts off, it cuts off in one direction.
    heads = 2
    cache, table, slots = _pages(1, n, heads, dim, 64, dtype)
    k = 0.05 * torch.randn(1, n, heads, dim, generator=_gen(1), device="cuda")
    v = 0.5 + torch.rand(1, n, heads, dim, generator=_gen(2), device="cuda")
    _write(cache, slots, k, v)
    q = _few_channels(1, queries, heads * share, dim, dtype, 1.0)
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = qr.kv8_attention(q, cache, table, lengths, window=window)
    _check(out, q, cache, slots, lengths, 4, window=window, rows=[0, 1, 300, -2, -1])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_sums_under_rising_scores(dim, dtype):
    # The largest score keeps growing, so what has been summed, and what was set aside, keeps being scaled down.
    heads, share, queries, n = 2, 8, 1024, 6000
    cache, table, slots = _pages(1, n, heads, dim, 64, dtype)
    k = 0.05 * torch.randn(1, n, heads, dim, generator=_gen(1), device="cuda")
    k[..., 0] = torch.linspace(0, 4, n, device="cuda")[None, :, None]
    v = 0.5 + torch.rand(1, n, heads, dim, generator=_gen(2), device="cuda")
    _write(cache, slots, k, v)
    q = _few_channels(1, queries, heads * share, dim, dtype, 1.0)
    q[..., 0] = torch.linspace(1, 8, heads * share, device="cuda") * dim**0.5 / 4
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    _check(qr.kv8_attention(q, cache, table, lengths), q, cache, slots, lengths, 4, rows=[0, 1, 300, -2, -1])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, heads, share, queries, n, window", [
    (40, 8, 4, 40, 200, None), (40, 8, 4, 40, 200, 60), (2, 2, 8, 12, 200, None), (2, 2, 8, 12, 200, 78), (2, 3, 1, 8, 197, None), (2, 3, 1, 8, 197, 79)])
def test_large_values_that_a_row_does_not_see(batch, heads, share, queries, n, window, dim, dtype):
    # the last page's values reach far beyond the others'; so do, with a window, those of a page that only the first queries see
    page = 16
    cache, table, slots = _pages(batch, n, heads, dim, page, dtype)
    _write(cache, slots, _randn(batch, n, heads, dim, seed=1), _randn(batch, n, heads, dim, seed=2))
    cache.range[..., 1] *= 2.0**-16
    q = _few_channels(batch, queries, heads * share, dim, dtype, 1.5 * dim**0.5)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    pos = n - queries + torch.arange(queries, device="cuda")
    blind = pos < 192  # pages 12 (tokens 192 on) and, with a window, 6 (tokens 96 to 111)
    pages = [12]
    if window:
        blind &= pos - window >= 111
        pages.append(6)
    assert blind.any() and not blind.all()
    want = qr.kv8_attention(q, cache, table, lengths, window=window)
    for up in (2.0**26, 2.0**29 if dtype == HF else 2.0**40):  # within fp16's range
        grown = qr.KV8Cache(cache.data, cache.range.clone(), page, dim, dtype)
        grown.range[table[:, pages].long(), :, 1] *= up
        out = qr.kv8_attention(q, grown, table, lengths, window=window)
        assert torch.equal(out[:, blind], want[:, blind]) and not torch.equal(out[:, ~blind], want[:, ~blind])
        _check(out[:1], q[:1], grown, slots, lengths, 4, window=window)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, heads, share, queries", [(40, 8, 4, 40), (2, 2, 8, 5), (2, 2, 8, 1), (1, 1, 1, 1)])
def test_large_values_without_weight(batch, heads, share, queries, dim, dtype):
    # pages of values 2^50 times the others', whose scores leave them a weight of about 2^-90
    n, page = 200, 16
    cache, table, slots = _pages(batch, n, heads, dim, page, dtype)
    k = torch.randn(batch, n, heads, dim, generator=_gen(1), device="cuda")
    k[..., 0] = 0
    k[:, 16:32, :, 0] = -8
    k[:, 192:, :, 0] = -8
    _write(cache, slots, k, _randn(batch, n, heads, dim, seed=2))
    cache.range[..., 1] *= 2.0**-20
    cache.range[table[:, [1, 12]].long(), :, 1] *= 2.0**50
    q = _few_channels(batch, queries, heads * share, dim, dtype, 0.5 * dim**0.5)
    q[..., 0] = 8 * dim**0.5
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out = qr.kv8_attention(q, cache, table, lengths)
    assert out.float().abs().amax() < 2.0**-14
    _check(out[:2], q[:2], cache, slots, lengths, 4)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, heads, share, queries", [(40, 8, 4, 40), (2, 2, 8, 12)])
def test_large_keys_that_a_row_does_not_see(batch, heads, share, queries, dim):
    # queries near 2^60 over keys near 2^-60, the last page's keys near 2^100 (of bf16's range)
    n, page = 200, 16
    cache, table, slots = _pages(batch, n, heads, dim, page, BF)
    _write(cache, slots, _randn(batch, n, heads, dim, seed=1), _randn(batch, n, heads, dim, seed=2))
    cache.range[..., 0] *= 2.0**-60
    q = _few_channels(batch, queries, heads * share, dim, BF, 1.5 * dim**0.5 * 2.0**60)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    want = qr.kv8_attention(q, cache, table, lengths)
    _check(want[:1], q[:1], cache, slots, lengths, 4)
    blind = n - queries + torch.arange(queries, device="cuda") < 192
    cache.range[table[:, 12].long(), :, 0] *= 2.0**160
    assert torch.equal(qr.kv8_attention(q, cache, table, lengths)[:, blind], want[:, blind])


@pytest.mark.parametrize("batch, heads, share, queries", [(40, 8, 4, 40), (2, 2, 8, 12), (1, 1, 1, 1)])
def test_scores_of_nothing_under_a_factor_beyond_32_bits(batch, heads, share, queries):
    # keys of zeros in pages whose range, with queries near 2^60, leaves 32 bits: their scores are 0
    n, page, dim = 200, 16, 128
    cache, table, slots = _pages(batch, n, heads, dim, page, BF)
    k = torch.zeros(batch, n, heads, dim, device="cuda")
    k[..., 10] = 1
    _write(cache, slots, k, _randn(batch, n, heads, dim, seed=2))
    cache.range[..., 0] *= 2.0**100
    q = _few_channels(batch, queries, heads * share, dim, BF, 2.0**60)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    _check(qr.kv8_attention(q, cache, table, lengths)[:2], q[:2], cache, slots, lengths, 0)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, heads, share, queries, n", [(40, 8, 4, 40, 200), (2, 2, 8, 12, 200), (1, 1, 1, 1, 200), (1, 1, 4, 1, 8192), (1, 2, 2, 1, 70000)])
@pytest.mark.parametrize("size", [2.0**126, 2.0**-100])
def test_values_near_the_largest_and_the_smallest(size, batch, heads, share, queries, n, dim):
    # of one sign under even weights: their unnormalised sum is beyond 32 bits' range, their mean is not
    cache, table, slots = _pages(batch, n, heads, dim, 16, BF)
    k = 0.05 * torch.randn(batch, n, heads, dim, generator=_gen(1), device="cuda")
    _write(cache, slots, k, 0.5 + 0.5 * torch.rand(batch, n, heads, dim, generator=_gen(2), device="cuda"))
    cache.range[..., 1] *= size
    q = _few_channels(batch, queries, heads * share, dim, BF, 1.0)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out = qr.kv8_attention(q, cache, table, lengths)
    assert out.isfinite().all()
    _check(out[:2], q[:2], cache, slots, lengths, 4)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, heads, share, queries", [(40, 8, 4, 40), (2, 2, 8, 12), (1, 1, 1, 1)])
@pytest.mark.parametrize("power", [10, 24, 27, 40])
def test_scores_next_to_which_a_values_step_is_lost(power, batch, heads, share, queries, dim, dtype):
    # every 29th token's score is near 2^power, the others' are 0; values reach 2^12, steps are near 2^5, and later pages' larger still
    n, page = 200, 16
    cache, table, slots = _pages(batch, n, heads, dim, page, dtype)
    k = torch.zeros(batch, n, heads, dim, device="cuda")
    k[:, ::29, :, 0] = 1
    v = torch.randn(batch, n, heads, dim, generator=_gen(1), device="cuda") * torch.linspace(3, 2000, n, device="cuda")[None, :, None, None]
    _write(cache, slots, k, v)
    q = torch.zeros(batch, queries, heads * share, dim, device="cuda")
    q[..., 0] = 8
    q = q.to(dtype)
    cache.range[..., 0] *= 2.0 ** (power - 3)  # a score is 8 / 8 of a key's entry, by the scale
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out = qr.kv8_attention(q, cache, table, lengths, scale=1.0)
    assert out.isfinite().all()
    if power == 10:
        return
    for b in range(min(batch, 2)):  # the same score for each of the tokens, and nothing for the others
        _, values, _ = _values(cache, slots[b])
        for i in range(queries):
            at = values[: n - queries + i + 1 : 29].repeat_interleave(share, 1)
            want, size = at.mean(0), at.abs().mean(0)
            assert torch.all((out[b, i].double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 2.0**-15 * size)
