"""Cases for the operators on 8-bit floating point and the 8-bit key/value cache: quantisation with a
scale for each block of 128, the product of such operands, the write and read-back of a cache whose
pages have a range for each head, and attention over that cache.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, where
``own`` is true, through the package's public entry points. ``exact`` restates each operator in
64 bits from its definition.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 128  # codes that share a scale
PAGE = 64  # tokens of a page, which share a head's range
TINY = 2.0**-100  # what is smaller throughout is held as zeros


def listed():
    return [
        # One sequence's next token before a projection: a single row, where the launch is the cost.
        {"name": "quantise one token", "op": "quantise", "rows": 1, "cols": 4096, "tile": 1, "dtype": "bf16"},
        # A master weight that does not fill its last blocks, into blocks of 128 x 128.
        {"name": "quantise ragged weights", "op": "quantise", "rows": 5000, "cols": 2040, "tile": 128, "dtype": "fp32"},
        # The activations of a full prefill batch.
        {"name": "quantise prefill", "op": "quantise", "rows": 16384, "cols": 4096, "tile": 1, "dtype": "bf16"},
        # Serving one token: the weights are read once for a single row.
        {"name": "linear one token", "op": "linear", "rows": 1, "outs": 4096, "depth": 4096, "dtype": "bf16", "bias": False},
        # A ragged batch with a bias, channels that do not fill the last tile and a depth that does not fill the last block.
        {"name": "linear ragged batch", "op": "linear", "rows": 333, "outs": 1000, "depth": 2000, "dtype": "fp16", "bias": True},
        # Prefill of a wide layer: the largest product.
        {"name": "linear prefill", "op": "linear", "rows": 8192, "outs": 8192, "depth": 4096, "dtype": "bf16", "bias": False},
        # One decode step of a batch: a token for each of 16 sequences, each in a page that already holds some.
        {"name": "cache decode step", "op": "cache", "batch": 16, "new": 1, "start": 1000, "heads": 8, "dim": 128, "dtype": "bf16"},
        # The next chunk of a long prompt batch, which begins inside a page.
        {"name": "cache prompt chunk", "op": "cache", "batch": 8, "new": 4096, "start": 13, "heads": 8, "dim": 128, "dtype": "bf16"},
        # One sequence's next token over a short context.
        {"name": "attention one token", "op": "attention", "batch": 1, "length": 513, "queries": 1, "heads": 8, "share": 4, "dim": 128,
         "window": 0, "ragged": False, "dtype": "bf16"},
        # Verifying five drafted tokens for a ragged batch that has an empty slot, with a sliding window.
        {"name": "attention drafted tokens", "op": "attention", "batch": 12, "length": 2047, "queries": 5, "heads": 4, "share": 3, "dim": 64,
         "window": 1000, "ragged": True, "dtype": "fp16"},
        # A full serving batch over long contexts: the whole cache is read for one token of each sequence.
        {"name": "attention serving batch", "op": "attention", "batch": 64, "length": 8192, "queries": 1, "heads": 8, "share": 8, "dim": 128,
         "window": 0, "ragged": False, "dtype": "bf16"},
        # The second half of two prompts over the first, already in the cache.
        {"name": "attention prompt chunk", "op": "attention", "batch": 2, "length": 4096, "queries": 2048, "heads": 4, "share": 4, "dim": 128,
         "window": 0, "ragged": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantise", "linear", "cache", "attention", "attention"])
    if op == "quantise":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return {"op": op, "rows": _log(rng, 1, 8192 if dtype == "fp32" else 16384), "cols": rng.choice([_log(rng, 64, 4096), 8 * _log(rng, 8, 512)]),
                "tile": rng.choice([1, 1, 128]), "dtype": dtype}
    if op == "linear":
        return {"op": op, "rows": _log(rng, 1, 6000), "outs": rng.choice([_log(rng, 64, 8192), 128 * _log(rng, 1, 64)]),
                "depth": rng.choice([_log(rng, 64, 4096), 64 * _log(rng, 2, 64)]), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "bias": rng.random() < 0.5}
    dim = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "cache":
        return {"op": op, "batch": _log(rng, 1, 6), "new": _log(rng, 1, 4096), "start": rng.randrange(0, 200), "heads": rng.choice([1, 2, 4, 8]),
                "dim": dim, "dtype": dtype}
    if rng.random() < 0.3:  # a prompt, or a chunk of one
        queries = _log(rng, 17, 2048)
        return {"op": op, "batch": rng.randrange(1, 3), "length": _log(rng, queries, 4096), "queries": queries, "heads": rng.choice([1, 2, 4]),
                "share": rng.randrange(1, 5), "dim": dim, "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "ragged": rng.random() < 0.6,
                "dtype": dtype}
    queries = rng.choice([1, 1, _log(rng, 2, 16)])
    return {"op": op, "batch": _log(rng, 1, 48 if queries == 1 else 8), "length": _log(rng, queries, 8192), "queries": queries, "heads": rng.choice([1, 2, 4, 8]),
            "share": rng.randrange(1, 9 if queries == 1 else 5), "dim": dim,
            "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "ragged": rng.random() < 0.6, "dtype": dtype}


def _lengths(case):
    """Tokens in the cache for each sequence: all full, or falling off to an empty slot in a ragged batch."""
    b, n = case["batch"], case["length"]
    if not case["ragged"]:
        return [n] * b
    return [0 if b >= 4 and i == b - 1 else max(min(n, case["queries"]), n - n * 7 * i // (8 * b)) for i in range(b)]


def _visible(case):
    """(token, query) pairs that each head sees, and the cached tokens that are read at all."""
    pairs = tokens = 0
    for n in _lengths(case):
        first = n
        for i in range(case["queries"]):
            position = n - case["queries"] + i
            if position >= 0:
                lo = max(0, position - case["window"] + 1) if case["window"] else 0
                pairs += position + 1 - lo
                first = min(first, lo)
        tokens += n - first
    return pairs, tokens


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    op, s = case["op"], BYTES[case["dtype"]]
    if op == "quantise":  # x in; the values that the codes stand for and the scales out
        n = case["rows"] * case["cols"]
        scales = -(-case["rows"] // case["tile"]) * _blocks(case["cols"])
        return {"bytes": 2 * s * n + 4 * scales, "flops": 6 * n}
    if op == "linear":
        m, n, k = case["rows"], case["outs"], case["depth"]
        scales = m * _blocks(k) + _blocks(n) * _blocks(k)
        return {"bytes": m * k + n * k + s * m * n + 4 * scales + (s * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "cache":  # new keys and values in, the cache's bytes of them, and the values of the pages written out
        new = case["batch"] * case["new"] * case["heads"] * case["dim"]
        read = case["batch"] * (case["new"] + case["start"] % PAGE) * case["heads"] * case["dim"]
        return {"bytes": 2 * new * (s + 1) + 2 * read * s + 8 * case["batch"] * case["new"], "flops": 8 * new}
    pairs, tokens = _visible(case)
    rows = case["batch"] * case["queries"] * case["heads"] * case["share"]
    return {"bytes": 2 * tokens * case["heads"] * case["dim"] + 2 * s * rows * case["dim"], "flops": 4 * pairs * case["heads"] * case["share"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pages(gen, batch, per_seq):
    """A block table whose pages are scattered over the pool, and the pool's size."""
    pool = batch * per_seq + 3
    table = torch.randperm(pool, generator=gen, device="cuda")[: batch * per_seq].reshape(batch, per_seq)
    return table.to(torch.int32).contiguous(), pool


def _keys_values(gen, tokens, heads, dim, dtype):
    """Keys whose channels differ in size and centre, as keys do, and plainer values; tokens differ in size."""
    size = torch.exp(0.3 * torch.randn(heads, dim, generator=gen, device="cuda"))
    centre = 0.5 * torch.randn(heads, dim, generator=gen, device="cuda")
    token = torch.exp(0.1 * torch.randn(tokens, heads, 1, generator=gen, device="cuda"))
    k = torch.randn(tokens, heads, dim, generator=gen, device="cuda") * size + centre
    v = torch.randn(tokens, heads, dim, generator=gen, device="cuda") * token
    return k.to(dtype), v.to(dtype)


def _matrix(gen, rows, cols, dtype):
    """Rows whose channels differ in size."""
    size = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
    return (torch.randn(rows, cols, generator=gen, device="cuda") * size).to(dtype)


def _cache_inputs(case, gen, dtype):
    b, end = case["batch"], case["start"] + case["new"]
    table, pool = _pages(gen, b, -(-end // PAGE))
    at = torch.arange(end, device="cuda")
    slots = table.long()[:, at // PAGE] * PAGE + at % PAGE  # batch, tokens
    k, v = (x.unflatten(0, (b, end)) for x in _keys_values(gen, b * end, case["heads"], case["dim"], dtype))
    return pool, slots, k, v


def _sequences(case, gen, dtype):
    """Keys and values of one sequence after the other."""
    for _ in range(case["batch"]):
        yield _keys_values(gen, case["length"], case["heads"], case["dim"], dtype)


def prepare(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": dict(case), "dtype": dtype}
    if case["op"] == "quantise":
        s["x"] = _matrix(gen, case["rows"], case["cols"], dtype)
    elif case["op"] == "linear":
        m, n, k = case["rows"], case["outs"], case["depth"]
        s["x"], s["x_scale"] = _to_fp8(_matrix(gen, m, k, torch.float32), 1)
        s["w"], s["w_scale"] = _to_fp8(torch.randn(n, k, generator=gen, device="cuda") * k**-0.5, BLOCK)
        s["bias"] = torch.randn(n, generator=gen, device="cuda").to(dtype) if case["bias"] else None
    elif case["op"] == "cache":
        pool, slots, k, v = _cache_inputs(case, gen, dtype)
        first = case["start"]
        s["cache"] = _cache(case, pool, dtype)
        if first:  # the tokens that came before
            _write(s["cache"], k[:, :first].flatten(0, 1), v[:, :first].flatten(0, 1), slots[:, :first].reshape(-1))
        s["k"], s["v"] = k[:, first:].flatten(0, 1).contiguous(), v[:, first:].flatten(0, 1).contiguous()
        s["slots"] = slots[:, first:].reshape(-1).contiguous()
        s["read"] = slots[:, first // PAGE * PAGE :].reshape(-1).contiguous()  # all of the pages written
    else:
        b, n, h, d = case["batch"], case["length"], case["heads"], case["dim"]
        s["table"], pool = _pages(gen, b, -(-n // PAGE))
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        s["q"] = torch.randn(b, case["queries"], h * case["share"], d, generator=gen, device="cuda").to(dtype)
        s["cache"] = _cache(case, pool, dtype)
        at = torch.arange(n, device="cuda")
        for i, (k, v) in enumerate(_sequences(case, gen, dtype)):
            _write(s["cache"], k, v, s["table"][i].long()[at // PAGE] * PAGE + at % PAGE)
    return s


def _cache(case, pool, dtype):
    if own:
        import qr_v2_b200_kernel_b200 as qr

        return qr.kv8_cache(pool, PAGE, case["heads"], case["dim"], dtype=dtype, device="cuda")
    one = lambda: {"codes": torch.zeros(pool, PAGE, case["heads"], case["dim"], dtype=torch.int8, device="cuda"),  # noqa: E731
                   "range": torch.zeros(pool, case["heads"], dtype=torch.float32, device="cuda")}
    return {"k": one(), "v": one()}


def _write(cache, k, v, slots):
    if own:
        import qr_v2_b200_kernel_b200 as qr

        qr.kv8_write(cache, k, v, slots)
        return
    _put(cache["k"], k, slots)
    _put(cache["v"], v, slots)


# ---- the plain forms ------------------------------------------------------------------------


def _spread(scale, rows, cols, tile):
    """A scale for every entry from one for each block of tile x 128."""
    return scale.repeat_interleave(tile, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _to_fp8(x, tile):
    """Codes and scales: each block's largest entry becomes 448, the largest code."""
    rows, cols = x.shape
    f = x.float()
    full = torch.zeros(-(-rows // tile) * tile, _blocks(cols) * BLOCK, device=x.device)
    full[:rows, :cols] = f.abs()
    a = full.reshape(-1, tile, _blocks(cols), BLOCK).amax((1, 3))
    fine = a >= TINY
    # In 64 bits: entries often lie midway between two codes, or so near that 32 bits lose on which side.
    q = f.double() * 448.0 / _spread(torch.where(fine, a, math.inf), rows, cols, tile)
    power = torch.clamp(torch.frexp(q).exponent, min=-5) - 4  # of the codes' spacing
    q = torch.ldexp(torch.round(torch.ldexp(q, -power)), power)
    return q.float().to(torch.float8_e4m3fn), torch.where(fine, a / 448.0, 0.0)


def _plain_quantise(s):
    c = s["case"]
    codes, scale = _to_fp8(s["x"], c["tile"])
    values = codes.float() * _spread(scale, c["rows"], c["cols"], c["tile"])
    return {"values": values.to(s["dtype"]), "scale": scale}


def _plain_linear(s):
    (m, k), n = s["x"].shape, s["w"].shape[0]
    x = s["x"].float() * _spread(s["x_scale"], m, k, 1)
    w = s["w"].float() * _spread(s["w_scale"], n, k, BLOCK)
    y = x @ w.T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["dtype"])


def _range(a):
    """The largest magnitude, rounded up to three significant bits."""
    part, power = torch.frexp(a)
    return torch.where(a >= TINY, torch.ldexp(torch.ceil(part * 8) / 8, power), 0.0)


def _put(part, x, slots):
    """A page's range grows to hold what is written, and its older codes follow; one whose first token is written begins anew."""
    page, at, f = slots // PAGE, slots % PAGE, x.float()
    top = torch.zeros_like(part["range"]).index_reduce_(0, page, f.abs().amax(-1), "amax")
    old = part["range"].clone()
    old[page[at == 0]] = 0.0
    new = torch.maximum(old, _range(top))
    safe = torch.where(new > 0, new, 1.0)
    grown = torch.unique(page)
    was = part["codes"][grown].float() * old[grown][:, None, :, None]
    part["codes"][grown] = torch.round(was / safe[grown][:, None, :, None]).to(torch.int8)
    part["codes"][page, at] = torch.round(f * 127.0 / safe[page].unsqueeze(-1)).to(torch.int8)
    part["range"].copy_(new)


def _get(part, slots):
    """The values, in 32 bits, that the cache stands for at these slots."""
    step = part["range"] / 127.0
    return part["codes"][slots // PAGE, slots % PAGE].float() * step[slots // PAGE].unsqueeze(-1)


def _plain_cache(s):
    _put(s["cache"]["k"], s["k"], s["slots"])
    _put(s["cache"]["v"], s["v"], s["slots"])
    return {"k": _get(s["cache"]["k"], s["read"]).to(s["dtype"]), "v": _get(s["cache"]["v"], s["read"]).to(s["dtype"])}


def _seen(case, lengths):
    """(batch, queries, tokens): which cached tokens each query sees."""
    at = torch.arange(case["length"], device="cuda")
    position = lengths.long().unsqueeze(1) - case["queries"] + torch.arange(case["queries"], device="cuda")
    seen = at <= position.unsqueeze(-1)
    if case["window"]:
        seen = seen & (at > position.unsqueeze(-1) - case["window"])
    return seen


def _plain_attention(s):
    c = s["case"]
    b, n, h, d, share, queries = c["batch"], c["length"], c["heads"], c["dim"], c["share"], c["queries"]
    at = torch.arange(n, device="cuda")
    slots = s["table"].long()[:, at // PAGE] * PAGE + at % PAGE
    k = _get(s["cache"]["k"], slots).permute(0, 2, 3, 1)  # batch, head, dim, token
    v = _get(s["cache"]["v"], slots).permute(0, 2, 1, 3)
    q = s["q"].float().reshape(b, queries, h, share, d).permute(0, 2, 3, 1, 4).reshape(b, h, share * queries, d)
    scores = (q @ k).reshape(b, h, share, queries, n) / math.sqrt(d)
    seen = _seen(c, s["lengths"])[:, None, None]
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = p.reshape(b, h, share * queries, n) @ v
    o = o.reshape(b, h, share, queries, d).permute(0, 3, 1, 2, 4).reshape(b, queries, h * share, d)
    return o.to(s["dtype"])


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"quantise": _plain_quantise, "linear": _plain_linear, "cache": _plain_cache, "attention": _plain_attention}[op](s)
    import qr_v2_b200_kernel_b200 as qr

    if op == "quantise":
        codes, scale = qr.quantize_fp8(s["x"], tile_rows=s["case"]["tile"])
        return {"values": qr.dequantize_fp8(codes, scale, s["dtype"], tile_rows=s["case"]["tile"]), "scale": scale}
    if op == "linear":
        return qr.fp8_linear(s["x"], s["x_scale"], s["w"], s["w_scale"], s["bias"], dtype=s["dtype"])
    if op == "cache":
        qr.kv8_write(s["cache"], s["k"], s["v"], s["slots"])
        k, v = qr.kv8_read(s["cache"], s["read"])
        return {"k": k, "v": v}
    return qr.kv8_attention(s["q"], s["cache"], s["table"], s["lengths"], window=s["case"]["window"] or None)


# ---- the definitions in 64 bits -------------------------------------------------------------


def _exact_fp8(x, tile):
    """(values, scales): to the nearest number of four significant bits, not below 2^-9, of a block whose top is 448."""
    rows, cols = x.shape
    values, scales = torch.zeros(rows, cols, dtype=torch.float64, device=x.device), []
    for c in range(0, cols, BLOCK):
        part = x[:, c : c + BLOCK].double()
        top = part.abs().amax(1)
        if tile > 1:
            top = torch.stack([t.amax() for t in top.split(tile)]).repeat_interleave(tile)[:rows]
        scale = top / 448
        q = part * 448 / top[:, None]
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(q.abs().clamp(min=2.0**-20))), min=-6) - 3)
        values[:, c : c + BLOCK] = (q / step).round() * step * scale[:, None]
        scales.append(scale[::tile])
    return values, torch.stack(scales, 1)


def _exact_range(a):
    power = torch.exp2(torch.floor(torch.log2(a)) - 2)
    return torch.ceil(a / power) * power


def _exact_pages(x, old):
    """What the cache makes of one sequence's (tokens, heads, dim), of which the first `old` came in an earlier call; from a page's start."""
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for p in range(0, x.shape[0], PAGE):
        page = x[p : p + PAGE].double()
        size = page.abs().amax(-1)  # tokens, heads
        new = _exact_range(size.amax(0))[None, :, None]
        before = max(0, min(PAGE, old - p))
        codes = (page * 127 / new).round()
        if before:
            was = _exact_range(size[:before].amax(0))[None, :, None]
            codes[:before] = ((page[:before] * 127 / was).round() * was / new).round()
        out[p : p + PAGE] = codes * new / 127
    return out


def exact(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    if case["op"] == "quantise":
        values, scale = _exact_fp8(_matrix(gen, case["rows"], case["cols"], dtype), case["tile"])
        return {"values": values, "scale": scale}
    if case["op"] == "linear":
        s = prepare({**case}, seed)
        k, n = case["depth"], case["outs"]
        y = torch.zeros(case["rows"], n, dtype=torch.float64, device="cuda")
        channel = torch.arange(n, device="cuda") // BLOCK
        for b in range(_blocks(k)):  # block by block of the depth
            at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            part = s["x"][:, at].double() @ s["w"][:, at].double().T
            y += part * s["x_scale"][:, b, None].double() * s["w_scale"][channel, b].double()
        return y + s["bias"].double() if s["bias"] is not None else y
    if case["op"] == "cache":
        _, _, k, v = _cache_inputs(case, gen, dtype)
        from_page = case["start"] // PAGE * PAGE
        both = ([_exact_pages(seq[from_page:], case["start"] - from_page) for seq in x] for x in (k, v))
        return {name: torch.cat(x) for name, x in zip(("k", "v"), both)}
    d, h, share, queries = case["dim"], case["heads"], case["share"], case["queries"]
    _pages(gen, case["batch"], -(-case["length"] // PAGE))
    q = torch.randn(case["batch"], queries, h * share, d, generator=gen, device="cuda").to(dtype)
    out = torch.zeros(case["batch"], queries, h * share, d, dtype=torch.float64, device="cuda")
    for i, (n, (k, v)) in enumerate(zip(_lengths(case), _sequences(case, gen, dtype))):
        k, v = _exact_pages(k, 0), _exact_pages(v, 0)  # pages are written whole, whatever of them is in use
        for j in range(0, queries, 128):  # some queries at a time
            m = min(128, queries - j)
            position = n - queries + j + torch.arange(m, device="cuda")
            last = n - queries + j + m
            if last <= 0:
                continue
            at = torch.arange(last, device="cuda")
            hidden = at > position[:, None]
            if case["window"]:
                hidden = hidden | (at <= position[:, None] - case["window"])
            scores = torch.einsum("qhgd,thd->hgqt", q[i, j : j + m].double().reshape(m, h, share, d), k[:last]) / math.sqrt(d)
            w = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
            w = torch.where(position[:, None] >= 0, w, 0.0)
            out[i, j : j + m] = torch.einsum("hgqt,thd->qhgd", w, v[:last]).reshape(m, h * share, d)
    return out
