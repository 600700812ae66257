"""Cases for the quantised operators: root-mean-square norm into 8 bits, the 8-bit matrix product,
the 4-bit key/value cache's write and read-back, and attention over that cache.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, where
``own`` is true, through the package's public entry points. ``exact`` restates each operator in
64 bits from its definition.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
PAGE = 64


def listed():
    return [
        # One sequence's next token: a single row, where the launch is the cost.
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "gain": True},
        # A ragged batch of short prompts through a narrow model without gain (folded into the weights).
        {"name": "norm ragged prompts", "op": "norm", "rows": 1777, "cols": 1000, "dtype": "fp16", "gain": False},
        # A full prefill batch of a wide model.
        {"name": "norm prefill", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "gain": True},
        # Serving one token: the weights are read once for a single row.
        {"name": "linear one token", "op": "linear", "rows": 1, "outs": 4096, "depth": 4096, "dtype": "bf16", "bias": False},
        # A ragged batch with a bias and channels that do not fill the last tile.
        {"name": "linear ragged batch", "op": "linear", "rows": 333, "outs": 1000, "depth": 2048, "dtype": "fp16", "bias": True},
        # Prefill of a wide layer: the largest product.
        {"name": "linear prefill", "op": "linear", "rows": 8192, "outs": 8192, "depth": 4096, "dtype": "bf16", "bias": False},
        # One decode step of a batch: a token for each of 16 sequences, each in a page of its own.
        {"name": "cache decode step", "op": "cache", "batch": 16, "new": 1, "start": 1023, "heads": 8, "dim": 128, "group": 128, "dtype": "bf16"},
        # Short prompts that begin and end inside a block of tokens, narrow heads in small groups.
        {"name": "cache ragged prompts", "op": "cache", "batch": 5, "new": 391, "start": 13, "heads": 4, "dim": 64, "group": 32, "dtype": "fp16"},
        # A long prompt batch.
        {"name": "cache prefill", "op": "cache", "batch": 8, "new": 4096, "start": 0, "heads": 8, "dim": 128, "group": 128, "dtype": "bf16"},
        # One sequence's next token over a short context.
        {"name": "attention one token", "op": "attention", "batch": 1, "length": 513, "queries": 1, "heads": 8, "share": 4, "dim": 128,
         "group": 128, "window": 0, "ragged": False, "dtype": "bf16"},
        # Verifying five drafted tokens for a ragged batch that has an empty slot, with a sliding window.
        {"name": "attention drafted tokens", "op": "attention", "batch": 12, "length": 2047, "queries": 5, "heads": 4, "share": 3, "dim": 64,
         "group": 32, "window": 1000, "ragged": True, "dtype": "fp16"},
        # A full serving batch over long contexts: the whole cache is read for one token of each sequence.
        {"name": "attention serving batch", "op": "attention", "batch": 64, "length": 8192, "queries": 1, "heads": 8, "share": 8, "dim": 128,
         "group": 128, "window": 0, "ragged": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "cache", "attention"])
    if op == "norm":
        cols = rng.choice([_log(rng, 64, 4096), 8 * _log(rng, 8, 512)])
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return {"op": op, "rows": _log(rng, 1, 8192 if dtype == "fp32" else 16384), "cols": cols, "dtype": dtype, "gain": rng.random() < 0.7}
    if op == "linear":
        return {"op": op, "rows": _log(rng, 1, 6000), "outs": rng.choice([_log(rng, 64, 8192), 128 * _log(rng, 1, 64)]),
                "depth": rng.choice([_log(rng, 64, 4096), 64 * _log(rng, 2, 64)]), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "bias": rng.random() < 0.5}
    dim = rng.choice([64, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "cache":
        return {"op": op, "batch": _log(rng, 1, 6), "new": _log(rng, 1, 4096), "start": rng.randrange(0, 200), "heads": rng.choice([1, 2, 4, 8]),
                "dim": dim, "group": group, "dtype": dtype}
    queries = rng.choice([1, 1, 1, _log(rng, 2, 16)])
    return {"op": op, "batch": _log(rng, 1, 48 if queries == 1 else 8), "length": _log(rng, queries, 8192), "queries": queries, "heads": rng.choice([1, 2, 4, 8]),
            "share": rng.randrange(1, 9 if queries == 1 else 5), "dim": dim, "group": group,
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


def work(case):
    op, s = case["op"], BYTES[case["dtype"]]
    if op == "norm":  # x and the residual in; the new residual and the values out; the scales
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * s * n + 4 * case["rows"] + (s * case["cols"] if case["gain"] else 0), "flops": 8 * n}
    if op == "linear":
        m, n, k = case["rows"], case["outs"], case["depth"]
        return {"bytes": m * k + n * k + s * m * n + 4 * (m + n) + (s * n if case["bias"] else 0), "flops": 2 * m * n * k}
    per_token = case["dim"] + 8 * (case["dim"] // case["group"])  # bytes of both codes, scales and minima, of one head
    if op == "cache":  # keys and values in, the cache's bytes, and their values out
        t = case["batch"] * case["new"] * case["heads"]
        return {"bytes": t * (4 * s * case["dim"] + per_token) + 8 * case["batch"] * case["new"], "flops": 12 * t * case["dim"]}
    pairs, tokens = _visible(case)
    rows = case["batch"] * case["queries"] * case["heads"] * case["share"]
    return {"bytes": tokens * case["heads"] * per_token + 2 * s * rows * case["dim"], "flops": 4 * pairs * case["heads"] * case["share"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------


def _pages(gen, batch, per_seq):
    """A block table whose pages are scattered over the pool, and the pool's size."""
    pool = batch * per_seq + 3
    table = torch.randperm(pool, generator=gen, device="cuda")[: batch * per_seq].reshape(batch, per_seq)
    return table.to(torch.int32).contiguous(), pool


def _keys_values(gen, tokens, heads, dim, dtype):
    """Keys whose channels differ in size and centre, as keys do, and plainer values."""
    size = torch.exp(0.4 * torch.randn(heads, dim, generator=gen, device="cuda"))
    centre = 0.7 * torch.randn(heads, dim, generator=gen, device="cuda")
    k = torch.randn(tokens, heads, dim, generator=gen, device="cuda") * size + centre
    v = torch.randn(tokens, heads, dim, generator=gen, device="cuda")
    return k.to(dtype), v.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": dict(case), "dtype": dtype}
    if case["op"] == "norm":
        size = torch.exp(0.5 * torch.randn(case["cols"], generator=gen, device="cuda"))
        s["x"] = (torch.randn(case["rows"], case["cols"], generator=gen, device="cuda") * size).to(dtype)
        s["residual"] = (2.0 * torch.randn(case["rows"], case["cols"], generator=gen, device="cuda") * size).to(dtype)
        s["gain"] = (1 + 0.2 * torch.randn(case["cols"], generator=gen, device="cuda")).to(dtype) if case["gain"] else None
    elif case["op"] == "linear":
        m, n, k = case["rows"], case["outs"], case["depth"]
        s["x"] = (35 * torch.randn(m, k, generator=gen, device="cuda")).round().clamp(-127, 127).to(torch.int8)
        s["w"] = (35 * torch.randn(n, k, generator=gen, device="cuda")).round().clamp(-127, 127).to(torch.int8)
        s["x_scale"] = 0.02 * torch.exp(0.3 * torch.randn(m, generator=gen, device="cuda"))
        s["w_scale"] = 0.002 * torch.exp(0.3 * torch.randn(n, generator=gen, device="cuda"))
        s["bias"] = torch.randn(n, generator=gen, device="cuda").to(dtype) if case["bias"] else None
    elif case["op"] == "cache":
        b, new, start = case["batch"], case["new"], case["start"]
        table, pool = _pages(gen, b, -(-(start + new) // PAGE))
        at = torch.arange(start, start + new, device="cuda")
        s["slots"] = (table.long()[:, at // PAGE] * PAGE + at % PAGE).reshape(-1)
        s["k"], s["v"] = _keys_values(gen, b * new, case["heads"], case["dim"], dtype)
        s["cache"] = _cache(case, pool, dtype)
    else:
        b, n, h, d = case["batch"], case["length"], case["heads"], case["dim"]
        s["table"], pool = _pages(gen, b, -(-n // PAGE))
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        s["q"] = torch.randn(b, case["queries"], h * case["share"], d, generator=gen, device="cuda").to(dtype)
        s["cache"] = _cache(case, pool, dtype)
        at = torch.arange(n, device="cuda")
        for i in range(b):
            k, v = _keys_values(gen, n, h, d, dtype)
            slots = s["table"][i].long()[at // PAGE] * PAGE + at % PAGE
            _write(s["cache"], k, v, slots, case["group"])
    return s


def _cache(case, pool, dtype):
    if own:
        import qr_v2_b200_kernel_b200 as qr

        return qr.kv4_cache(pool, PAGE, case["heads"], case["dim"], group_size=case["group"], dtype=dtype, device="cuda")
    h, d, groups = case["heads"], case["dim"], case["dim"] // case["group"]
    one = lambda: {"codes": torch.zeros(pool * PAGE, h, d, dtype=torch.uint8, device="cuda"),  # noqa: E731
                   "scale": torch.zeros(pool * PAGE, h, groups, dtype=dtype, device="cuda"),
                   "low": torch.zeros(pool * PAGE, h, groups, dtype=dtype, device="cuda")}
    return {"k": one(), "v": one()}


def _write(cache, k, v, slots, group):
    if own:
        import qr_v2_b200_kernel_b200 as qr

        qr.kv4_write(cache, k, v, slots)
        return
    _put(cache["k"], k, slots, group)
    _put(cache["v"], v, slots, group)


# ---- the plain forms ------------------------------------------------------------------------


def _put(part, x, slots, group):
    """Each group's minimum and step in the cache's type, and its codes relative to those."""
    t, h, d = x.shape
    g = x.float().reshape(t, h, d // group, group)
    lo, hi = g.amin(-1), g.amax(-1)
    fine = torch.isfinite(lo) & torch.isfinite(hi)
    step = torch.where(fine, hi * (1 / 15) - lo * (1 / 15), float("nan")).to(x.dtype)
    low = torch.where(fine, lo, float("nan")).to(x.dtype)
    inv = torch.where(step.float() >= 2.0**-126, 1 / step.float(), 0.0)
    codes = torch.clamp(torch.round((g - low.float().unsqueeze(-1)) * inv.unsqueeze(-1)), 0, 15)
    codes = torch.where(fine.unsqueeze(-1), codes, 0.0)
    part["codes"][slots] = codes.reshape(t, h, d).to(torch.uint8)
    part["scale"][slots] = step
    part["low"][slots] = low


def _get(part, slots):
    """The values, in 32 bits, that the cache stands for at these slots."""
    codes, step, low = part["codes"][slots].float(), part["scale"][slots].float(), part["low"][slots].float()
    g = codes.unflatten(-1, (step.shape[-1], -1))
    return (low.unsqueeze(-1) + step.unsqueeze(-1) * g).flatten(-2)


def _plain_norm(s):
    h = s["x"].float() + s["residual"].float()
    t = h * s["gain"].float() if s["gain"] is not None else h
    a = t.abs().amax(-1, keepdim=True)
    scale = a * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) / 127
    codes = torch.round(t * (127.0 / a))
    return {"values": (codes * scale).to(s["dtype"]), "scale": scale.squeeze(-1), "residual": h.to(s["dtype"])}


def _plain_linear(s):
    y = (s["x"].float() @ s["w"].float().T) * s["x_scale"].unsqueeze(1) * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["dtype"])


def _plain_cache(s):
    _put(s["cache"]["k"], s["k"], s["slots"], s["case"]["group"])
    _put(s["cache"]["v"], s["v"], s["slots"], s["case"]["group"])
    return {"k": _get(s["cache"]["k"], s["slots"]).to(s["dtype"]), "v": _get(s["cache"]["v"], s["slots"]).to(s["dtype"])}


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
        return {"norm": _plain_norm, "linear": _plain_linear, "cache": _plain_cache, "attention": _plain_attention}[op](s)
    import qr_v2_b200_kernel_b200 as qr

    if op == "norm":
        codes, scale, residual = qr.rms_norm_int8(s["x"], s["gain"], s["residual"], eps=EPS)
        return {"values": qr.dequantize_int8(codes, scale, s["dtype"]), "scale": scale, "residual": residual}
    if op == "linear":
        return qr.int8_linear(s["x"], s["x_scale"], s["w"], s["w_scale"], s["bias"], dtype=s["dtype"])
    if op == "cache":
        qr.kv4_write(s["cache"], s["k"], s["v"], s["slots"])
        k, v = qr.kv4_read(s["cache"], s["slots"])
        return {"k": k, "v": v}
    return qr.kv4_attention(s["q"], s["cache"], s["table"], s["lengths"], window=s["case"]["window"] or None)


# ---- the definitions in 64 bits -------------------------------------------------------------


def _exact_values(x, group):
    """What a 4-bit cache makes of x: the group's range in fifteen steps, its ends held in x's type."""
    g = x.double().unflatten(-1, (-1, group))
    low = g.min(-1, keepdim=True).values
    step = ((g.max(-1, keepdim=True).values - low) / 15).to(x.dtype).double()
    codes = torch.where(step > 0, ((g - low) / torch.where(step > 0, step, 1.0)).round(), 0.0).clamp(0, 15)
    return (low + codes * step).flatten(-2)


def exact(case, seed):
    s = prepare({**case}, seed)
    if case["op"] == "norm":
        h = s["x"].double() + s["residual"].double()
        y = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
        if s["gain"] is not None:
            y = y * s["gain"].double()
        scale = y.abs().amax(-1, keepdim=True) / 127
        return {"values": (y / scale).round() * scale, "scale": scale.squeeze(-1), "residual": h}
    if case["op"] == "linear":
        y = s["x"].double() @ s["w"].double().T * s["x_scale"].double()[:, None] * s["w_scale"].double()
        return y + s["bias"].double() if s["bias"] is not None else y
    if case["op"] == "cache":
        return {"k": _exact_values(s["k"], case["group"]), "v": _exact_values(s["v"], case["group"])}
    d, h, share, queries = case["dim"], case["heads"], case["share"], case["queries"]
    out = torch.zeros(case["batch"], queries, h * share, d, dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lengths(case)):  # sequence by sequence, query by query
        at = torch.arange(n, device="cuda")
        slots = s["table"][i].long()[at // PAGE] * PAGE + at % PAGE
        k, v = (torch.addcmul(p["low"][slots].double().unsqueeze(-1), p["scale"][slots].double().unsqueeze(-1),
                              p["codes"][slots].double().unflatten(-1, (-1, case["group"]))).flatten(-2) for p in (s["cache"]["k"], s["cache"]["v"]))
        for j in range(queries):
            position = n - queries + j
            first = max(0, position - case["window"] + 1) if case["window"] else 0
            if position < 0:
                continue
            q = s["q"][i, j].double().reshape(h, share, d)
            w = torch.softmax(torch.einsum("hgd,thd->hgt", q, k[first : position + 1]) / math.sqrt(d), -1)
            out[i, j] = torch.einsum("hgt,thd->hgd", w, v[first : position + 1]).reshape(h * share, d)
    return out
