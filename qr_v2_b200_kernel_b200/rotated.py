"""A quantised attention layer in rotated coordinates: what the orthogonal matrices of this package
    are for.

    python -m qr_v2_b200_kernel_b200.rotated [--hidden 1024] [--tokens 200] [--steps 8]

    The residual stream of a transformer has a few channels far larger than the rest, and a scale
    for a whole row then wastes the 8 bits of the others. An orthogonal ``Q`` (hidden x hidden, from
    :func:`custom_kernel` and :func:`householder_product`) spreads them: the stream is kept as ``h
    Q``, a root-mean-square norm without gain commutes with ``Q``, and the weights on either side
    absorb it (``W diag(gain) Q`` reads the stream, ``Q^T W`` writes it). In each head a second one,
    ``R`` (head_dim x head_dim), does the same for the 4-bit cache: ``(q R).(k R) = q.k``, and the
    output projection takes ``R`` back. Nothing is added to a step:

    rms_norm_int8 -> int8_linear -> kv4_write -> kv4_attention -> quantize_int8 -> int8_linear

    The command runs a prompt and some single tokens through one layer, with and without the
    rotation, and prints how far each is from the same layer in 64 bits. (No positional rotation:
    with one, ``R`` is applied after it.)
    """

from __future__ import annotations

import argparse
import json

import torch

from . import gen
from .quant import int8_linear, kv4_attention, kv4_cache, kv4_write, quantize_int8, rms_norm_int8

__all__ = ["RotatedAttention"]


class RotatedAttention:
    """One attention layer: int8 projections, a 4-bit cache, one sequence per row of ``block_table``.

    ``wq`` (heads * head_dim, hidden), ``wk`` and ``wv`` (kv_heads * head_dim, hidden), ``wo``
    (hidden, heads * head_dim) and ``gain`` (hidden,): floating point, on a CUDA device.
    ``q_hidden`` (hidden, hidden) and ``q_head`` (head_dim, head_dim): orthogonal, or ``None`` for
    no rotation. Weights are rotated in 64 bits and quantised once.
    """

    def __init__(self, wq, wk, wv, wo, gain, head_dim: int, q_hidden=None, q_head=None, dtype=torch.bfloat16):
        self.head_dim, self.dtype = head_dim, dtype
        self.heads, self.kv_heads = wq.shape[0] // head_dim, wk.shape[0] // head_dim
        eye = lambda n: torch.eye(n, dtype=torch.float64, device=wq.device)  # noqa: E731
        q = eye(wq.shape[1]) if q_hidden is None else q_hidden.double()
        r = eye(head_dim) if q_head is None else q_head.double()

        def into_heads(w):  # each head's rows, times R, reading the rotated stream
            w = w.double() * gain.double()
            return torch.einsum("de,hdi,ij->hej", r, w.unflatten(0, (-1, head_dim)), q).flatten(0, 1)

        out = torch.einsum("ij,ihd,de->jhe", q, wo.double().unflatten(1, (-1, head_dim)), r).flatten(1)
        self.qkv, self.qkv_scale = quantize_int8(torch.cat([into_heads(w) for w in (wq, wk, wv)]).float())
        self.out, self.out_scale = quantize_int8(out.float())

    def new_cache(self, pages: int, page_size: int = 64):
        return kv4_cache(pages, page_size, self.kv_heads, self.head_dim, dtype=self.dtype, device=self.qkv.device)

    def __call__(self, x, residual, cache, block_table, lengths, slots):
        """``(update, residual)`` for ``x`` (batch, queries, hidden), added to ``residual`` first (``None``:
        x is the stream).

        ``slots`` (batch * queries,): where the new tokens go in the cache; ``lengths`` (batch,):
        tokens with them. ``update`` is the layer's output, to be added to ``residual`` by the next
        norm.
        """
        batch, queries, _ = x.shape
        codes, scale, stream = rms_norm_int8(x, residual=residual)
        qkv = int8_linear(codes, scale, self.qkv, self.qkv_scale, dtype=self.dtype)
        q, k, v = qkv.unflatten(-1, (-1, self.head_dim)).split([self.heads, self.kv_heads, self.kv_heads], dim=2)
        kv4_write(cache, k.flatten(0, 1), v.flatten(0, 1), slots)
        o = kv4_attention(q, cache, block_table, lengths)
        codes, scale = quantize_int8(o.flatten(2))
        return int8_linear(codes, scale, self.out, self.out_scale, dtype=self.dtype), stream


def exact_layer(stream, wq, wk, wv, wo, gain, head_dim):
    """The layer in 64 bits, causal, without rotation or quantisation: the update for every token of ``stream``."""
    h = stream.double()
    n = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gain.double()
    q, k, v = ((n @ w.double().T).unflatten(-1, (-1, head_dim)).transpose(1, 2) for w in (wq, wk, wv))
    k, v = (x.repeat_interleave(q.shape[1] // x.shape[1], 1) for x in (k, v))
    s = q @ k.transpose(-1, -2) * head_dim**-0.5
    t = s.shape[-1]
    s = s.masked_fill(torch.ones(t, t, dtype=torch.bool, device=s.device).triu(1), float("-inf"))
    return (s.softmax(-1) @ v).transpose(1, 2).flatten(2) @ wo.double().T


def run(hidden: int = 1024, head_dim: int = 128, kv_heads: int = 2, batch: int = 3, tokens: int = 200, steps: int = 8,
        seed: int = 0, device="cuda") -> dict:
    """Relative error of the layer's updates, rotated and plain, over a prompt of ``tokens - steps`` tokens and ``steps`` single ones."""
    g = torch.Generator(device=device).manual_seed(seed)
    heads = hidden // head_dim
    rand = lambda *s: torch.randn(*s, generator=g, device=device, dtype=torch.float64)  # noqa: E731
    weights = [rand(n * head_dim, hidden) * hidden**-0.5 for n in (heads, kv_heads, kv_heads)] + [rand(hidden, hidden) * hidden**-0.5]
    weights[1][::29] *= 6  # a few key channels stand out
    gain = 1 + 0.1 * rand(hidden)
    stream = rand(batch, tokens, hidden)
    stream[..., ::97] *= 30  # and a few of the stream
    want = exact_layer(stream, *weights, gain, head_dim)
    q_hidden = gen.haar_orthogonal(1, hidden, g, device)[0].double()
    q_head = gen.haar_orthogonal(1, head_dim, g, device)[0].double()
    errors = {}
    for name, q, r in (("rotated", q_hidden, q_head), ("plain", None, None)):
        layer = RotatedAttention(*weights, gain, head_dim, q, r)
        page, per = 64, -(-tokens // 64)
        cache = layer.new_cache(batch * per, page)
        table = torch.randperm(batch * per, generator=g, device=device).reshape(batch, per).int()
        h = (stream @ q if q is not None else stream).to(layer.dtype)
        got, done = [], 0
        for new in [tokens - steps] + [1] * steps:
            at = torch.arange(done, done + new, device=device)
            slots = (table.long()[:, at // page] * page + at % page).reshape(-1)
            done += new
            lengths = torch.full((batch,), done, dtype=torch.int32, device=device)
            update, _ = layer(h[:, done - new : done], None, cache, table, lengths, slots)
            got.append(update)
        got = torch.cat(got, 1).double()
        got = got @ q.T if q is not None else got
        errors[name] = ((got - want).norm() / want.norm()).item()
    return errors


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--tokens", type=int, default=200)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    print(json.dumps({"relative_error": run(hidden=a.hidden, tokens=a.tokens, steps=a.steps)}))


if __name__ == "__main__":
    main()
