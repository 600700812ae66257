"""The attention layer over the 8-bit cache and with products in 8-bit floating point: those operators together, as a
user runs them."""

import json
import subprocess
import sys

import pytest
import torch

from qr_v2_b200_kernel_b200 import rotated

pytestmark = pytest.mark.gpu


def test_an_8_bit_cache_is_closer_than_a_4_bit_one():
    """A step of the 8-bit cache is at most 1.25 / 127 of a page's largest entry, some 5 sigma: 0.05 sigma, 0.014 rms, and a
    few times that where the range grew. That and two products of rows in 8 bits, under 1 % each, make a few
    hundredths; a 4-bit step alone is 0.12 sigma rms."""
    errors = rotated.run(cache_bits=8)
    assert errors["rotated"] < 0.08
    assert errors["rotated"] < 0.5 * rotated.run()["rotated"]


@pytest.mark.parametrize("cache_bits", [4, 8])
def test_products_in_8_bit_floating_point(cache_bits):
    """Codes of four significant bits are off by up to 2^-4 of the entry, 0.036 rms at most: 0.051 for a product of two. Scores,
    of size one, are off by 0.07 then and the values by 0.05; the second product adds 0.05: about 0.1, and 0.15 with the 4-bit
    cache. Without the rotation blocks still have scales of their own, so little is lost."""
    errors = rotated.run(products="fp8", cache_bits=cache_bits)
    assert errors["rotated"] < 0.25 and errors["plain"] < (0.25 if cache_bits == 8 else 0.6)


@pytest.mark.parametrize("products", ["int8", "fp8"])
def test_a_prompt_and_single_tokens_agree(products):
    """How tokens are grouped moves a product in 8-bit floating point by 32-bit roundings only (not at all in integers), so keys
    and values agree to a bf16 rounding; a page's range is the same, and its codes were rounded again where it grew: by half a step each
    time, of at most 1.25 / 127 of the largest, where four steps of the range double it."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w = lambda *s: torch.randn(*s, generator=g, device="cuda") * s[1] ** -0.5  # noqa: E731
    layer = rotated.RotatedAttention(w(512, 512), w(256, 512), w(256, 512), w(512, 512), torch.ones(512, device="cuda"), 64, products=products,
                                     cache_bits=8)
    x = torch.randn(2, 37, 512, generator=g, device="cuda").bfloat16()
    table = torch.tensor([[2, 0, 5], [1, 4, 3]], dtype=torch.int32, device="cuda")
    at = lambda lo, hi: (table.long()[:, torch.arange(lo, hi, device="cuda") // 16] * 16  # noqa: E731
                         + torch.arange(lo, hi, device="cuda") % 16).reshape(-1)
    full = lambda n: torch.full((2,), n, dtype=torch.int32, device="cuda")  # noqa: E731
    a, b = layer.new_cache(6, 16), layer.new_cache(6, 16)
    whole, stream = layer(x, None, a, table, full(37), at(0, 37))
    assert stream is x
    parts = torch.cat([layer(x[:, i : i + 1], None, b, table, full(i + 1), at(i, i + 1))[0] for i in range(37)], 1)
    if products == "int8":
        assert torch.equal(a.range, b.range)
    assert torch.all((a.range - b.range).abs() <= 0.25 * a.range)  # a rounding may take the largest entry past a step of the range
    assert torch.all((whole.float() - parts.float()).abs() <= 0.1 * whole.float().abs().max())


def test_residual_and_refusals():
    layer = rotated.RotatedAttention(*(torch.randn(64, 64, device="cuda") for _ in range(4)), torch.ones(64, device="cuda"), 64, products="fp8", cache_bits=8)
    x = torch.randn(1, 3, 64, device="cuda").bfloat16()
    table, slots = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.arange(3, device="cuda")
    n = torch.full((1,), 3, dtype=torch.int32, device="cuda")
    update, stream = layer(x, x, layer.new_cache(1, 16), table, n, slots)
    assert torch.equal(stream, x + x) and torch.equal(update, layer(x + x, None, layer.new_cache(1, 16), table, n, slots)[0])
    for change in (dict(products="fp4"), dict(cache_bits=16)):
        with pytest.raises(ValueError):
            rotated.RotatedAttention(*(torch.randn(64, 64, device="cuda") for _ in range(4)), torch.ones(64, device="cuda"), 64, **change)


def test_the_command():
    out = subprocess.run([sys.executable, "-m", "qr_v2_b200_kernel_b200.rotated", "--hidden", "256", "--tokens", "40", "--products", "fp8", "--cache-bits", "8"],
                         capture_output=True, text=True, check=True).stdout
    assert set(json.loads(out)["relative_error"]) == {"rotated", "plain"}
