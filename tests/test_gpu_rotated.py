"""The quantised attention layer in rotated coordinates: the operators together, as a user runs them."""

import pytest
import torch

from qr_v2_b200_kernel_b200 import rotated

pytestmark = pytest.mark.gpu


def test_rotation_makes_the_layer_fit_its_bits():
    """Rows in 8 bits lose up to half of 1/127 of their largest entry an entry, about 3 rms once rotated (and 30 in the
    outlying channels' rows before): under 1 % of the rms a product, and a 4-bit step is some 6 sigma / 15,
    0.12 sigma rms, on the keys and values. Updates average values, so a few tenths bound them safely."""
    errors = rotated.run()
    assert errors["rotated"] < 0.25
    assert errors["rotated"] < 0.7 * errors["plain"]


def test_a_prompt_and_single_tokens_agree():
    """The projections sum integers, so they do not depend on how tokens are grouped; the attention's grouping moves its
    result by less than its rounding, and the 8-bit codes of the next product by a step at most."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w = lambda *s: torch.randn(*s, generator=g, device="cuda") * s[1] ** -0.5  # noqa: E731
    layer = rotated.RotatedAttention(w(512, 512), w(256, 512), w(256, 512), w(512, 512), torch.ones(512, device="cuda"), 64)
    x = torch.randn(2, 37, 512, generator=g, device="cuda").bfloat16()
    table = torch.tensor([[2, 0, 5], [1, 4, 3]], dtype=torch.int32, device="cuda")
    at = lambda lo, hi: (table.long()[:, torch.arange(lo, hi, device="cuda") // 16] * 16  # noqa: E731
                         + torch.arange(lo, hi, device="cuda") % 16).reshape(-1)
    full = lambda n: torch.full((2,), n, dtype=torch.int32, device="cuda")  # noqa: E731
    a, b = layer.new_cache(6, 16), layer.new_cache(6, 16)
    whole, stream = layer(x, None, a, table, full(37), at(0, 37))
    assert stream is x
    parts = torch.cat([layer(x[:, i : i + 1], None, b, table, full(i + 1), at(i, i + 1))[0] for i in range(37)], 1)
    assert torch.equal(a.data, b.data)  # the caches, bit for bit
    assert torch.all((whole.float() - parts.float()).abs() <= 0.02 * whole.float().abs().max())
