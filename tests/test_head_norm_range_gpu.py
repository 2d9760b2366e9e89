"""The norm of heads whose squares are beyond what FP32 holds, above and below."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import linear_oracle  # noqa: E402
from test_head_norm_gpu import check  # noqa: E402


@pytest.mark.parametrize("activation", ["none", "silu", "sigmoid"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,heads", [(7, 3), (9001, 32)])
def test_norms_of_large_and_small_heads(package, tokens, heads, dim, activation):
    """Each head goes by its own numbers, those beside it in a warp included."""
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    x = torch.randn(tokens, heads, dim, generator=g, device="cuda").bfloat16()
    gate = torch.randn(tokens, heads, dim, generator=g, device="cuda").bfloat16() if activation != "none" else None
    weight = torch.randn(dim, generator=g, device="cuda").bfloat16()
    most = torch.finfo(torch.bfloat16).max
    x[0::7, 0] *= 2.0 ** 62
    x[1::7, 1] *= 2.0 ** 100
    x[2::7, 2] = torch.where(x[2::7, 2] < 0, -most, most)
    x[3::7] *= 2.0 ** -30
    check(package.head_norm(x, weight, gate=gate, activation=activation), linear_oracle.head_norm(x, weight, 0.0, gate, activation))
    x[4::7, 0] *= 2.0 ** -48                     # with an epsilon that is no larger than these
    x[5::7, 1] *= 2.0 ** -62
    x[6::7, 2] *= 2.0 ** -100
    for eps in (0.0, 2.0 ** -120):
        check(package.head_norm(x, weight, gate=gate, activation=activation, eps=eps), linear_oracle.head_norm(x, weight, 0.0, gate, activation, eps=eps))


def test_infinities_and_zeros_beside_large_heads(package):
    x = torch.randn(5, 8, 64, device="cuda").bfloat16()
    x[0] *= 2.0 ** 90
    x[1, 2, 5], x[1, 3, 7], x[2] = float("inf"), float("nan"), 0.0
    weight = torch.randn(64, device="cuda").bfloat16()
    for eps in (1.0e-6, 0.0):
        want = linear_oracle.head_norm(x, weight, eps=eps)
        got = package.head_norm(x, weight, eps=eps)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = ~torch.isnan(want)
        assert bool(((got.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -18) + 2.0 ** -133)[fine].all())
