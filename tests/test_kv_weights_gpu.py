"""GPU tests of the attention's weights over their whole range, against oracle/kv_oracle.py in 64 bits.

The values are positive, so that an error that all weights of a size share shows in the output in full.  Tolerance: the output is rounded
to BF16 (2^-8), a weight may be held to 8 bits (2^-8 of itself), and 2^-9 is for scores, exponentials and sums in FP32."""
from __future__ import annotations

import math

import pytest
import torch

from test_kv_cache_gpu import Setup, _check_attention

pytestmark = pytest.mark.gpu


def _sink(package, length, new, heads, gaps, page=64, sink=3):
    """Keys that are zero but for one, whose score is `gaps` (log2 units, spread over the query heads) above all others; its
    value is zero, so that the output is what the small weights give."""
    q_heads, kv_heads, dim = heads
    setup = Setup(package, [length], [new], heads, page, 0, seed=length + new + dim)
    setup.gpu[2].fill_(2.0 ** -4)
    codes = torch.zeros(setup.gpu[0].shape)
    codes[int(setup.table[0, sink // page]), :, sink % page, 0] = 448.0
    setup.gpu[0].copy_(codes.to(torch.float8_e4m3fn).cuda())
    setup.gpu[1].copy_(setup.gpu[1].float().abs().clamp_min(1.0).to(torch.float8_e4m3fn))
    setup.gpu[1].view(torch.uint8)[int(setup.table[0, sink // page]), :, sink % page] = 0
    q = torch.zeros(new, q_heads, dim)
    low, high = gaps
    steps = torch.linspace(low, high, new * q_heads).view(new, q_heads)
    q[..., 0] = steps * math.log(2.0) * dim ** 0.5 / 28.0            # 448 / 16 = 28
    return setup, q.bfloat16()


@pytest.mark.parametrize("length", [60, 300, 1024])
@pytest.mark.parametrize("new", [1, 2, 5])
@pytest.mark.parametrize("heads", [(16, 2, 256), (16, 2, 128), (8, 1, 64), (8, 8, 64)])
def test_small_weights_of_few_rows_keep_their_bits(package, heads, new, length):
    """One position outweighs all others by 2^12 .. 2^27 and brings nothing."""
    for low, high in ((12.0, 16.0), (16.0, 20.0), (20.0, 24.0), (24.0, 27.0)):
        _check_attention(*_sink(package, length, new if new * heads[0] // heads[1] <= 16 else 1, heads, (low, high)))


@pytest.mark.parametrize("length", [60, 300, 1024])
@pytest.mark.parametrize("heads", [(16, 2, 256), (16, 2, 128), (8, 1, 64), (8, 8, 64)])
def test_small_weights_of_prompts_keep_their_bits(package, heads, length):
    """The same for many rows, up to where heads of 256 hold the weights beside the largest to 2^-8: 2^-22 of it."""
    for low, high in ((12.0, 16.0), (16.0, 19.0), (19.0, 22.0)) + (((22.0, 26.0),) if heads[2] < 256 else ()):
        _check_attention(*_sink(package, length, 40, heads, (low, high)))
