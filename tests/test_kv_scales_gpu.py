"""GPU tests of appends to pages whose scales came from elsewhere: any positive number, not only the powers of two that an append writes.
Tolerances as in test_kv_cache_gpu.py."""
from __future__ import annotations

import pytest
import torch

from test_kv_cache_gpu import Setup, _check_append, _check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1.5 * 2.0 ** -7, 0.01, 2.0 ** 124, 1.25 * 2.0 ** 121, 2.0 ** -90, 1.75 * 2.0 ** -66])
@pytest.mark.parametrize("heads", [(16, 2, 256), (2, 2, 64)])
def test_a_page_keeps_the_scale_it_has_while_the_new_tokens_fit(package, heads, scale):
    setup = Setup(package, [40, 70], [5, 3], heads, 64, 0, seed=5)
    for which in (2, 3):
        setup.cpu[which].fill_(scale)
        setup.gpu[which].fill_(scale)
    k, v = (setup.randn(setup.tokens, *heads[1:]).float().clamp(-4, 4) * min(scale, 2.0 ** 120) for _ in range(2))
    touched = _check_append(setup, k.bfloat16(), v.bfloat16())
    assert len(touched) == 2 * heads[1]
    for page, h in touched:
        assert all(float(setup.gpu[which][page, h]) == torch.tensor(scale).float() for which in (2, 3))


@pytest.mark.parametrize("scale", [1.5 * 2.0 ** -7, 0.01, 2.0 ** -90])
def test_a_scale_that_is_too_small_grows_to_a_power_of_two(package, scale):
    setup = Setup(package, [40, 70], [5, 3], (16, 2, 256), 64, 0, seed=6)
    for which in (2, 3):
        setup.cpu[which].fill_(scale)
        setup.gpu[which].fill_(scale)
    k, v = (setup.randn(setup.tokens, 2, 256, std=10.0) for _ in range(2))
    setup.cache.append(1, setup.batch, k.cuda(), v.cuda())
    setup.cache.sync()
    for codes, scales, x in ((0, 2, k), (1, 3, v)):
        before = setup.cpu[codes].double() * setup.cpu[scales].double()[..., None, None]
        after = setup.gpu[codes].cpu().double() * setup.gpu[scales].cpu().double()[..., None, None]
        for s, (length, new) in enumerate(zip(setup.lengths, setup.new)):
            page, slot, row = int(setup.table[s, (length - 1) // 64]), (length - 1) % 64 + 1, setup.offsets[s]
            held = slot - new
            grown = setup.gpu[scales].cpu().double()[page]
            amax = x[row:row + new].double().abs().amax((0, 2))
            assert (torch.frexp(grown)[0] == 0.5).all() and ((amax <= 448 * grown) & (amax > 224 * grown)).all()
            wish = torch.cat([before[page, :, :held], x[row:row + new].double().transpose(0, 1)], 1)
            # one rounding each: half a step of e4m3, whose steps end at 2^-9 of the scale
            bound = torch.maximum(wish.abs() * 2.0 ** -4, grown[:, None, None] * 2.0 ** -10) + wish.abs() * 2.0 ** -22
            assert ((after[page, :, :slot] - wish).abs() <= bound).all()
    _check_attention(setup, setup.randn(setup.tokens, 16, 256))
