"""Linear-attention layers with numbers near the ends of what BF16 and FP32 hold, in both forms of the delta rule."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from linear_cases import DIM, Problem, check_delta  # noqa: E402


def check(p):
    wanted = p.delta_wanted()
    assert bool(torch.isfinite(wanted["out"]).all()) and float(wanted["states"].abs().max()) < 2.0 ** 127
    got = p.delta()
    p.layer.sync()
    check_delta(got, p.states, wanted, max(p.rows))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows", [[28, 20], [29, 20], [150, 90]])
def test_large_corrections_while_the_state_decays(package, rows, gated):
    """Values and states of 2^120 in a state that has decayed by 2^-15, 2^-28 and more: all that the formula has stays finite."""
    p = Problem(package, rows, earlier=[3] * len(rows), seed=11, gated=False)
    p.a, p.v = p.a.clone(), p.v.clone()
    p.a_log.zero_()
    p.dt_bias.zero_()
    p.a.zero_()                                  # decay 1/2
    p.a[::7] = -4.0                              # nearly none
    p.a[5::13] = 30.0                            # nearly all
    columns = [0, 1, 3, 126] if not gated else [3]
    p.v[:, 1, columns] *= 2.0 ** 120
    p.states[:, 2, :, 4] *= 2.0 ** 120
    p.states[:, 3, :, 5] *= 2.0 ** 124
    check(p)


@pytest.mark.parametrize("rows", [[12, 9], [28, 29], [100, 90]])
def test_large_and_small_keys_and_queries(package, rows):
    """Keys and queries count by their direction, whatever their length, until it falls below the norm's epsilon."""
    p = Problem(package, rows, earlier=[3] * len(rows), seed=12, gated=True)
    p.q, p.k = p.q.clone(), p.k.clone()
    most = torch.finfo(torch.bfloat16).max
    for x, at in ((p.k, 2), (p.q, 3)):
        x[at] *= 2.0 ** 62
        x[at + 2, 0] *= 2.0 ** 100
        x[at + 4] = torch.where(x[at + 4] < 0, -most, most)
        x[at + 6] *= 2.0 ** -80
        x[at + 8] *= 2.0 ** -9
    check(p)


@pytest.mark.parametrize("rows", [[12, 9], [28, 29], [100, 90], [600]])
def test_large_outputs_are_normed(package, rows):
    """Outputs whose squares are beyond FP32 under the gate's norm."""
    p = Problem(package, rows, earlier=[3] * len(rows), seed=13, gated=True)
    p.v = p.v.clone()
    p.v[:, 1] *= 2.0 ** 66
    p.states[:, 1] *= 2.0 ** 66
    p.v[:, 2] *= 2.0 ** 110
    p.states[:, 2] *= 2.0 ** 110
    p.v[:, 3, ::2] *= 2.0 ** 90
    check(p)


@pytest.mark.parametrize("gated", [False, True])
def test_decays_between_tokens_behind_a_strong_one(package, gated):
    """One token of each 16 lets the state decay by 2^-62, those behind it by 2^-0.02 or so.  With one key for all tokens, a rate of 1 and
    one value, the state is key x value after every token, and what the last token corrects away shows the decay from the strong one to
    it as the kernel has it.  Keys of 64 ones have a length that is exact, and products that are.

    Independent roundings, whose squares add up over many heads: two exponentials (2^-22 each), four products in FP32 (2^-24 each), two
    terms of the entry of T and of the correction (2^-23 each), a substitution of up to 15 products (2^-25 each), the decays of up to 12
    corrections (2^-24 each): 1.94 * 2^-22 of the state in all."""
    rows = [66 + i for i in range(12)]
    heads = 64
    p = Problem(package, rows, k_heads=1, v_heads=heads, earlier=[3] * len(rows), seed=14, gated=gated)
    g = torch.Generator(device="cuda").manual_seed(15)
    sign = torch.where(torch.randn(DIM, generator=g, device="cuda") < 0, -1.0, 1.0)
    sign[torch.randperm(DIM, generator=g, device="cuda")[:64]] = 0.0
    p.k = sign.bfloat16().expand(p.tokens, 1, DIM)
    p.q = p.k
    p.v = torch.randn(1, heads, DIM, generator=g, device="cuda").bfloat16().expand(p.tokens, -1, -1)
    p.a_log.zero_()
    p.dt_bias.zero_()
    p.a = (torch.randn(p.tokens, heads, generator=g, device="cuda") * 0.5 - 4.0).bfloat16()
    for s, row0 in enumerate(p.batch["offsets"][:-1]):
        p.a[row0 + 1:row0 + rows[s]:16] = 43.0                  # softplus(43) = 43 = 62 log 2
    p.b = torch.full_like(p.a, 100.0)
    wanted = p.delta_wanted()
    got = p.delta()
    p.layer.sync()
    check_delta(got, p.states, wanted, max(rows))
    slots = p.batch["slots"]
    norm = float((p.states[slots].double() - wanted["states"][slots]).norm() / wanted["states"][slots].norm())
    assert norm <= 2.0 ** -21, norm
