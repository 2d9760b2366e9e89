"""Outputs of the gated delta rule in chunks where values are corrected away: what is left is a small difference of what its products add
up, which both 16-bit terms of every operand of the outputs are needed for.

The limit is on the norm of all outputs' errors.  A rounding to BF16 is off by at most half a step, 2^-8 of 1 to 2, so by 2^-8 / sqrt(3)
in the mean, over numbers with a mean square of about 1.5^2: 0.0015 to 0.0017 of the norm.  States are 64 times as large as values
here, so operands good to 22 bits add 64 * 2^-22 * a few, below 2^-12 in all; operands of 11 bits add 64 * 2^-12 / sqrt(3), 2^-7 or so.
2^-9 (0.00195) lies between."""
from __future__ import annotations

import math

import pytest
import torch

import linear_oracle

DIM, CHUNK = 128, 64
LIMIT = 2.0 ** -9


def problem(rows, k_heads=2, v_heads=4, seed=0, gated=False):
    """Inputs on the CPU: nearly one key for all tokens, queries along it, rates near 1, decays of a few percent, states of 64."""
    g = torch.Generator().manual_seed(100 + seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    key = normal(1, k_heads, DIM)
    p = {"q": (key + 1.0e-3 * normal(rows, k_heads, DIM)).bfloat16(), "k": (key + 1.0e-3 * normal(rows, k_heads, DIM)).bfloat16(),
         "v": normal(rows, v_heads, DIM).bfloat16(), "a": (-3.0 + 0.5 * normal(rows, v_heads)).bfloat16(), "b": (9.0 + normal(rows, v_heads)).bfloat16(),
         "a_log": torch.zeros(v_heads), "dt_bias": torch.zeros(v_heads), "states": 64.0 * normal(1, v_heads, DIM, DIM),
         "gate": normal(rows, v_heads, DIM).bfloat16() if gated else None, "norm_weight": (1.0 + 0.1 * normal(DIM)).bfloat16()}
    return p


def wanted(p):
    rows = p["q"].shape[0]
    return linear_oracle.delta(p["q"], p["k"], p["v"], p["a"], p["b"], p["a_log"], p["dt_bias"], p["states"],
                               {"slots": [0], "offsets": [0, rows], "lengths": None, "keep": None}, gate=p["gate"], norm_weight=p["norm_weight"])


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def held(x, terms):
    """x in 16-bit terms, of columns' common power of two: the largest lies in 8 .. 16."""
    scale = 2.0 ** (3 - torch.floor(torch.log2(x.abs().amax(0, keepdim=True).clamp_min(1e-300))))
    first = (x * scale).half().double()
    second = (x * scale - first).half().double() if terms == 2 else 0.0
    return (first + second) / scale


def in_chunks(p, single=()):
    """The form in chunks in 64 bits, but for its 16-bit operands; those named in `single` have one term."""
    def terms(name, x, columns=True):
        if columns:
            return held(x, 1 if name in single else 2)
        first = x.half().double()                                  # T and the scores have no common factor
        return first if name in single else first + (x - first).half().double()

    rows, heads = p["v"].shape[:2]
    group = heads // p["k"].shape[1]
    unit = [(x.double() / torch.sqrt(x.double().square().sum(-1, keepdim=True) + 1.0e-6)).repeat_interleave(group, dim=1) for x in (p["q"], p["k"])]
    g = -torch.exp(p["a_log"].double()) * torch.nn.functional.softplus(p["a"].double() + p["dt_bias"].double())
    beta = torch.sigmoid(p["b"].double())
    out = torch.empty(rows, heads, DIM, dtype=torch.float64)
    for h in range(heads):
        s = p["states"][0, h].double()
        for begin in range(0, rows, CHUNK):
            at = slice(begin, min(begin + CHUNK, rows))
            q, k, v, rate, total = unit[0][at, h], unit[1][at, h], p["v"][at, h].double(), beta[at, h, None], g[at, h].cumsum(0)
            n = len(k)
            decay = torch.exp(total[:, None] - total[None, :]).tril()
            a = (rate * decay * (k @ k.T)).tril(-1)
            inverse = torch.linalg.inv(torch.eye(n, dtype=torch.float64) + a)
            right = rate * v - rate * torch.exp(total)[:, None] * (k @ terms("state for corrections", s))
            d = terms("T", inverse, False) @ terms("right side", right)
            o = terms("scores", decay * (q @ k.T), False) @ terms("corrections for outputs", d)
            out[at, h] = (torch.exp(total)[:, None] * (q @ terms("state for outputs", s)) + o) / math.sqrt(DIM)
            stay = torch.exp(total[-1] - total)[:, None]
            s = torch.exp(total[-1]) * s + k.T @ terms("corrections for the state", stay * d)
    if p["gate"] is not None:
        z = p["gate"].double()
        out = out / torch.sqrt(out.square().mean(-1, keepdim=True) + 1.0e-6) * p["norm_weight"].double() * z * torch.sigmoid(z)
    return out.bfloat16()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows", [70, 130])
def test_the_limit_tells_one_term_from_two(rows, gated):
    p = problem(rows, seed=rows, gated=gated)
    want = wanted(p)["out"]
    assert off(want.bfloat16(), want) <= 0.0018
    assert off(in_chunks(p), want) <= LIMIT
    for name in ("scores", "corrections for outputs", "state for outputs", "state for corrections", "T", "right side"):
        assert off(in_chunks(p, (name,)), want) > 1.5 * LIMIT, name


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows", [70, 130, 300, 1000])
def test_outputs_that_are_small_differences(package, rows, gated):
    """Chunks of one pass, and from 400 rows on segments, against 64 bits."""
    p = problem(rows, seed=rows, gated=gated)
    want = wanted(p)
    layer = package.LinearAttention(k_heads=2, v_heads=4, slots=1, max_sequences=1, max_tokens=rows)
    on = {name: x.cuda() if x is not None else None for name, x in p.items()}
    layer.bind_layer(0, states=on["states"], a_log=on["a_log"], dt_bias=on["dt_bias"], norm_weight=on["norm_weight"])
    got = layer.delta(0, layer.batch(torch.zeros(1, dtype=torch.int32, device="cuda"), tokens=rows), on["q"], on["k"], on["v"], on["a"], on["b"], gate=on["gate"])
    layer.sync()
    got, states = got.cpu(), on["states"].cpu()
    for h in range(4):
        assert off(got[:, h], want["out"][:, h]) <= LIMIT, h
    assert off(got, want["out"]) <= LIMIT
    assert off(states, want["states"]) <= 2.0 ** -19
