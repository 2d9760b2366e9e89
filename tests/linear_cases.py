"""What the tests of the linear-attention layers share: inputs, batches and the comparison with the 64-bit oracle."""
from __future__ import annotations

import math

import torch

import linear_oracle

DIM = 128
HALF_STEP = 2.0 ** -8            # of a BF16 rounding, relative
UNIT = 2.0 ** -24                # of an FP32 rounding


def offsets_of(rows):
    return [sum(rows[:i]) for i in range(len(rows) + 1)]


class Problem:
    """A batch with its inputs on the GPU.  rows: new tokens of each sequence; earlier: tokens before them (None: no lengths given)."""

    def __init__(self, package, rows, *, k_heads=2, v_heads=4, width=4, earlier=None, keep=None, slots=None, spare=2, gated=False, fused=True,
                 seed=0, behind=0, short=None):
        g = torch.Generator(device="cuda").manual_seed(1000 + seed)

        def normal(*shape, std=1.0, dtype=torch.bfloat16):
            return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

        count = len(rows)
        tokens = sum(rows) + behind                     # rows behind the last sequence
        self.rows, self.tokens, self.k_heads, self.v_heads = rows, tokens, k_heads, v_heads
        channels = (2 * k_heads + v_heads) * DIM
        slots = slots if slots is not None else [int(i) for i in torch.randperm(count + spare, generator=g, device="cuda")[:count]]
        lengths = None if earlier is None else [n + e for n, e in zip(rows, earlier)]
        for s, length in (short or {}).items():         # shorter than its rows: the first of them are inactive
            lengths[s] = length
        self.batch = {"slots": slots, "offsets": offsets_of(rows), "lengths": lengths, "keep": keep}
        self.layer = package.LinearAttention(k_heads=k_heads, v_heads=v_heads, conv_width=width, slots=count + spare, max_sequences=max(count, 1),
                                             max_tokens=tokens)
        row = normal(tokens, (channels + v_heads * DIM + 2 * v_heads + 7) // 8 * 8)
        self.x = row[:, :channels] if fused else row[:, :channels].contiguous()
        self.conv_weight = normal(channels, width, std=0.5)
        self.conv_states = normal(count + spare, width - 1, channels)
        y = torch.nn.functional.silu(self.x)
        y = y.view(tokens, -1, DIM) if fused else y.view(tokens, -1, DIM).transpose(0, 1).contiguous().transpose(0, 1)
        self.q, self.k, self.v = y.split([k_heads, k_heads, v_heads], dim=1)
        ab = row[:, channels + v_heads * DIM:] if fused else normal(tokens, 2 * v_heads)
        self.b, self.a = ab[:, :v_heads], ab[:, v_heads:2 * v_heads]
        self.a_log = torch.empty(v_heads, device="cuda").uniform_(0.01, 16.0, generator=g).log()
        self.dt_bias = torch.empty(v_heads, device="cuda").uniform_(-6.0, -2.0, generator=g)
        self.gate = (row[:, channels:channels + v_heads * DIM].view(tokens, v_heads, DIM) if fused else normal(tokens, v_heads, DIM)) if gated else None
        self.norm_weight = normal(DIM, std=0.1) + 1.0
        self.states = normal(count + spare, v_heads, DIM, DIM, std=0.1, dtype=torch.float32)
        self.device_batch = self.make_batch()
        self.bind()

    def bind(self):
        self.layer.bind_layer(0, conv_weight=self.conv_weight, conv_states=self.conv_states, states=self.states, a_log=self.a_log,
                              dt_bias=self.dt_bias, norm_weight=self.norm_weight)

    def make_batch(self):
        def device(x):
            return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")

        b = self.batch
        return self.layer.batch(device(b["slots"]), tokens=self.tokens, lengths=device(b["lengths"]), row_offsets=device(b["offsets"]),
                                max_new_tokens=max(max(self.rows), 1), keep=device(b["keep"]))

    # -- convolution -----------------------------------------------------------
    def conv(self, out=None):
        return self.layer.conv(0, self.device_batch, self.x, out=out)

    def conv_wanted(self):
        return linear_oracle.conv(self.x, self.conv_weight, self.conv_states, self.batch)

    @staticmethod
    def check_conv(got, states, wanted, rows=None):
        """Up to four products and as many sums in FP32 (each off by half a step of at most the sizes' sum), the slope of silu is below 1.1,
        its own arithmetic is good to 2^-20, and the result is rounded to BF16 once (2^-133: half of the least step)."""
        out, size, want_states = wanted
        rows = slice(None) if rows is None else rows
        bound = out.abs() * (HALF_STEP + 2.0 ** -20) + 1.1 * 8 * UNIT * size + 2.0 ** -133
        off = (got.double() - out).abs()
        assert bool((off <= bound)[rows].all()), float((off / bound)[rows].max())
        assert torch.equal(states.double(), want_states)          # copies of inputs

    # -- delta rule ------------------------------------------------------------
    def delta(self, outputs=True, out=None, batch=None):
        return self.layer.delta(0, batch or self.device_batch, self.q, self.k, self.v, self.a, self.b, gate=self.gate, outputs=outputs, out=out)

    def delta_wanted(self, states=None, batch=None):
        return linear_oracle.delta(self.q, self.k, self.v, self.a, self.b, self.a_log, self.dt_bias, self.states if states is None else states,
                                   batch or self.batch, gate=self.gate, norm_weight=self.norm_weight, floor=constants(max(self.rows))[1])


def constants(rows):
    """c of the bound by the form that a batch of at most so many rows a sequence takes, and its floor in units of c.

    Token by token: a dot of 128 products is a chain of 16 and three sums by pairs (19 roundings), normalised keys are off by 12 (128
    squares in a chain of 4 and 5 pairs, a root, a product), decay and rate by 8, the update by 3: below 64 in all.

    Chunks of 64 tokens: a dot with the state is a sum of 128 products in FP32 and, its operand being held in two 11-bit terms, off by
    another 2^-22 of each: 128 + 4; the corrections of a chunk come from a sum over up to 64 tokens, each with an operand pair good to
    2^-21 (64 + 8 each, on numbers no larger than those of the bound): 64 * 72 if all of them count, whose sizes add up to the column's
    length with the chunk's; so 8192 covers both forms of the sum.  Floor: the second term has steps of 2^-24 where the column's largest
    number is 1/2 or more, so an operand is off by 2^-24 of that; 12 of them in a dot with a key of length 1 (the sum of its elements' sizes
    is at most sqrt(128)) and 64 corrections: 768 roundings."""
    return (64.0, 0.0) if rows <= STEP_ROWS else (8192.0, 768.0 / 8192.0)


STEP_ROWS = 28


def check_delta(got, states, wanted, most, typical=True):
    """got against the oracle's out (None: not looked at), states against its; `most`: the largest number of rows of a sequence."""
    c, _ = constants(most)
    if got is not None:
        out = wanted["out"]
        fine = torch.isfinite(out)
        bound = out.abs() * (HALF_STEP + 2.0 ** -18) + c * UNIT * wanted["out_error"] + 2.0 ** -133
        off = (got.double() - out).abs()
        worst = (off / bound)[fine]
        assert worst.numel() == 0 or float(worst.max()) <= 1.0, float(worst.max())
    error = (states.double() - wanted["states"]).abs()
    # the bound is of the worst case; roundings of either sign add up to a few of 2^-22 over a whole state
    size = torch.where(torch.isfinite(wanted["states"]), wanted["states"], 0.0)
    if typical:
        norm = float(torch.where(torch.isfinite(error), error, 0.0).norm() / size.norm())
        assert norm <= 2.0 ** -19, norm
    # of a column of the state: its length errs by so much, so does each element
    bound = c * UNIT * wanted["state_error"][:, :, None, :] + UNIT * wanted["states"].abs()
    fine = torch.isfinite(wanted["states"])
    worst = (error / bound.clamp_min(1e-45))[fine & (error > 0)]
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, float(worst.max())
    assert torch.equal(torch.isfinite(states), fine)
