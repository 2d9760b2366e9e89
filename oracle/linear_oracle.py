"""The linear-attention layers' convolution and gated delta rule and the head norm, restated in 64 bits, one sequence and one token at
a time.  Tensors are those of the library's interface (on any device); results are float64.

The delta rule comes with a bound on what 32-bit arithmetic may change, in units of the rounding: a state's column errs by e with
    e <- alpha e + c (alpha n (1 + |g|) + beta |v|),        n: the column's length before the token,
because the token's correction (1 - beta k k^T) shortens no error less than 1, and every number that the token adds is a product or a
sum of numbers no larger than the column's length and the value."""
from __future__ import annotations

import math

import torch

DIM = 128


def sequences(batch: dict):
    """(sequence, first row, rows, first active row, kept rows, fresh, slot) of a batch {slots, offsets, lengths, keep}, as lists."""
    for s, slot in enumerate(batch["slots"]):
        row0, rows = batch["offsets"][s], batch["offsets"][s + 1] - batch["offsets"][s]
        length = batch["lengths"][s] if batch.get("lengths") is not None else None
        kept = rows if batch.get("keep") is None else min(max(batch["keep"][s], 0), rows)
        fresh = length is not None and length <= rows
        first = rows if slot < 0 else rows - length if fresh else 0
        yield s, row0, rows, first, kept, fresh, slot


def conv(x, weight, states, batch):
    """(out, sum of the products' sizes [tokens, channels], states): rows of no sequence are NaN in out."""
    width = weight.shape[1]
    w, x, states = weight.double(), x.double(), states.double().clone()
    out = torch.full_like(x, math.nan)
    size = torch.zeros_like(x)
    for _, row0, rows, first, kept, fresh, slot in sequences(batch):
        out[row0:row0 + rows] = 0.0
        if first == rows:
            continue
        before = torch.zeros_like(states[slot]) if fresh else states[slot]
        line = torch.cat([before, x[row0 + first:row0 + rows]])
        n = rows - first
        y = sum(line[j:j + n] * w[:, j] for j in range(width))
        size[row0 + first:row0 + rows] = sum((line[j:j + n] * w[:, j]).abs() for j in range(width))
        out[row0 + first:row0 + rows] = y * torch.sigmoid(y)
        if kept > first:
            states[slot] = line[kept - first:kept - first + width - 1]
    return out, size, states


def delta(q, k, v, a, b, a_log, dt_bias, states, batch, eps=1.0e-6, gate=None, norm_weight=None, floor=0.0):
    """{"out", "states", "out_error", "state_error", "reach"}.  `floor` is for arithmetic in chunks of 64 tokens, which holds a column and its
    values to so much of the largest that they come to within a chunk and the one before: that much is added to e with every chunk.  out_error [tokens, heads, 128] and state_error [slots, heads, 128] (of a
    column) are the bound above for c = 1 and a rounding of 1; reach [tokens, heads, 128] is the length of the column that the query
    reads, and with it of what it has added up, over sqrt(128).  Rows of no sequence are NaN."""
    device = v.device
    heads = v.shape[1]
    group = heads // k.shape[1]
    unit = [(x.double() / torch.sqrt(x.double().square().sum(-1, keepdim=True) + eps)).repeat_interleave(group, dim=1) for x in (q, k)]
    q, k, v = unit[0] / math.sqrt(DIM), unit[1], v.double()
    x = a.double() + dt_bias.double()
    g = -torch.exp(a_log.double()) * torch.where(x > 30, x, torch.log1p(torch.exp(x.clamp_max(30))))
    alpha, beta = torch.exp(g), torch.sigmoid(b.double())
    states = states.double().clone()
    out = torch.full((v.shape[0], heads, DIM), math.nan, dtype=torch.float64, device=device)
    out_error, reach = torch.zeros_like(out), torch.zeros_like(out)
    state_error = torch.zeros(states.shape[0], heads, DIM, dtype=torch.float64, device=device)
    for _, row0, rows, first, kept, fresh, slot in sequences(batch):
        out[row0:row0 + rows] = 0.0
        if first == rows:
            continue
        s = torch.zeros_like(states[slot]) if fresh else states[slot].clone()
        e = torch.zeros(heads, DIM, dtype=torch.float64, device=device)
        n = s.square().sum(1).sqrt()
        largest, largest_before = torch.zeros_like(n), torch.zeros_like(n)
        for t in range(row0 + first, row0 + rows):
            largest = torch.maximum(largest, torch.maximum(n, v[t].abs()).nan_to_num(0.0, 0.0))
            al, be, kt = alpha[t, :, None], beta[t, :, None], k[t][..., None]
            e = al * e + al * n * (1.0 + g[t].abs()[:, None]) + be * v[t].abs()
            s = s * al[..., None]
            d = be * (v[t] - (s * kt).sum(1))
            s = s + kt * d[:, None, :]
            before, n = n, s.square().sum(1).sqrt()
            out[t] = (s * q[t][..., None]).sum(1)
            reach[t] = (al * before + be * v[t].abs() + n) / math.sqrt(DIM)
            out_error[t] = e / math.sqrt(DIM) + reach[t]
            here, last = t - row0 - first, t == row0 + rows - 1
            if t - row0 + 1 == kept:
                states[slot], state_error[slot] = s, e + floor * torch.maximum(largest, largest_before)
            if here % 64 == 63 or last:
                held = torch.maximum(largest, largest_before)
                out_error[t - here % 64:t + 1] += floor * held / math.sqrt(DIM)
                e = e + floor * held
                largest_before, largest = largest, torch.zeros_like(n)
    result = {"out": out, "states": states, "out_error": out_error, "state_error": state_error, "reach": reach}
    if gate is not None:
        z, w = gate.double(), norm_weight.double()
        scale = 1.0 / torch.sqrt(out.square().mean(-1, keepdim=True) + eps)
        factor = (w * z * torch.sigmoid(z)).abs() * scale
        result["out"] = out * scale * w * z * torch.sigmoid(z)
        for name in ("out_error", "reach"):           # of the output itself, and of its head's norm
            result[name] = factor * (result[name] + out.abs() * scale * result[name].square().mean(-1, keepdim=True).sqrt())
    return result


def head_norm(x, weight=None, offset=0.0, gate=None, activation="none", eps=1.0e-6):
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    if gate is not None:
        z = gate.double()
        y = y * torch.sigmoid(z) * (z if activation == "silu" else 1.0)
    return y
