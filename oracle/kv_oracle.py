"""The full-attention cache and the verification of drafted tokens, restated in 64 bits, one sequence, page, row and token at a
time.  Tensors are those of the library's interface; results are float64 (codes as the numbers they are) or Python integers."""
from __future__ import annotations

import math

import torch

LARGEST, MIN_EXPONENT, MAX_EXPONENT = 448.0, -64, 120


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 number (ties to even), saturating at 448: three bits after the leading one, steps of 2^-9 at the least."""
    x = x.double()
    _, exponent = torch.frexp(x)                                  # |x| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(x), (exponent - 1).clamp_min(-6) - 3)
    return (torch.round(x / step) * step).clamp(-LARGEST, LARGEST)


def exponent_for(amax: float) -> int:
    """The least e, within the range, with amax <= 448 * 2^e."""
    if amax == 0.0:
        return MIN_EXPONENT
    e = math.frexp(amax)[1] - 9
    while amax > math.ldexp(LARGEST, e):
        e += 1
    return min(max(e, MIN_EXPONENT), MAX_EXPONENT)


def rotate(x: torch.Tensor, table_row: torch.Tensor) -> torch.Tensor:
    """x [heads, dim] at one position; table_row: cosines, then sines."""
    half = table_row.numel() // 2
    c, s = table_row[:half].double(), table_row[half:].double()
    y = x.double().clone()
    a, b = x[:, :half].double(), x[:, half:2 * half].double()
    y[:, :half] = a * c - b * s
    y[:, half:2 * half] = b * c + a * s
    return y


def rows_of(lengths: list[int], offsets: list[int]):
    """(sequence, row, position) of every row of a sequence."""
    for s, length in enumerate(lengths):
        rows = offsets[s + 1] - offsets[s]
        for i in range(rows):
            yield s, offsets[s] + i, length - rows + i


def append(keys, values, key_scales, value_scales, table, offsets, lengths, k, v, rotation, page_tokens):
    """Updates the four float64 tensors in place (codes as numbers); returns {(page, head): (old exponents or None)} of what it touched."""
    heads = keys.shape[1]
    touched: dict = {}
    for s, row, position in rows_of(lengths, offsets):
        if position < 0:
            continue
        page = int(table[s][position // page_tokens])
        turned = rotate(k[row], rotation[position])
        for h in range(heads):
            entry = touched.setdefault((page, h), {"first": position % page_tokens, "rows": []})
            entry["rows"].append((position % page_tokens, turned[h], v[row, h].double()))
    for (page, h), entry in touched.items():
        held = entry["first"]
        sound = [(slot, a, b) for slot, a, b in entry["rows"] if bool(torch.isfinite(a).all() and torch.isfinite(b).all())]
        for which, codes, scales in ((1, keys, key_scales), (2, values, value_scales)):
            amax = max((float(r[which].abs().max()) for r in sound), default=0.0)
            scale, old = 2.0 ** exponent_for(amax), float(scales[page, h])
            if held > 0 and amax <= LARGEST * old:
                scale = old                                       # the page keeps the one it has
            elif held > 0:
                codes[page, h, :held] = e4m3(codes[page, h, :held] * (old / scale))
            entry["amax%d" % which] = amax
            scales[page, h] = scale
            for r in entry["rows"]:
                codes[page, h, r[0]] = e4m3(r[which] / scale)
        for slot, a, b in entry["rows"]:
            if not bool(torch.isfinite(a).all() and torch.isfinite(b).all()):
                keys[page, h, slot] = math.nan
                values[page, h, slot] = 0.0
    return touched


def attention(keys, values, key_scales, value_scales, table, offsets, lengths, q, scale, page_tokens):
    """(out, spread) float64 [tokens, heads, dim]: spread is the same average over |v|, the unit that errors of the weights come in."""
    tokens, q_heads, dim = q.shape
    kv_heads = keys.shape[1]
    group = q_heads // kv_heads
    out = torch.zeros(tokens, q_heads, dim, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    for s, length in enumerate(lengths):
        rows = offsets[s + 1] - offsets[s]
        if rows == 0 or length == 0:
            continue
        pages = torch.as_tensor(table[s][:(length + page_tokens - 1) // page_tokens], device=q.device).long()
        k, v = ((x[pages].double() * y[pages].double()[..., None, None]).transpose(0, 1).reshape(kv_heads, -1, dim)[:, :length]
                for x, y in ((keys, key_scales), (values, value_scales)))
        position = torch.arange(length - rows, length, device=q.device)
        hidden = torch.arange(length, device=q.device)[None, :] > position[:, None]
        seen = position >= 0
        for h in range(q_heads):
            scores = (q[offsets[s]:offsets[s + 1], h].double() @ k[h // group].T) * scale
            scores = scores.masked_fill(hidden, -math.inf)
            p = torch.softmax(scores, -1)
            p[~seen] = 0.0
            # a masked position contributes nothing, whatever it holds
            out[offsets[s]:offsets[s + 1], h] = p @ v[h // group]
            spread[offsets[s]:offsets[s + 1], h] = p @ v[h // group].abs()
    return out, spread


def verify(target, drafts, uniforms, draft=None, counts=None):
    """(accepted, tokens) as lists; target, drafts, ... are CPU tensors."""
    def number(x):                     # NaN and negative numbers count as 0
        x = float(x)
        return x if x > 0.0 else 0.0

    def product32(a, b):
        return float(torch.tensor(a, dtype=torch.float32) * torch.tensor(b, dtype=torch.float32))

    accepted, tokens = [], []
    most, vocabulary = drafts.shape[1], target.shape[2]
    for s in range(target.shape[0]):
        n = most if counts is None else min(max(int(counts[s]), 0), most)
        a = 0
        while a < n:
            x = int(drafts[s, a])
            if not 0 <= x < vocabulary:
                break
            q = 1.0 if draft is None else number(draft[s, a, x])
            if not product32(number(uniforms[s, a]), q) < number(target[s, a, x]):
                break
            a += 1
        p = torch.nan_to_num(target[s, a].float(), nan=0.0).clamp_min(0.0)
        rest = p.clone()
        if a < n and draft is not None:
            rest = p - torch.nan_to_num(draft[s, a].float(), nan=0.0).clamp_min(0.0)
        elif a < n and 0 <= int(drafts[s, a]) < vocabulary:
            rest[int(drafts[s, a])] = 0.0
        token = -1
        for weights in (rest, p):
            whole = (weights.double().clamp(0.0, 1.0) * 2.0 ** 40).floor().long()
            total = int(whole.sum())
            if total:
                step = int(min(max(number(uniforms[s, most]), 0.0), 1.0 - 2.0 ** -24) * 2 ** 24)
                below = (total >> 24) * step + (((total & 0xFFFFFF) * step) >> 24)
                token = int((whole.cumsum(0) <= below).sum())
                break
        accepted.append(a)
        tokens.append([int(x) for x in drafts[s, :a]] + [token] + [-1] * (most - a))
    return accepted, tokens
