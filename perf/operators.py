"""The operators around the full-attention layers' cache, as cases that can be timed one by one, with their plain forms.

kv_append     rotates the new keys (and queries) by their positions and stores keys and values in a paged cache of 8-bit floating
              point numbers (e4m3) with one power-of-two scale for each page and head.
kv_attention  attention of the new queries over that cache: one token, a few drafted ones, or whole chunks of prompts.
verify        accepts or rejects drafted tokens against the target's probabilities and draws the token that follows.

Sizes: the model's full-attention layers have 16 query heads and 2 key/value heads of 256 with 64 rotated elements, and their
queries, gates, keys and values come as one row of 9216 from the fused input projection; 32/8 heads of 128 and 8/8 heads of
64 stand for other models.  Prompts come in chunks of up to 8192 tokens, the vocabulary has 248 320 entries.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

VOCAB = 248320
MAX_EXPONENT, MIN_EXPONENT = 119, -64        # of a scale
LARGEST = 448.0                              # of e4m3


def listed() -> list[dict]:
    return [
        # the smallest call: one token of one conversation joins the cache of one layer
        {"name": "append_1", "kind": "append", "sequences": 1, "new": 1, "length": 1000, "page": 64, "heads": "16/2/256", "fused": True},
        # a decode step of 64 conversations of different lengths
        {"name": "append_64", "kind": "append", "sequences": 64, "new": 1, "length": 2111, "page": 64, "heads": "16/2/256", "fused": True},
        # one chunk of a long prompt, the largest prefill bucket
        {"name": "append_8192", "kind": "append", "sequences": 1, "new": 8192, "length": 16384, "page": 64, "heads": "16/2/256", "fused": True},
        # one token of one conversation with a long context
        {"name": "attend_1x32768", "kind": "attend", "sequences": 1, "new": 1, "length": 32768, "page": 64, "heads": "16/2/256"},
        # a decode step of 64 conversations, up to 8192 tokens each
        {"name": "attend_64x8192", "kind": "attend", "sequences": 64, "new": 1, "length": 8192, "page": 64, "heads": "16/2/256"},
        # four drafted tokens and the one before them, odd lengths, small pages
        {"name": "attend_16x5", "kind": "attend", "sequences": 16, "new": 5, "length": 4111, "page": 16, "heads": "16/2/256"},
        # a prompt that starts a conversation, the smallest prefill bucket
        {"name": "attend_prompt_1024", "kind": "attend", "sequences": 1, "new": 1024, "length": 1024, "page": 64, "heads": "16/2/256"},
        # the last chunk of a prompt of 32768 tokens
        {"name": "attend_chunk_8192", "kind": "attend", "sequences": 1, "new": 8192, "length": 32768, "page": 64, "heads": "16/2/256"},
        # prompts of different, odd lengths in one call, with the heads of another model
        {"name": "attend_ragged_7", "kind": "attend", "sequences": 7, "new": 1531, "length": 2999, "page": 128, "heads": "32/8/128"},
        # one conversation's drafts from a lookup, so without probabilities of their own
        {"name": "verify_1x4", "kind": "verify", "sequences": 1, "drafts": 4, "vocab": VOCAB, "probabilities": False},
        # 32 conversations with a draft model
        {"name": "verify_32x5", "kind": "verify", "sequences": 32, "drafts": 5, "vocab": VOCAB, "probabilities": True},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "verify", "verify"])
    if kind == "verify":
        return {"kind": kind, "sequences": _log_int(rng, 1, 32), "drafts": rng.randint(1, 7), "vocab": _log_int(rng, 1000, VOCAB),
                "probabilities": rng.random() < 0.6}
    case = {"kind": kind, "page": rng.choice([16, 32, 64, 128]), "heads": rng.choice(["16/2/256", "16/2/256", "32/8/128", "8/8/64"])}
    form = rng.choice(["token", "token", "drafts", "prompt", "prompt"])
    if form == "token":
        case.update(sequences=_log_int(rng, 1, 64), new=1)
    elif form == "drafts":
        case.update(sequences=_log_int(rng, 1, 32), new=rng.randint(2, 8))
    else:
        case.update(sequences=rng.choice([1, 1, 2, 3, 5]), new=_log_int(rng, 9, 4096))
    total = 65536 if form == "prompt" else 262144
    most = min(32768, total // case["sequences"])
    if form == "prompt":
        most = min(most, (1 << 27) // (case["sequences"] * case["new"]))
    case["length"] = max(case["new"], _log_int(rng, 1, most))
    if kind == "append":
        case["fused"] = rng.random() < 0.5
    return case


def _shape(case: dict) -> tuple[int, int, int, int]:
    q_heads, kv_heads, dim = (int(x) for x in case["heads"].split("/"))
    return q_heads, kv_heads, dim, min(64, dim)


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and tokens in the cache with them, of each sequence: the case's own, down to half of them."""
    count = case["sequences"]
    new = [max(1, case["new"] - (i * case["new"]) // (2 * count)) for i in range(count)]
    length = [max(n, case["length"] - (i * case["length"]) // (2 * count)) for i, n in enumerate(new)]
    return new, length


def _rotation(positions: int, rotary: int) -> torch.Tensor:
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * (1.0e7 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary))
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 29)
    state: dict = {"kind": case["kind"]}
    if case["kind"] == "verify":
        count, drafts, vocab = case["sequences"], case["drafts"], case["vocab"]
        logits = torch.empty(count, drafts + 1, vocab, device="cuda").normal_(0.0, 3.0, generator=g)
        state["target"] = torch.softmax(logits, dim=-1)
        draft = torch.softmax(logits[:, :drafts] + 0.5 * torch.empty(count, drafts, vocab, device="cuda").normal_(generator=g), dim=-1)
        # a lookup's drafts are often right: the likeliest token; a draft model's are drawn from its probabilities
        state["drafts"] = (torch.multinomial(draft.view(-1, vocab), 1, generator=g).view(count, drafts) if case["probabilities"]
                           else logits[:, :drafts].argmax(-1)).int()
        state["draft"] = draft if case["probabilities"] else None
        state["uniforms"] = torch.rand(count, drafts + 1, device="cuda", generator=g)
        if not case["probabilities"]:
            state["uniforms"][:, :drafts] *= state["target"].amax(-1)[:, :drafts] * 1.5
        state["lengths"] = torch.randint(drafts + 1, 32768, (count,), device="cuda", generator=g, dtype=torch.int32)
        return state

    q_heads, kv_heads, dim, rotary = _shape(case)
    page = case["page"]
    new, length = _lengths(case)
    pages = [(n + page - 1) // page for n in length]
    total = sum(pages)
    order = torch.randperm(total, device="cuda", generator=g).int()        # pages are given out in no order
    table = torch.zeros(len(pages), max(pages), dtype=torch.int32, device="cuda")
    first = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[first:first + n]
        first += n
    state.update(page=page, dim=dim, scale=dim ** -0.5, table=table, new=max(new),
                 offsets=torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda"),
                 lengths=torch.tensor(length, dtype=torch.int32, device="cuda"))
    for name in ("keys", "values"):
        codes = torch.empty(total, kv_heads, page, dim, device="cuda").normal_(0.0, 64.0, generator=g).clamp_(-LARGEST, LARGEST)
        state[name] = codes.to(torch.float8_e4m3fn)
        state[name[:-1] + "_scales"] = torch.exp2(-torch.randint(5, 8, (total, kv_heads), device="cuda", generator=g).float())
    tokens = sum(new)
    if case["kind"] == "append":
        if case.get("fused"):      # one row of the fused projection: per query head its query and its gate, then keys, then values
            row = torch.empty(tokens, (2 * q_heads + 2 * kv_heads) * dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
            state["q"] = row[:, :2 * q_heads * dim].view(tokens, q_heads, 2 * dim)[:, :, :dim]
            state["k"], state["v"] = row[:, 2 * q_heads * dim:].view(tokens, 2, kv_heads, dim).unbind(1)
        else:
            state["q"] = torch.empty(tokens, q_heads, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
            state["k"] = torch.empty(tokens, kv_heads, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
            state["v"] = torch.empty(tokens, kv_heads, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        state["k"][..., ::37] *= 4          # a few channels of the keys are large
        state["rotation"] = _rotation(max(length), rotary)
    else:
        state["q"] = torch.empty(tokens, q_heads, dim, dtype=torch.bfloat16, device="cuda").normal_(0.0, 1.5, generator=g)
    if own:                       # the handle that a serving process keeps; the inputs are the same
        aima = importlib.import_module("aima-amd395-qwen36-35b-linux-engine_b200")
        cache = aima.KvCache(q_heads=q_heads, kv_heads=kv_heads, head_dim=dim, page_tokens=page, pages=total, rotary_dim=rotary,
                             max_sequences=len(new))
        cache.bind_layer(0, state["keys"], state["values"], state["key_scales"], state["value_scales"])
        if case["kind"] == "append":
            cache.set_rotation(state["rotation"])
        state["cache"] = cache
        state["batch"] = cache.batch(table, state["lengths"], tokens=tokens, row_offsets=state["offsets"], max_new_tokens=max(new))
    return state


def run(state: dict):
    if state["kind"] == "verify":
        if own:
            aima = importlib.import_module("aima-amd395-qwen36-35b-linux-engine_b200")
            return aima.verify_drafts(state["target"], state["drafts"], state["uniforms"], draft_probabilities=state["draft"],
                                      cache_lengths=state["lengths"])
        return _plain_verify(state)
    if state["kind"] == "append":
        if own:
            q = state["cache"].append(0, state["batch"], state["k"], state["v"], q=state["q"])
        else:
            q = _plain_append(state)
        return {"q": q, **{name: state[name] for name in ("keys", "values", "key_scales", "value_scales")}}
    if own:
        return state["cache"].attention(0, state["batch"], state["q"])
    return _plain_attention(state)


# -- plain forms ------------------------------------------------------------------------------------------------------------

def _places(state: dict, tokens: int):
    """Sequence and position of every new row."""
    row = torch.arange(tokens, device="cuda")
    offsets = state["offsets"].long()
    sequence = torch.searchsorted(offsets[1:], row, right=True)
    first = state["lengths"].long() - (offsets[1:] - offsets[:-1])
    return sequence, first[sequence] + row - offsets[sequence]


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], dim=-1)


def _exponent(amax: torch.Tensor) -> torch.Tensor:
    """The least e with amax <= 448 * 2^e."""
    mantissa, exponent = torch.frexp(amax)
    return (exponent - 9 + (mantissa > 0.875).int()).clamp(MIN_EXPONENT, MAX_EXPONENT).masked_fill(amax == 0, MIN_EXPONENT)


def _codes(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_append(state: dict) -> torch.Tensor:
    tokens, kv_heads, dim = state["k"].shape
    sequence, position = _places(state, tokens)
    cos, sin = state["rotation"][position].unsqueeze(1).chunk(2, dim=-1)
    q = _rotate(state["q"].float(), cos, sin).bfloat16()
    k, v = _rotate(state["k"].float(), cos, sin), state["v"].float()
    sound = (torch.isfinite(k) & torch.isfinite(v)).all(-1)                 # [tokens, heads]
    page, slot = state["table"][sequence, position // state["page"]].long(), position % state["page"]
    # the page that a sequence's first new token goes to holds older ones, unless the token is its first
    begin = state["lengths"].long() - (state["offsets"][1:] - state["offsets"][:-1]).long()
    opened, held = state["table"].gather(1, (begin // state["page"])[:, None]).long()[:, 0], begin % state["page"]
    older = torch.arange(state["page"], device="cuda")[None, None, :, None] < held[:, None, None, None]
    for name, x in (("key", k), ("value", v)):
        codes, scales = state[name + "s"].view(torch.uint8), state[name + "_scales"]
        amax = torch.where(sound, x.abs().amax(-1), 0.0)
        highest = torch.zeros_like(scales).scatter_reduce_(0, page[:, None].expand(-1, kv_heads), amax, "amax")
        exponent = _exponent(highest)
        before = scales[opened]
        grown = torch.where((held > 0)[:, None], torch.maximum(exponent[opened], torch.frexp(before)[1] - 1), exponent[opened])
        exponent[opened] = grown
        written = torch.zeros(scales.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, page, True)
        # older tokens of a page whose scale grew
        ratio = (before / torch.exp2(grown.float()))[..., None, None]
        kept = _codes(state[name + "s"].view(torch.uint8)[opened].view(torch.float8_e4m3fn).float() * ratio)
        codes[opened] = torch.where(older, kept, codes[opened])
        scales.copy_(torch.where(written[:, None], torch.exp2(exponent.float()), scales))
        fresh = _codes(torch.where(sound[..., None], x, 0.0) * torch.exp2(-exponent.float())[page][..., None])
        if name == "key":
            fresh = torch.where(sound[..., None], fresh, torch.full_like(fresh, 0x7F))
        codes[page, :, slot] = fresh
    return q


def _plain_attention(state: dict) -> torch.Tensor:
    tokens, q_heads, dim = state["q"].shape
    kv_heads, page = state["keys"].shape[1], state["page"]
    count, columns = state["table"].shape
    group, span = q_heads // kv_heads, columns * page
    table, lengths = state["table"].long(), state["lengths"].long()

    def gather(name):
        x = state[name + "s"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * state[name + "_scales"][table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(count, kv_heads, span, dim)

    sequence, position = _places(state, tokens)
    at = torch.arange(tokens, device="cuda") - state["offsets"].long()[sequence]
    q = torch.zeros(count, state["new"], q_heads, dim, device="cuda")
    q[sequence, at] = state["q"].float()
    q = q.view(count, state["new"], kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(count, kv_heads, group * state["new"], dim)
    where = torch.full((count, state["new"]), -1, dtype=torch.long, device="cuda")
    where[sequence, at] = position
    column = torch.arange(span, device="cuda")
    hidden = column > where[:, :, None]                                                  # [count, new, span]
    s = torch.matmul(q, gather("key").transpose(2, 3)).mul_(state["scale"])
    s.view(count, kv_heads, group, state["new"], span).masked_fill_(hidden[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    weight = p.sum(-1, keepdim=True)
    v = gather("value").masked_fill_((column >= lengths[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(p, v) / weight.masked_fill(weight == 0.0, 1.0)
    out = out.view(count, kv_heads, group, state["new"], dim).permute(0, 3, 1, 2, 4).reshape(count, state["new"], q_heads, dim)
    return out[sequence, at].bfloat16()


def _plain_verify(state: dict):
    target, drafts, uniforms, draft = state["target"], state["drafts"].long(), state["uniforms"], state["draft"]
    count, most = drafts.shape
    p = target[:, :most].gather(2, drafts[..., None])[..., 0]
    q = draft.gather(2, drafts[..., None])[..., 0] if draft is not None else torch.ones_like(p)
    accepted = (uniforms[:, :most] * q < p).long().cumprod(1).sum(1)
    each = torch.arange(count, device="cuda")
    row, last = target[each, accepted], (accepted == most)[:, None]
    at = accepted.clamp(max=most - 1)
    if draft is not None:
        rest = (row - draft[each, at].masked_fill(last, 0.0)).clamp_min_(0.0)
    else:
        rest = row.scatter(1, drafts.gather(1, at[:, None]), row.gather(1, drafts.gather(1, at[:, None])) * last)
    whole = (rest * 2.0 ** 40).long()
    whole = torch.where(whole.sum(1, keepdim=True) == 0, (row * 2.0 ** 40).long(), whole)
    sums = whole.cumsum(1)
    total, u = sums[:, -1], (uniforms[:, most] * 2.0 ** 24).long()
    below = (total >> 24) * u + (((total & 0xFFFFFF) * u) >> 24)
    token = (sums <= below[:, None]).sum(1)
    step = torch.arange(most + 1, device="cuda")
    tokens = torch.where(step < accepted[:, None], torch.nn.functional.pad(drafts, (0, 1)),
                         torch.where(step == accepted[:, None], token[:, None], -1))
    return accepted.int(), tokens.int(), (state["lengths"] - most + accepted).int()


# -- 64 bits, from the definitions --------------------------------------------------------------------------------------------

def _e4m3(x: torch.Tensor) -> torch.Tensor:
    """x rounded to the nearest multiple of its binade's step (three bits after the leading one, 2^-9 at the least), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(x / step) * step


def _exact_append(case: dict, seed: int) -> dict:
    s = prepare(case, seed)
    new, length = _lengths(case)
    kv_heads, rotary, page = s["k"].shape[1], s["rotation"].shape[1], s["page"]
    half, table = rotary // 2, s["table"].cpu()
    out = {name: s[name].to(torch.float64) for name in ("keys", "values", "key_scales", "value_scales")}
    rotated, row = [], 0
    for b, (n, total) in enumerate(zip(new, length)):
        angle = s["rotation"][total - n:total].double()
        c, d = angle[:, None, :half], angle[:, None, half:]

        def turn(x):
            y = x.double().clone()
            y[..., :half] = x[..., :half].double() * c - x[..., half:rotary].double() * d
            y[..., half:rotary] = x[..., half:rotary].double() * c + x[..., :half].double() * d
            return y

        rotated.append(turn(s["q"][row:row + n]))
        k, v = turn(s["k"][row:row + n]), s["v"][row:row + n].double()
        first = (total - n) // page
        for column in range(first, (total - 1) // page + 1):
            low, high = max(total - n, column * page), min(total, (column + 1) * page)
            at, from_, to = int(table[b, column]), low - column * page, high - column * page
            for name, x in (("key", k), ("value", v)):
                piece = x[low - (total - n):high - (total - n)].transpose(0, 1)           # [heads, rows, dim]
                scale = torch.exp2(torch.ceil(torch.log2(piece.abs().amax((1, 2)) / LARGEST)))
                if from_ > 0:
                    old = out[name + "_scales"][at].clone()
                    scale = torch.maximum(scale, old)
                    out[name + "s"][at, :, :from_] = _e4m3(out[name + "s"][at, :, :from_] * (old / scale)[:, None, None])
                out[name + "s"][at, :, from_:to] = _e4m3(piece / scale[:, None, None])
                out[name + "_scales"][at] = scale
        row += n
    return {"q": torch.cat(rotated), **out}


def _exact_attention(case: dict, seed: int) -> torch.Tensor:
    s = prepare(case, seed)
    new, length = _lengths(case)
    q_heads, kv_heads, dim, _ = _shape(case)
    group, page, row, outs = q_heads // kv_heads, s["page"], 0, []
    for b, (n, total) in enumerate(zip(new, length)):
        pages = s["table"][b, :(total + page - 1) // page].long()
        k, v = ((s[name + "s"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * s[name + "_scales"][pages].double()[..., None, None])
                .transpose(0, 1).reshape(kv_heads, -1, dim)[:, :total] for name in ("key", "value"))
        out = torch.empty(n, q_heads, dim, dtype=torch.float64, device="cuda")
        for low in range(0, n, 512):
            high = min(n, low + 512)
            seen = total - n + torch.arange(low, high, device="cuda")
            for h in range(q_heads):
                scores = (s["q"][row + low:row + high, h].double() @ k[h // group].T) / math.sqrt(dim)
                scores[torch.arange(total, device="cuda")[None, :] > seen[:, None]] = -math.inf
                out[low:high, h] = torch.softmax(scores, -1) @ v[h // group]
        outs.append(out)
        row += n
    return torch.cat(outs)


def exact(case: dict, seed: int):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    if case["kind"] == "attend":
        return _exact_attention(case, seed)
    return None            # whole numbers


def work(case: dict) -> dict:
    if case["kind"] == "verify":
        # per sequence the drafts' own probabilities, then one row of the target's and, at a rejected draft, of the draft's
        rows = 1 + (1 if case["probabilities"] else 0)
        return {"bytes": case["sequences"] * (rows * case["vocab"] * 4 + case["drafts"] * 16), "flops": case["sequences"] * case["vocab"] * 4}
    q_heads, kv_heads, dim, rotary = _shape(case)
    new, length = _lengths(case)
    tokens = sum(new)
    if case["kind"] == "append":
        pages = sum((n - 1) // case["page"] - (n - m) // case["page"] + 1 for m, n in zip(new, length))
        return {"bytes": tokens * (4 * q_heads * dim + 6 * kv_heads * dim + 4 * rotary) + pages * (4 + 16 * kv_heads),
                "flops": tokens * (3 * rotary * (q_heads + kv_heads) + 4 * kv_heads * dim)}
    pairs = sum(m * n - m * (m - 1) // 2 for m, n in zip(new, length))
    return {"bytes": sum(length) * 2 * kv_heads * dim + sum((n + case["page"] - 1) // case["page"] for n in length) * (4 + 8 * kv_heads)
            + 4 * tokens * q_heads * dim, "flops": 4 * q_heads * dim * pairs}
