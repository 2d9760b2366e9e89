"""The operators around the linear-attention layers, and the head norm and output gate of the full-attention ones, as cases that can
be timed one by one, with their plain forms.

conv       a short causal convolution over each channel of q, k and v with SiLU; the last inputs of a sequence are its state.
delta      the gated delta rule: a state of 128 x 128 for each value head that decays, is corrected along each key and is read by
           each query; one token, a few drafted ones, or chunks of prompts.  With a gate its output's heads are normed and gated.
head_norm  root mean square norm of each head, with a gate or without; or the gate alone.

Sizes: the model's linear-attention layers have 16 key heads and 32 value heads of 128, a convolution over 4 positions, and one row
of 12352 from the fused input projection: queries, keys, values, output gates, then two numbers per value head.  Its
full-attention layers have 16 query heads of 256 in a row of 9216.  Other numbers of heads stand for other models.  Prompts come
in chunks of up to 8192 tokens.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

DIM = 128                    # of a key and of a value
EPSILON = 1.0e-6             # of both norms
CHUNK = 64


def listed() -> list[dict]:
    return [
        # the smallest call: one token of one conversation
        {"name": "conv_1", "kind": "conv", "sequences": 1, "new": 1, "heads": "16/32", "width": 4, "fused": True, "fresh": False, "keep": False},
        # a decode step of 64 conversations
        {"name": "conv_64", "kind": "conv", "sequences": 64, "new": 1, "heads": "16/32", "width": 4, "fused": True, "fresh": False, "keep": False},
        # a chunk of a long prompt, the largest prefill bucket
        {"name": "conv_8192", "kind": "conv", "sequences": 1, "new": 8192, "heads": "16/32", "width": 4, "fused": True, "fresh": False, "keep": False},
        # one token of one conversation, with the norm and gate that follow
        {"name": "delta_1", "kind": "delta", "sequences": 1, "new": 1, "heads": "16/32", "fused": True, "fresh": False, "keep": False, "gated": True},
        # a decode step of 64 conversations
        {"name": "delta_64", "kind": "delta", "sequences": 64, "new": 1, "heads": "16/32", "fused": True, "fresh": False, "keep": False, "gated": True},
        # four drafted tokens and the one before them, of which some enter the state
        {"name": "delta_16x5", "kind": "delta", "sequences": 16, "new": 5, "heads": "16/32", "fused": True, "fresh": False, "keep": True, "gated": False},
        # a prompt that starts a conversation, the smallest prefill bucket
        {"name": "delta_prompt_1024", "kind": "delta", "sequences": 1, "new": 1024, "heads": "16/32", "fused": True, "fresh": True, "keep": False, "gated": True},
        # a later chunk of a long prompt, the largest prefill bucket
        {"name": "delta_chunk_8192", "kind": "delta", "sequences": 1, "new": 8192, "heads": "16/32", "fused": True, "fresh": False, "keep": False, "gated": True},
        # prompts of different, odd lengths in one call, with as many key heads as value heads
        {"name": "delta_ragged_7", "kind": "delta", "sequences": 7, "new": 1531, "heads": "16/16", "fused": False, "fresh": False, "keep": False, "gated": False},
        # the queries of a decode step of 64 conversations in a full-attention layer
        {"name": "norm_query_64", "kind": "norm", "tokens": 64, "heads": 16, "dim": 256, "norm": True, "gate": "none", "offset": 1.0, "fused": True},
        # the output of a linear-attention layer for a chunk of a prompt
        {"name": "norm_silu_8192", "kind": "norm", "tokens": 8192, "heads": 32, "dim": 128, "norm": True, "gate": "silu", "offset": 0.0, "fused": True},
        # the output gate of a full-attention layer for the same chunk
        {"name": "gate_sigmoid_8192", "kind": "norm", "tokens": 8192, "heads": 16, "dim": 256, "norm": False, "gate": "sigmoid", "offset": 0.0, "fused": True},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["conv", "conv", "delta", "delta", "delta", "delta", "norm", "norm"])
    if kind == "norm":
        gate = rng.choice(["none", "silu", "sigmoid"])
        case = {"kind": kind, "tokens": _log_int(rng, 1, 8192), "heads": rng.choice([2, 4, 16, 31, 32]), "dim": rng.choice([64, 128, 256]),
                "norm": gate == "none" or rng.random() < 0.7, "gate": gate, "offset": rng.choice([0.0, 1.0]), "fused": rng.random() < 0.5}
        case["tokens"] = min(case["tokens"], 8192 * 4096 // (case["heads"] * case["dim"]))
        return case
    case = {"kind": kind, "heads": rng.choice(["16/32", "16/32", "16/16", "4/12", "2/8"]), "fused": rng.random() < 0.5,
            "fresh": rng.random() < 0.3, "keep": rng.random() < 0.3}
    form = rng.choice(["token", "token", "drafts", "prompt", "prompt"])
    if form == "token":
        case.update(sequences=_log_int(rng, 1, 64), new=1)
    elif form == "drafts":
        case.update(sequences=_log_int(rng, 1, 32), new=rng.randint(2, 8))
    else:
        sequences = rng.choice([1, 1, 2, 3, 5])
        case.update(sequences=sequences, new=_log_int(rng, 9, 8192 // sequences))
    if kind == "conv":
        case["width"] = rng.choice([4, 4, 3, 2])
    else:
        case["gated"] = rng.random() < 0.5
    return case


def _new(case: dict) -> list[int]:
    """New tokens of each sequence: the case's own, down to half of them."""
    count = case["sequences"]
    return [max(1, case["new"] - (i * case["new"]) // (2 * count)) for i in range(count)]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 31)

    def normal(*shape: int, std: float = 1.0) -> torch.Tensor:
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, std, generator=g)

    state: dict = {"kind": case["kind"]}
    if case["kind"] == "norm":
        tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
        # of a fused projection's row, per head: what is normed or the attention's gate, and its neighbour
        row = normal(tokens, heads, 2 * dim) if case["fused"] else None
        state["x"] = row[:, :, :dim] if case["fused"] and case["gate"] == "none" else normal(tokens, heads, dim)
        state["gate"] = None if case["gate"] == "none" else row[:, :, dim:] if case["fused"] else normal(tokens, heads, dim)
        state["weight"] = normal(dim, std=0.1) + (1.0 - case["offset"]) if case["norm"] else None
        state.update(activation=case["gate"], offset=case["offset"])
        return state

    k_heads, v_heads = (int(x) for x in case["heads"].split("/"))
    new = _new(case)
    count, tokens, channels = len(new), sum(new), (2 * k_heads + v_heads) * DIM
    state.update(k_heads=k_heads, v_heads=v_heads, new=max(new), tokens=tokens,
                 offsets=torch.tensor([sum(new[:i]) for i in range(count + 1)], dtype=torch.int32, device="cuda"),
                 slots=torch.randperm(count + 3, device="cuda", generator=g)[:count].int(), keep=None)
    earlier = torch.zeros(count, dtype=torch.int32, device="cuda")
    if not case["fresh"]:
        earlier = torch.randint(1, 32768, (count,), device="cuda", generator=g, dtype=torch.int32)
        earlier[1:3] = 0            # some of a batch start with this call
    rows = state["offsets"][1:] - state["offsets"][:-1]
    state["lengths"] = earlier + rows
    if case["keep"]:
        state["keep"] = (torch.rand(count, device="cuda", generator=g) * (rows + 1)).int()
    # one row of the fused projection: queries, keys and values, the output's gates, then two numbers per value head
    width = channels + v_heads * DIM + 2 * v_heads
    row = normal(tokens, width) if case["fused"] else None
    if case["kind"] == "conv":
        state["x"] = row[:, :channels] if case["fused"] else normal(tokens, channels)
        state["weight"] = normal(channels, case["width"], std=0.5)
        state["conv_states"] = normal(count + 3, case["width"] - 1, channels)
    else:
        x = torch.nn.functional.silu(normal(tokens, channels))       # what the convolution gives
        if not case["fused"]:
            x = x.view(tokens, -1, DIM).transpose(0, 1).contiguous().transpose(0, 1)          # heads first
        else:
            x = x.view(tokens, -1, DIM)
        state["q"], state["k"], state["v"] = x.split([k_heads, k_heads, v_heads], dim=1)
        ab = row[:, channels + v_heads * DIM:] if case["fused"] else normal(tokens, 2 * v_heads)
        state["b"], state["a"] = ab[:, :v_heads], ab[:, v_heads:]
        state["a_log"] = torch.empty(v_heads, device="cuda").uniform_(0.01, 16.0, generator=g).log()
        step = torch.exp(torch.empty(v_heads, device="cuda").uniform_(math.log(0.001), math.log(0.1), generator=g))
        state["dt_bias"] = step + torch.log(-torch.expm1(-step))
        state["gate"] = None
        if case["gated"]:
            state["gate"] = row[:, channels:channels + v_heads * DIM].view(tokens, v_heads, DIM) if case["fused"] else normal(tokens, v_heads, DIM)
        state["norm_weight"] = normal(DIM, std=0.1) + 1.0
        state["states"] = torch.empty(count + 3, v_heads, DIM, DIM, device="cuda").normal_(0.0, 0.1, generator=g)
    if own:                       # the handle that a serving process keeps; the inputs are the same
        aima = importlib.import_module("aima-amd395-qwen36-35b-linux-engine_b200")
        layer = aima.LinearAttention(k_heads=k_heads, v_heads=v_heads, conv_width=case.get("width", 4), slots=count + 3,
                                     max_sequences=count, max_tokens=tokens)
        if case["kind"] == "conv":
            layer.bind_layer(0, conv_weight=state["weight"], conv_states=state["conv_states"])
        else:
            layer.bind_layer(0, a_log=state["a_log"], dt_bias=state["dt_bias"], norm_weight=state["norm_weight"], states=state["states"])
        state["layer"] = layer
        state["batch"] = layer.batch(state["slots"], tokens=tokens, lengths=state["lengths"], row_offsets=state["offsets"],
                                     max_new_tokens=max(new), keep=state["keep"])
    return state


def run(state: dict):
    if state["kind"] == "norm":
        if own:
            aima = importlib.import_module("aima-amd395-qwen36-35b-linux-engine_b200")
            return aima.head_norm(state["x"], state["weight"], offset=state["offset"], gate=state["gate"], activation=state["activation"],
                                  eps=EPSILON)
        return _plain_norm(state["x"].float(), state["weight"], state["offset"], state["gate"], state["activation"]).bfloat16()
    if state["kind"] == "conv":
        out = state["layer"].conv(0, state["batch"], state["x"]) if own else _plain_conv(state)
        return {"out": out, "conv_states": state["conv_states"]}
    if own:
        out = state["layer"].delta(0, state["batch"], state["q"], state["k"], state["v"], state["a"], state["b"], gate=state["gate"])
    else:
        out = _plain_delta(state)
    return {"out": out, "states": state["states"]}


# -- plain forms ------------------------------------------------------------------------------------------------------------

def _activation(x: torch.Tensor, name: str) -> torch.Tensor:
    return x * torch.sigmoid(x) if name == "silu" else torch.sigmoid(x)


def _plain_norm(x: torch.Tensor, weight, offset: float, gate, activation: str) -> torch.Tensor:
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * (weight.float() + offset)
    return x if gate is None else x * _activation(gate.float(), activation)


def _places(state: dict):
    """Sequence of every row, and which of its rows it is."""
    row = torch.arange(state["tokens"], device="cuda")
    offsets = state["offsets"].long()
    sequence = torch.searchsorted(offsets[1:], row, right=True)
    return sequence, row - offsets[sequence]


def _counts(state: dict):
    """Rows of every sequence, those that enter its state, and whether it starts with them."""
    rows = (state["offsets"][1:] - state["offsets"][:-1]).long()
    return rows, rows if state["keep"] is None else state["keep"].long(), state["lengths"].long() <= rows


def _plain_conv(state: dict) -> torch.Tensor:
    sequence, at = _places(state)
    rows, kept, starts = _counts(state)
    weight, slots = state["weight"].float(), state["slots"].long()
    channels, width = weight.shape
    count = rows.numel()
    x = torch.zeros(count, width - 1 + state["new"], channels, device="cuda")
    x[:, :width - 1] = torch.where(starts[:, None, None], 0.0, state["conv_states"][slots].float())
    x[sequence, width - 1 + at] = state["x"].float()
    y = sum(x[:, j:j + state["new"]] * weight[:, j] for j in range(width))
    last = kept[:, None] + torch.arange(width - 1, device="cuda")
    after = x.gather(1, last[..., None].expand(-1, -1, channels)).bfloat16()
    state["conv_states"][slots] = torch.where((kept > 0)[:, None, None], after, state["conv_states"][slots])
    return _activation(y, "silu")[sequence, at].bfloat16()


def _plain_delta(state: dict) -> torch.Tensor:
    sequence, at = _places(state)
    rows, kept, starts = _counts(state)
    count, v_heads, slots = rows.numel(), state["v_heads"], state["slots"].long()
    chunk = min(CHUNK, state["new"])
    chunks = (state["new"] + chunk - 1) // chunk

    def spread(x: torch.Tensor) -> torch.Tensor:
        """Rows [tokens, v_heads, ...] by sequence, head, chunk and place in it, zeros where a sequence has fewer."""
        out = torch.zeros(count, chunks * chunk, *x.shape[1:], dtype=x.dtype, device="cuda")
        out[sequence, at] = x
        return out.transpose(1, 2).unflatten(2, (chunks, chunk))

    def unit(x: torch.Tensor) -> torch.Tensor:
        x = x.float()
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPSILON)
        return spread(x.repeat_interleave(v_heads // x.shape[1], dim=1))

    q, k, v = unit(state["q"]) * DIM ** -0.5, unit(state["k"]), spread(state["v"].float())
    step = state["a"].float() + state["dt_bias"]
    g = spread(-state["a_log"].exp() * (step.clamp_min(0.0) + torch.log1p(torch.exp(-step.abs())))).double()
    beta = spread(torch.sigmoid(state["b"].float()))
    before = torch.where(starts[:, None, None, None], 0.0, state["states"][slots])

    def passes(beta: torch.Tensor, g: torch.Tensor, outputs: bool):
        total = g.cumsum(-1)
        lower = torch.ones(chunk, chunk, dtype=torch.bool, device="cuda").tril()
        decay = torch.where(lower, (total[..., :, None] - total[..., None, :]), -math.inf).float().exp()      # from a column's token to a row's
        overlap = (beta[..., None] * (k @ k.transpose(-1, -2)) * decay).tril(-1)
        inverse = torch.eye(chunk, device="cuda").expand_as(overlap).clone()              # of 1 + overlap, row by row
        for i in range(1, chunk):
            inverse[..., i, :i] = -(overlap[..., i, None, :i] @ inverse[..., :i, :i]).squeeze(-2)
        fresh = inverse @ (beta[..., None] * v)
        known = inverse @ ((beta * total.exp().float())[..., None] * k)
        within = (q @ k.transpose(-1, -2)) * decay
        reach, left = total.exp().float()[..., None], (total[..., -1:] - total).exp().float()[..., None]
        s, outs = before, []
        for c in range(chunks):
            d = fresh[:, :, c] - known[:, :, c] @ s
            if outputs:
                outs.append((q[:, :, c] * reach[:, :, c]) @ s + within[:, :, c] @ d)
            s = s * reach[:, :, c, -1:] + (k[:, :, c] * left[:, :, c]).transpose(-1, -2) @ d
        return torch.cat(outs, dim=2) if outputs else None, s

    out, after = passes(beta, g, True)
    if state["keep"] is not None:            # the state without the rows that do not stay
        place = torch.arange(chunks * chunk, device="cuda").view(chunks, chunk)
        stays = (place < kept[:, None, None])[:, None]
        _, after = passes(beta * stays, g * stays, False)
    state["states"][slots] = torch.where((kept > 0)[:, None, None, None], after, state["states"][slots])
    out = out.transpose(1, 2)[sequence, at]
    if state["gate"] is not None:
        out = _plain_norm(out, state["norm_weight"], 0.0, state["gate"], "silu")
    return out.bfloat16()


# -- 64 bits, from the definitions --------------------------------------------------------------------------------------------

def _exact_norm(s: dict) -> torch.Tensor:
    x = s["x"].double()
    if s["weight"] is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPSILON) * (s["weight"].double() + s["offset"])
    if s["gate"] is not None:
        z = s["gate"].double()
        x = x * (z if s["activation"] == "silu" else 1.0) / (1.0 + torch.exp(-z))
    return x


def _exact_conv(case: dict, s: dict) -> dict:
    width, outs, states, row = case["width"], [], s["conv_states"].double(), 0
    for i, n in enumerate(_new(case)):
        slot = int(s["slots"][i])
        before = states[slot] * (0.0 if int(s["lengths"][i]) == n else 1.0)
        x = torch.cat([before, s["x"][row:row + n].double()])
        y = torch.zeros_like(x[:n])
        for j in range(width):
            y += x[j:j + n] * s["weight"][:, j].double()
        outs.append(y / (1.0 + torch.exp(-y)))
        kept = n if s["keep"] is None else int(s["keep"][i])
        if kept > 0:
            states[slot] = x[kept:kept + width - 1]
        row += n
    return {"out": torch.cat(outs), "conv_states": states}


def _exact_delta(case: dict, s: dict) -> dict:
    """One token after the other, all sequences that still have one at once."""
    new = _new(case)
    k_heads, v_heads = s["k_heads"], s["v_heads"]
    group, first, slots = v_heads // k_heads, s["offsets"].tolist(), s["slots"].long()
    kept = new if s["keep"] is None else s["keep"].tolist()
    memory = s["states"].double()[slots]
    for i, n in enumerate(new):
        if int(s["lengths"][i]) == n:
            memory[i] = 0.0
    states, out = s["states"].double(), torch.empty(s["tokens"], v_heads, DIM, dtype=torch.float64, device="cuda")
    a, b = s["a"].double() + s["dt_bias"].double(), s["b"].double()
    decay = torch.exp(-torch.exp(s["a_log"].double()) * torch.logaddexp(a, torch.zeros_like(a)))
    rate = 1.0 / (1.0 + torch.exp(-b))
    q, k = ((x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPSILON)).repeat_interleave(group, dim=1) for x in (s["q"].double(), s["k"].double()))
    v = s["v"].double()
    for t in range(max(new)):
        active = [i for i, n in enumerate(new) if t < n]                # the first ones: no sequence has more rows than one before it
        rows = slice(first[0] + t, first[0] + t + 1) if len(active) == 1 else [first[i] + t for i in active]
        m = memory[:len(active)]
        m *= decay[rows][..., None, None]
        key = k[rows][..., None]
        m += key * (rate[rows][..., None] * (v[rows] - (m * key).sum(-2)))[..., None, :]
        out[rows] = (m * q[rows][..., None]).sum(-2) / math.sqrt(DIM)
        for i in active:
            if t + 1 == kept[i]:
                states[slots[i]] = memory[i]
    if s["gate"] is not None:
        out = _exact_norm({"x": out, "weight": s["norm_weight"], "offset": 0.0, "gate": s["gate"], "activation": "silu"})
    return {"out": out, "states": states}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(s)
    return _exact_conv(case, s) if case["kind"] == "conv" else _exact_delta(case, s)


def work(case: dict) -> dict:
    if case["kind"] == "norm":
        size = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": size * (4 if case["gate"] == "none" else 6) + case["dim"] * 2 * case["norm"], "flops": size * 8}
    k_heads, v_heads = (int(x) for x in case["heads"].split("/"))
    count, tokens, channels = case["sequences"], sum(_new(case)), (2 * k_heads + v_heads) * DIM
    read = 0 if case["fresh"] else max(1, count - 2) if count > 1 else 1           # states that are read
    if case["kind"] == "conv":
        return {"bytes": channels * (4 * tokens + 2 * case["width"] + 2 * (case["width"] - 1) * (read + count)), "flops": tokens * channels * (2 * case["width"] + 4)}
    bytes_ = tokens * (2 * channels + 2 * v_heads * (DIM + 2) + (2 * v_heads * DIM if case["gated"] else 0)) + 4 * v_heads * DIM * DIM * (read + count)
    return {"bytes": bytes_, "flops": tokens * v_heads * 7 * DIM * DIM}
