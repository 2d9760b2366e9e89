"""The speculative decoding example with linear-attention layers: after steps of drafts, verification and second calls, their states are
those that the accepted tokens alone give."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

import linear_oracle  # noqa: E402

PATH = Path(__file__).resolve().parents[1] / "examples" / "speculative_decode.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("speculative_decode_linear", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_states_hold_the_accepted_tokens(package, example):
    sequences, prompt_tokens, drafts, steps = 3, 70, 3, 10
    results = []
    for _ in range(2):
        model = example.Model(sequences, 1, prompt_tokens + (steps + 1) * (drafts + 1), sequences * prompt_tokens, vocabulary=512, linear=2)
        prompt = torch.randint(0, 512, (sequences, prompt_tokens), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
        results.append((model, *example.run(model, prompt, drafts, steps)))
    (other, *_), (model, accepted, tokens) = results
    assert torch.equal(results[0][1], accepted) and torch.equal(results[0][2], tokens)
    for mine, its in zip(model.states, other.states):
        assert all(torch.equal(a, b) for a, b in zip(mine, its))
    other.release()
    assert 0 < int(accepted.sum()) < accepted.numel() * drafts               # some drafts stay, some go
    conv_states, states = model.states[0]                                    # of the first layer: its inputs are the tokens' alone
    weights = model.linear_weights[0]
    for s in range(sequences):
        generated = [t for t in tokens[:, s].flatten().tolist() if t >= 0]
        row = torch.cat([prompt[s].cpu(), torch.tensor(generated[:-1], dtype=torch.int32)]).cuda()          # the last one drawn is not in yet
        _, normed = model.moe.rmsnorm(model.embedding[row.long()], model.norms[0])
        rows = model.moe.gemm(normed, model.linear_in[0])
        x, _, b, a = rows.split([example.CHANNELS, example.V_HEADS * 128, example.V_HEADS, example.V_HEADS], dim=1)
        where = {"slots": [0], "offsets": [0, len(row)], "lengths": [len(row)]}
        y, _, want_conv = linear_oracle.conv(x, weights["conv_weight"], conv_states[s:s + 1], where)
        q, k, v = y.bfloat16().view(len(row), -1, 128).split([example.K_HEADS, example.K_HEADS, example.V_HEADS], dim=1)
        want = linear_oracle.delta(q, k, v, a, b, weights["a_log"], weights["dt_bias"], states[s:s + 1], where)
        # a product's BF16 result may differ by a step in another call's tiles
        assert bool(((conv_states[s].double() - want_conv[0]).abs() <= want_conv[0].abs() * 2.0 ** -7 + 2.0 ** -10).all())
        assert float((states[s].double() - want["states"][0]).norm() / want["states"][0].norm()) <= 2.0 ** -6
    model.release()
