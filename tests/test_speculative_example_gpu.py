"""The speculative decoding example: what its cache holds after steps of append, attention, verification and rollback is what the
accepted tokens alone would have put there, and the attention over it is right."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

import kv_oracle  # noqa: E402

PATH = Path(__file__).resolve().parents[1] / "examples" / "speculative_decode.py"


@pytest.fixture(scope="module")
def example(package):
    spec = importlib.util.spec_from_file_location("speculative_decode", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_cache_holds_the_accepted_tokens(package, example):
    sequences, prompt_tokens, drafts, steps = 3, 70, 3, 12
    results = []
    for _ in range(2):
        model = example.Model(sequences, 1, prompt_tokens + (steps + 1) * (drafts + 1), sequences * prompt_tokens, vocabulary=512)
        prompt = torch.randint(0, 512, (sequences, prompt_tokens), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
        results.append((model, *example.run(model, prompt, drafts, steps)))
    (other, *_), (model, accepted, tokens) = results
    assert torch.equal(results[0][1], accepted) and torch.equal(results[0][2], tokens)
    other.release()
    assert 0 < int(accepted.sum()) < accepted.numel() * drafts               # some drafts stay, some go
    lengths = model.lengths.tolist()
    table = model.table.tolist()
    keys, values, key_scales, value_scales = (t.cpu().double() for t in model.pages[0])
    rotation = model.rotation.cpu()
    for s in range(sequences):
        generated = [t for t in tokens[:, s].flatten().tolist() if t >= 0]
        assert lengths[s] == prompt_tokens + int(accepted[:, s].sum()) + steps
        assert len(generated) == lengths[s] - prompt_tokens + 1              # the last one drawn is not in the cache yet
        row = torch.cat([prompt[s].cpu(), torch.tensor(generated[:-1], dtype=torch.int32)]).cuda()
        _, normed = model.moe.rmsnorm(model.embedding[row.long()], model.norms[0])
        _, _, k, v = (t.cpu() for t in model.projection(0, normed))
        for position in range(lengths[s]):
            page, slot = table[s][position // example.PAGE], position % example.PAGE
            turned = kv_oracle.rotate(k[position], rotation[position])
            # one rounding to e4m3 and, where a scale grew, others at the lower end (a page sees at most four steps' growths that
            # matter: each is a factor of two or more); a product's BF16 result may differ by a step in another call's tiles
            partner = kv_oracle.rotate(k[position].abs(), rotation[position].abs())
            for codes, scales, x, size in ((keys, key_scales, turned, k[position].double().abs().amax(-1, keepdim=True) + partner.abs()),
                                           (values, value_scales, v[position].double(), v[position].double().abs())):
                have = codes[page, :, slot] * scales[page][:, None]
                bound = x.abs() * 2.0 ** -4 + scales[page][:, None] * 4 * 2.0 ** -10 + size * 2.0 ** -7
                assert ((have - x).abs() <= bound).all()
    # the next step's attention over it
    g = torch.Generator().manual_seed(9)
    q = torch.randn(sequences, 16, 256, generator=g).bfloat16()
    batch = model.cache.batch(model.table, model.lengths, tokens=sequences)
    out = model.cache.attention(0, batch, q.cuda()).cpu().double()
    model.cache.sync()
    want, spread = kv_oracle.attention(*(t.cpu().float() for t in model.pages[0]), table, list(range(sequences + 1)), lengths, q, 1 / 16, example.PAGE)
    assert ((out - want).abs() <= want.abs() * 2.0 ** -8 + spread * (2.0 ** -8 + 2.0 ** -9)).all()
    model.release()
