"""GPU parity of the verification of drafted tokens through the C ABI: accepted counts, tokens and lengths equal those of
oracle/kv_oracle.py (whole numbers throughout, so there is no tolerance)."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import kv_oracle  # noqa: E402


def _case(sequences, drafts, vocabulary, seed, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(sequences, drafts + 1, vocabulary, generator=g) * sharp
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits[:, :drafts] + torch.randn(sequences, drafts, vocabulary, generator=g) * 0.5, -1)
    tokens = torch.multinomial(draft.reshape(-1, vocabulary), 1, generator=g).view(sequences, drafts).int() if drafts else torch.zeros(sequences, 0, dtype=torch.int32)
    return target, draft, tokens, torch.rand(sequences, drafts + 1, generator=g), g


def _check(package, target, tokens, uniforms, draft=None, counts=None, gpu=None):
    lengths = torch.arange(100, 100 + target.shape[0], dtype=torch.int32)
    want, wish = kv_oracle.verify(target, tokens, uniforms, draft, counts)
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    big = gpu or (up(target), up(draft))
    accepted, out, new = package.verify_drafts(big[0], up(tokens), up(uniforms), draft_probabilities=big[1], draft_counts=up(counts),
                                               cache_lengths=lengths.cuda())
    assert accepted.tolist() == want and out.tolist() == wish
    n = [tokens.shape[1]] * len(want) if counts is None else [min(max(int(c), 0), tokens.shape[1]) for c in counts]
    assert new.tolist() == [int(l) - (c - a) for l, c, a in zip(lengths, n, want)]
    return want, wish


@pytest.mark.parametrize("sequences,drafts,vocabulary", [(1, 1, 1), (1, 4, 2), (3, 5, 31), (5, 3, 1000), (17, 7, 4099), (2, 64, 257), (3, 0, 333), (2, 4, 248320)])
@pytest.mark.parametrize("probabilities", [True, False])
def test_verify(package, sequences, drafts, vocabulary, probabilities):
    target, draft, tokens, uniforms, _ = _case(sequences, drafts, vocabulary, seed=sequences * 7 + drafts)
    if not probabilities:
        uniforms[:, :drafts] *= 0.3
    want, _ = _check(package, target, tokens, uniforms, draft if probabilities and drafts else None)
    if sequences >= 5:
        assert len(set(want)) > 1                                 # some accepted, some rejected


@pytest.mark.parametrize("sequences,drafts,vocabulary", [(33, 2, 8191), (64, 2, 20000), (100, 2, 33001), (150, 2, 5000), (70, 1, 140000)])
def test_verify_of_many_sequences(package, sequences, drafts, vocabulary):
    """Eight, four, two and one block per sequence."""
    target, draft, tokens, uniforms, _ = _case(sequences, drafts, vocabulary, seed=sequences, sharp=4.0)
    _check(package, target, tokens, uniforms, draft)


def test_every_draft_accepted_and_none(package):
    target, draft, tokens, uniforms, _ = _case(4, 3, 501, seed=2)
    uniforms[:, :3] = 0.0
    want, _ = _check(package, target, tokens, uniforms, draft)
    assert want == [3] * 4
    tokens[:] = 17
    target[:, :, 17] = 0.0
    want, wish = _check(package, target, tokens, uniforms, draft)
    assert want == [0] * 4 and all(row[0] != 17 for row in wish)


def test_ends_of_the_uniform_numbers(package):
    """0 takes the first token that has a weight, the largest number below 1 (and anything above) the last one."""
    target, draft, tokens, uniforms, _ = _case(3, 2, 777, seed=3)
    uniforms[:, :2] = 1.0                                         # rejected, unless p > q
    target[:, :, :5] = 0.0
    target[:, :, 770:] = 0.0
    for value in (0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan):
        uniforms[:, 2] = value
        _check(package, target, tokens, uniforms)
        _check(package, target, tokens, uniforms, draft)


def test_counts_and_drafts_out_of_range(package):
    target, draft, tokens, uniforms, _ = _case(6, 4, 300, seed=4)
    uniforms[:, :4] *= 0.2
    counts = torch.tensor([0, 1, 2, 4, 9, -3], dtype=torch.int32)
    _check(package, target, tokens, uniforms, draft, counts)
    _check(package, target, tokens, uniforms, None, counts)
    uniforms[:, :4] = 0.0
    tokens[:, 1] = torch.tensor([-1, 300, 2 ** 30, -2 ** 31, 299, 0], dtype=torch.int32)
    want, _ = _check(package, target, tokens, uniforms, draft)
    assert want[:4] == [1] * 4
    _check(package, target, tokens, uniforms)


def test_nothing_left_to_draw_from(package):
    """A draft's row equal to the target's leaves no residual: the target's row is drawn from.  A row of zeros gives -1."""
    target, draft, tokens, uniforms, _ = _case(3, 2, 120, seed=5)
    draft[:] = target[:, :2]
    uniforms[:, :2] = 1.0
    want, wish = _check(package, target, tokens, uniforms, draft)
    assert want == [0] * 3 and all(row[0] >= 0 for row in wish)
    target[:] = 0.0
    _, wish = _check(package, target, tokens, uniforms, draft)
    assert all(row[0] == -1 for row in wish)
    target[:] = math.nan
    target[:, :, 11] = 0.25
    _, wish = _check(package, target, tokens, uniforms, None)
    draft[:, :, 5] = math.nan
    _check(package, target, tokens, uniforms, draft)


@pytest.mark.parametrize("vocabulary", [64, 1001])
def test_strided_rows(package, vocabulary):
    target, draft, tokens, uniforms, g = _case(3, 4, vocabulary, seed=6)
    for width in (vocabulary + 3, vocabulary + 4):
        a = torch.rand(3, 5, width, generator=g)
        b = torch.rand(3, 4, width, generator=g)
        a[..., 1:1 + vocabulary], b[..., 1:1 + vocabulary] = target, draft
        _check(package, target, tokens, uniforms, draft, gpu=(a.cuda()[..., 1:1 + vocabulary], b.cuda()[..., 1:1 + vocabulary]))


def test_the_draw_follows_the_weights(package):
    """Accepted and drawn tokens together are distributed as the target: 40 000 trials over 8 tokens, each frequency within 5
    standard deviations."""
    trials = 40000
    g = torch.Generator().manual_seed(7)
    p = torch.tensor([0.3, 0.0, 0.2, 0.05, 0.25, 0.1, 0.06, 0.04])
    q = torch.tensor([0.1, 0.1, 0.2, 0.2, 0.05, 0.15, 0.1, 0.1])
    drafts = torch.multinomial(q, trials, replacement=True, generator=g).int().view(trials, 1)
    target, draft = p.expand(trials, 2, 8).contiguous().cuda(), q.expand(trials, 1, 8).contiguous().cuda()
    uniforms = torch.rand(trials, 2, generator=g).cuda()
    _, tokens = package.verify_drafts(target, drafts.cuda(), uniforms, draft_probabilities=draft)
    share = torch.bincount(tokens[:, 0].cpu().long(), minlength=8).double() / trials
    assert ((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / trials).sqrt() + 1e-12).all()


def test_refusals(package):
    target, draft, tokens, uniforms, _ = _case(2, 3, 50, seed=8)
    target, draft, tokens, uniforms = target.cuda(), draft.cuda(), tokens.cuda(), uniforms.cuda()
    for bad in (dict(target=target.half()), dict(target=target[:, :3]), dict(draft_tokens=tokens.long()), dict(uniforms=uniforms[:, :3]),
                dict(draft_probabilities=draft[:, :2]), dict(target=target.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(target=target.cpu()), dict(draft_counts=tokens[:, 0].long())):
        with pytest.raises(ValueError):
            package.verify_drafts(**{"target": target, "draft_tokens": tokens, "uniforms": uniforms, **bad})
    many = torch.rand(1, 66, 8, device="cuda")
    with pytest.raises(package.AimaMoeError) as error:
        package.verify_drafts(many, torch.zeros(1, 65, dtype=torch.int32, device="cuda"), torch.rand(1, 66, device="cuda"))
    assert error.value.status == -1
