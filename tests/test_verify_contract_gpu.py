"""GPU tests of the numbers that decide over a draft at and beyond the ends of their range: u_i q < p as it stands, a number that is
negative or NaN counts as 0.  Only u_n, which draws, is clamped to [0, 1)."""
from __future__ import annotations

import math

import pytest
import torch

import kv_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("u,stands", [(0.0, True), (0.5, True), (1.0 - 2.0 ** -24, True), (1.0, False), (1.5, False), (math.inf, False),
                                      (-1.0, True), (-math.inf, True), (math.nan, True)])
@pytest.mark.parametrize("probabilities", [True, False])
def test_a_draft_that_is_certain(package, u, stands, probabilities):
    """p = q = 1 at the draft: it stands while u < 1."""
    target, draft = torch.zeros(1, 2, 64), torch.zeros(1, 1, 64)
    target[0, :, 9] = draft[0, 0, 9] = 1.0
    drafts, uniforms = torch.tensor([[9]], dtype=torch.int32), torch.tensor([[u, 0.5]])
    given = draft if probabilities else None
    accepted, tokens = package.verify_drafts(target.cuda(), drafts.cuda(), uniforms.cuda(), draft_probabilities=None if given is None else given.cuda())
    assert accepted.tolist() == [int(stands)]
    assert (accepted.tolist(), tokens.tolist()) == kv_oracle.verify(target, drafts, uniforms, given)


def test_a_number_above_one_that_the_probabilities_outweigh(package):
    target, draft = torch.full((1, 2, 4), 0.25), torch.full((1, 1, 4), 0.125)
    drafts = torch.tensor([[2]], dtype=torch.int32)
    for u, stands in ((1.5, 1), (1.999, 1), (2.0, 0), (3.0, 0)):
        uniforms = torch.tensor([[u, 0.3]])
        accepted, tokens = package.verify_drafts(target.cuda(), drafts.cuda(), uniforms.cuda(), draft_probabilities=draft.cuda())
        assert accepted.tolist() == [stands]
        assert (accepted.tolist(), tokens.tolist()) == kv_oracle.verify(target, drafts, uniforms, draft)
