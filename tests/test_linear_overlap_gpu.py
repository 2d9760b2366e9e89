"""Row offsets that fall, so that two sequences claim the same rows although there is room for both: reported by every form."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from linear_cases import DIM, Problem  # noqa: E402


@pytest.mark.parametrize("offsets", [[0, 10, 5, 20], [0, 100, 40, 150], [0, 600, 590, 1200]])
@pytest.mark.parametrize("what", ["conv", "delta", "states"])
def test_rows_of_two_sequences_are_reported(package, offsets, what):
    tokens = offsets[-1]
    p = Problem(package, [tokens, 0, 0], earlier=[5, 5, 5], gated=True)
    batch = p.layer.batch(p.device_batch.slots, tokens=tokens, row_offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"), max_new_tokens=tokens)
    states, conv_states = p.states.clone(), p.conv_states.clone()
    if what == "conv":
        room = torch.full((tokens + 32, p.x.shape[1]), 7.0, dtype=torch.bfloat16, device="cuda")
        p.layer.conv(0, batch, p.x, out=room[:tokens])
    else:
        room = torch.full((tokens + 32, p.v_heads, DIM), 7.0, dtype=torch.bfloat16, device="cuda")
        p.delta(batch=batch, out=room[:tokens], outputs=what == "delta")
    with pytest.raises(package.AimaMoeError):
        p.layer.sync()
    p.layer.sync()
    assert bool((room[tokens:] == 7.0).all())
    claimed = [p.batch["slots"][i] for i in (0, 2)]                     # the one between has no rows
    others = [i for i in range(states.shape[0]) if i not in claimed]
    assert torch.equal(p.states[others], states[others]) and torch.equal(p.conv_states[others], conv_states[others])
