"""Linear-attention layers at the ends of their ranges: sizes and offsets that pass 32 bits, the borders of the rules that choose a form,
graphs that share a handle, row offsets that claim rows twice."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from linear_cases import DIM, Problem, check_delta, constants  # noqa: E402

import linear_oracle  # noqa: E402


def compare(p, *, outputs=True):
    wanted, conv_wanted = p.delta_wanted(), p.conv_wanted()
    got, conv = p.delta(outputs=outputs), p.conv()
    p.layer.sync()
    check_delta(got, p.states, wanted, max(p.rows))
    p.check_conv(conv, p.conv_states, conv_wanted)


@pytest.mark.parametrize("rows", [[3], [130]])
def test_states_behind_four_gigabytes(package, rows):
    """The slot begins 2^31 elements behind the first one's state."""
    heads, slot = 32, 4096                                  # 4096 * 32 * 128 * 128 = 2^31
    small = Problem(package, rows, k_heads=16, v_heads=heads, earlier=[5], slots=[0], spare=0, gated=True)
    layer = package.LinearAttention(k_heads=16, v_heads=heads, slots=slot + 1, max_sequences=1, max_tokens=sum(rows))
    conv_states, states = layer.allocate_layer()
    states[slot].copy_(small.states[0])
    conv_states[slot].copy_(small.conv_states[0])
    layer.bind_layer(0, conv_weight=small.conv_weight, conv_states=conv_states, states=states, a_log=small.a_log, dt_bias=small.dt_bias,
                     norm_weight=small.norm_weight)
    batch = layer.batch(torch.tensor([slot], dtype=torch.int32, device="cuda"), tokens=sum(rows), lengths=torch.tensor([rows[0] + 5], dtype=torch.int32, device="cuda"))
    out = layer.delta(0, batch, small.q, small.k, small.v, small.a, small.b, gate=small.gate)
    conv = layer.conv(0, batch, small.x)
    layer.sync()
    assert torch.equal(out, small.delta()) and torch.equal(conv, small.conv())
    assert torch.equal(states[slot], small.states[0]) and torch.equal(conv_states[slot], small.conv_states[0])
    assert bool((states[slot - 1] == 0).all()) and bool((states[0] == 0).all())


@pytest.mark.parametrize("rows", [20, 600])
def test_rows_behind_four_gigabytes(package, rows):
    """Rows 2^32 elements from the first to the last, and more."""
    p = Problem(package, [rows], k_heads=1, v_heads=2, earlier=[0], gated=True)
    stride = (1 << 32) // (rows - 1) // 8 * 8 + 8
    row = torch.empty((rows - 1) * stride + 4096, dtype=torch.bfloat16, device="cuda")

    def spread(x, at):
        shape = x.shape[1:]
        strides = (shape[-1], 1) if len(shape) == 2 else (1,)
        y = row.as_strided(x.shape, (stride, *strides), at)
        y.copy_(x)
        return y

    wanted, conv_wanted = p.delta_wanted(), p.conv_wanted()
    p.q, p.k, p.v, p.gate = spread(p.q, 0), spread(p.k, 128), spread(p.v, 256), spread(p.gate, 512)
    p.a, p.b, p.x = spread(p.a, 768), spread(p.b, 776), spread(p.x, 1024)
    got, conv = p.delta(), p.conv()
    p.layer.sync()
    check_delta(got, p.states, wanted, rows)
    p.check_conv(conv, p.conv_states, conv_wanted)


@pytest.mark.parametrize("rows", [[28], [29], [28, 29, 1], [64], [65], [29] * 20])
def test_where_the_forms_meet(package, rows):
    compare(Problem(package, rows, earlier=[3 * (i % 2) for i in range(len(rows))], gated=True))


@pytest.mark.parametrize("heads,rows", [((16, 32), [2100]), ((2, 8), [1700]), ((1, 1), [2900]), ((16, 32), [900, 1500]), ((24, 48), [1300]), ((2, 74), [1100]),
                                        ((1, 75), [1100]), ((2, 2), [1500, 700, 2000])])
def test_sequences_cut_into_segments(package, heads, rows):
    """Some and none of the cuts, by heads and length; short sequences beside long ones leave segments empty."""
    compare(Problem(package, rows, k_heads=heads[0], v_heads=heads[1], earlier=[0, 9, 2][:len(rows)],
                    gated=True))


@pytest.mark.parametrize("rows", [[1], [2, 1], [40]])
def test_the_most_heads(package, rows):
    compare(Problem(package, rows, k_heads=128, v_heads=256, earlier=[1, 0][:len(rows)], spare=0))


def test_two_graphs_of_one_handle(package):
    """They share its workspace: replayed in turn on one stream, each gives what the eager call gives."""
    p = Problem(package, [1500], earlier=[7], gated=True, k_heads=4, v_heads=8)
    first = p.states.clone()
    one = p.layer.batch(p.device_batch.slots, tokens=70, lengths=torch.tensor([100], dtype=torch.int32, device="cuda"))
    calls = [lambda: p.delta(), lambda: p.layer.delta(0, one, p.q[:70], p.k[:70], p.v[:70], p.a[:70], p.b[:70], gate=p.gate[:70])]
    eager = []
    for call in calls:
        p.states.copy_(first)
        eager.append((call(), p.states.clone()))
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for call in calls:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(call())
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(stream)
    for i in (0, 1, 1, 0, 1):
        p.states.copy_(first)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], eager[i][0]) and torch.equal(p.states, eager[i][1])
    p.layer.sync()


def test_rows_claimed_more_often_than_there_is_room_for(package):
    """Offsets that fall, so that every second sequence has the same rows: reported, and nothing is written outside the call's tensors."""
    count, tokens = 16, 640
    p = Problem(package, [tokens] + [0] * (count - 1), earlier=[5] * count, gated=True)
    offsets = torch.tensor([0, tokens] * (count // 2) + [0], dtype=torch.int32, device="cuda")
    lengths = torch.full((count,), 5 + tokens, dtype=torch.int32, device="cuda")
    batch = p.layer.batch(p.device_batch.slots, tokens=tokens, lengths=lengths, row_offsets=offsets, max_new_tokens=tokens)
    spare = [i for i in range(count + 2) if i not in p.batch["slots"]]
    before = p.states.clone()
    room = torch.full((tokens + 64, p.v_heads, DIM), 7.0, dtype=torch.bfloat16, device="cuda")
    p.delta(out=room[:tokens], batch=batch)
    with pytest.raises(package.AimaMoeError):
        p.layer.sync()
    assert bool((room[tokens:] == 7.0).all()) and torch.equal(p.states[spare], before[spare])
    falling = p.batch["slots"][1::2]                        # without rows: untouched
    assert torch.equal(p.states[falling], before[falling])
    p.states.copy_(before)                                  # and the handle goes on working
    wanted = p.delta_wanted()
    check_delta(p.delta(), p.states, wanted, tokens)
    p.layer.sync()


def test_float64_reference_of_one_long_sequence(package):
    """10000 tokens: the state after 157 chunks is as near as after a few."""
    p = Problem(package, [10000], k_heads=1, v_heads=1, earlier=[0])
    wanted = linear_oracle.delta(p.q, p.k, p.v, p.a, p.b, p.a_log, p.dt_bias, p.states, p.batch, floor=constants(10000)[1])
    got = p.delta()
    p.layer.sync()
    check_delta(got, p.states, wanted, 10000)
