"""Convolution and gated delta rule of the linear-attention layers against the 64-bit oracle."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import linear_oracle  # noqa: E402
from linear_cases import DIM, HALF_STEP, Problem, check_delta, constants  # noqa: E402

# rows of each sequence, tokens before them
BATCHES = {
    "one_token": ([1], [100]),
    "first_token": ([1], [0]),
    "decode": ([1] * 9, [5, 0, 1000, 1, 2, 3, 0, 77, 8]),
    "drafts": ([5, 3, 1, 8], [100, 0, 4, 1]),
    "with_empty": ([0, 4, 0, 1, 0], [3, 9, 0, 2, 0]),
    "two_runs": ([17], [64]),
    "edges": ([15, 16, 17, 31, 32, 33], [1, 0, 2, 3, 0, 9]),
    "chunk_edges": ([63, 64, 65, 1, 129, 2], [7, 0, 1, 0, 3, 9]),
    "prompt": ([300], [0]),
    "long": ([1000], [7]),
    "long_and_short": ([650, 33, 700, 1], [0, 64, 3, 5]),
    "mixed": ([1, 130, 1, 1, 67, 3, 1], [9, 0, 0, 5, 11, 2, 800]),
}


def most(rows):
    return max(rows)


# -- convolution -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("name", BATCHES)
def test_convolution(package, name, width):
    rows, earlier = BATCHES[name]
    p = Problem(package, rows, width=width, earlier=earlier, fused=width != 3, seed=width)
    wanted = p.conv_wanted()
    got = p.conv()
    p.layer.sync()
    p.check_conv(got, p.conv_states, wanted)


@pytest.mark.parametrize("keep", [[0, 0, 0, 0], [1, 2, 0, 3], [3, 3, 1, 8], [-5, 100, 1, 4]])
def test_convolution_keeps_what_it_is_told(package, keep):
    p = Problem(package, [5, 3, 1, 8], earlier=[100, 0, 4, 1], keep=keep)
    wanted = p.conv_wanted()
    got = p.conv()
    p.layer.sync()
    p.check_conv(got, p.conv_states, wanted)


def test_convolution_without_lengths_and_offsets(package):
    p = Problem(package, [6, 6, 6], k_heads=1, v_heads=1)
    p.device_batch = p.layer.batch(p.device_batch.slots, tokens=18)
    wanted = p.conv_wanted()
    p.check_conv(p.conv(), p.conv_states, wanted)


def test_convolution_of_a_padded_batch(package):
    """Sequences that are not there and rows before a sequence's first position give zeros; rows behind the last sequence stay."""
    p = Problem(package, [4, 20, 4, 40], earlier=[9, 3, 0, 0], slots=[-1, 2, 0, 5], behind=3, short={2: 2, 3: 0})
    wanted = p.conv_wanted()
    out = torch.full((p.tokens, p.x.shape[1]), 7.0, dtype=torch.bfloat16, device="cuda")
    p.conv(out=out)
    p.layer.sync()
    p.check_conv(out, p.conv_states, wanted, rows=slice(0, 68))
    assert bool((out[68:] == 7.0).all()) and bool((out[:4] == 0.0).all()) and bool((out[24:26] == 0.0).all()) and bool((out[28:68] == 0.0).all())


def test_convolution_in_pieces(package):
    """A prompt in three calls gives the bits of one."""
    whole = Problem(package, [150], earlier=[0], seed=3)
    want = whole.conv()
    pieces = Problem(package, [150], earlier=[0], seed=3)
    outs, row = [], 0
    for n in (1, 70, 79):
        batch = pieces.layer.batch(pieces.device_batch.slots, tokens=n, lengths=torch.tensor([row + n], dtype=torch.int32, device="cuda"))
        outs.append(pieces.layer.conv(0, batch, pieces.x[row:row + n]))
        row += n
    assert torch.equal(torch.cat(outs), want) and torch.equal(pieces.conv_states, whole.conv_states)


def test_convolution_of_extreme_inputs(package):
    """Infinities and NaN stay in their channel and behind their row; the largest and smallest numbers are not special."""
    p = Problem(package, [40, 40], earlier=[3, 3])
    p.x[5, 7], p.x[20, 9], p.x[30, 11] = float("nan"), float("inf"), float("-inf")
    p.x[1, 64:72] = torch.finfo(torch.bfloat16).max
    p.x[2, 64:72] = torch.finfo(torch.bfloat16).tiny
    p.conv_weight[64:72] = 1.0e-3
    out, size, states = p.conv_wanted()
    got = p.conv().double()
    bad = ~torch.isfinite(out)
    assert not bool(torch.isfinite(got[bad & torch.isnan(out)]).any())
    bound = out.abs() * (HALF_STEP + 2.0 ** -20) + 1.1 * 8 * 2.0 ** -24 * size + 2.0 ** -133
    assert bool(((got - out).abs() <= bound)[~bad].all())
    assert bool((got[40:][:, [7, 9, 11]].isfinite()).all()) and bool(got[:5, 7].isfinite().all()) and bool(got[9:40, 7].isfinite().all())


# -- delta rule --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("name", BATCHES)
def test_delta_rule(package, name, gated):
    rows, earlier = BATCHES[name]
    p = Problem(package, rows, earlier=earlier, gated=gated, fused=not gated, seed=len(rows))
    wanted = p.delta_wanted()
    got = p.delta()
    p.layer.sync()
    check_delta(got, p.states, wanted, most(rows))


@pytest.mark.parametrize("heads", [(1, 1), (1, 5), (3, 3), (16, 32)])
@pytest.mark.parametrize("rows", [[1], [4, 2], [70, 9], [900]])
def test_delta_rule_heads(package, heads, rows):
    p = Problem(package, rows, k_heads=heads[0], v_heads=heads[1], earlier=[3] * len(rows), gated=True, seed=7)
    wanted = p.delta_wanted()
    got = p.delta()
    p.layer.sync()
    check_delta(got, p.states, wanted, most(rows))


@pytest.mark.parametrize("rows", [[5, 3, 1, 8], [200, 70, 1, 64], [700, 70, 1, 129]])
@pytest.mark.parametrize("keep", [[0, 0, 0, 0], [1, 2, 0, 3], [3, 3, 1, 8], [-5, 1000, 1, 4], [5, 64, 1, 63], [641, 70, 0, 128]])
@pytest.mark.parametrize("outputs", [True, False])
def test_delta_rule_keeps_what_it_is_told(package, rows, keep, outputs):
    p = Problem(package, rows, earlier=[100, 0, 4, 1], keep=keep, gated=True)
    wanted = p.delta_wanted()
    got = p.delta(outputs=outputs)
    p.layer.sync()
    assert (got is None) == (not outputs)
    check_delta(got, p.states, wanted, most(rows))
    for s, kept in enumerate(keep):           # nothing enters: not a bit moves
        if kept <= 0:
            assert torch.equal(p.states[p.batch["slots"][s]].double(), wanted["states"][p.batch["slots"][s]])


def test_delta_rule_without_lengths_and_offsets(package):
    p = Problem(package, [6, 6, 6], k_heads=1, v_heads=2)
    p.device_batch = p.layer.batch(p.device_batch.slots, tokens=18)
    wanted = p.delta_wanted()
    check_delta(p.delta(), p.states, wanted, 6)


@pytest.mark.parametrize("rows,short", [([4, 20, 4, 3], {2: 2, 3: 0}), ([4, 200, 100, 70], {2: 50, 3: 0}), ([4, 200, 130, 70], {2: 65, 3: 5}), ([4, 700, 650, 640], {2: 600, 3: 0})])
def test_delta_rule_of_a_padded_batch(package, rows, short):
    p = Problem(package, rows, earlier=[9, 3, 0, 0], slots=[-1, 2, 0, 5], behind=3, short=short)
    wanted = p.delta_wanted()
    before = p.states.clone()
    out = torch.full((p.tokens, p.v_heads, DIM), 7.0, dtype=torch.bfloat16, device="cuda")
    p.delta(out=out)
    p.layer.sync()
    total = sum(rows)
    for name in ("out", "out_error", "reach"):
        wanted[name] = wanted[name][:total]
    check_delta(out[:total], p.states, wanted, most(rows))
    assert bool((out[total:] == 7.0).all()) and bool((out[:4] == 0.0).all())
    for slot in (1, 3, 4):
        assert torch.equal(p.states[slot], before[slot])


@pytest.mark.parametrize("pieces", [(1, 70, 79), (64, 64, 22), (40, 1, 1, 1, 107)])
def test_delta_rule_in_pieces(package, pieces):
    p = Problem(package, [150], earlier=[0], seed=3, gated=True)
    wanted = p.delta_wanted()
    outs, row = [], 0
    for n in pieces:
        batch = p.layer.batch(p.device_batch.slots, tokens=n, lengths=torch.tensor([row + n], dtype=torch.int32, device="cuda"))
        part = slice(row, row + n)
        outs.append(p.layer.delta(0, batch, p.q[part], p.k[part], p.v[part], p.a[part], p.b[part], gate=p.gate[part]))
        row += n
    check_delta(torch.cat(outs), p.states, wanted, 150)


def test_drafts_then_what_stands_of_them(package):
    """The way of a speculative step: outputs with nothing kept, then the states alone."""
    p = Problem(package, [5, 5, 5], earlier=[10, 0, 30], keep=[0, 0, 0], gated=True)
    before = p.states.clone()
    wanted = p.delta_wanted()
    got = p.delta()
    check_delta(got, p.states, wanted, 5)
    assert torch.equal(p.states, before)
    p.batch["keep"] = [1, 5, 3]
    p.device_batch = p.make_batch()
    wanted = p.delta_wanted()
    assert p.delta(outputs=False) is None
    p.layer.sync()
    check_delta(None, p.states, wanted, 5)


@pytest.mark.parametrize("rows", [[12, 12], [100, 90]])
def test_delta_rule_of_extreme_gates(package, rows):
    """Decays from none to all at once, rates of 0 and 1, zero keys, equal keys, values far apart in size."""
    p = Problem(package, rows, earlier=[3, 3], seed=5)
    p.a, p.b = p.a.clone(), p.b.clone()
    p.q, p.k, p.v = p.q.clone(), p.k.clone(), p.v.clone()
    p.a[0], p.a[3], p.a[4], p.a[7] = 60.0, -60.0, 0.0, 1000.0
    p.b[1], p.b[5], p.b[6] = 100.0, -100.0, 0.0
    p.b[0] = 100.0
    p.k[2], p.q[6] = 0.0, 0.0
    p.k[8:] = p.k[8:9]                           # the same key again and again
    p.v[9] *= 1.0e4
    p.v[10] *= 1.0e-6
    p.v[:, :, 3] *= 1.0e20
    p.v[:, :, 4] *= 1.0e-20
    p.k[11] *= 1.0e-4                            # below the norm's epsilon
    p.a_log[0], p.a_log[1] = -20.0, 3.0
    wanted = p.delta_wanted()
    got = p.delta()
    p.layer.sync()
    check_delta(got, p.states, wanted, most(rows), typical=False)


@pytest.mark.parametrize("rows", [[30, 30], [150, 130], [600, 520]])
@pytest.mark.parametrize("what", ["v", "k", "q", "a", "b", "inf", "state"])
def test_a_nan_reaches_what_depends_on_it_alone(package, rows, what):
    p = Problem(package, rows, earlier=[3, 3], seed=9)
    p.a, p.b = p.a.clone(), p.b.clone()
    p.q, p.k, p.v = p.q.clone(), p.k.clone(), p.v.clone()
    at = 17
    if what == "v":
        p.v[at, 1, 5] = float("nan")
    elif what == "inf":
        p.v[at, 1, 5] = float("inf")
    elif what == "state":
        p.states[p.batch["slots"][0], 1, 3, 5] = float("nan")
    elif what in "ab":
        getattr(p, what)[at, 1] = float("nan")
    else:
        getattr(p, what)[at, 0, 5] = float("nan")            # of heads 0 and 1
    wanted = p.delta_wanted()
    got = p.delta()
    p.layer.sync()
    check_delta(got, p.states, wanted, most(rows))
    finite = torch.isfinite(got)
    n, first = rows[0], slice(0, rows[0])
    assert bool(finite[n:].all()) and bool(finite[first, 2:].all())
    column = torch.arange(DIM, device="cuda") == 5
    if what in ("v", "inf"):
        assert bool(finite[first, 0].all()) and bool(finite[first, 1][:, ~column].all())
        assert bool(finite[:at, 1].all()) and not bool(finite[at:n, 1, 5].any())
    elif what == "state":
        assert not bool(finite[first, 1, 5].any()) and bool(finite[first, 1][:, ~column].all()) and bool(finite[first, 0].all())
    elif what == "q":
        assert bool(finite[:at].all()) and bool(finite[at + 1:].all()) and not bool(finite[at, :2].any())
        assert bool(torch.isfinite(p.states).all())
    elif what in "ab":
        assert bool(finite[:at].all()) and bool(finite[first, 0].all()) and not bool(finite[at:n, 1].any())
    else:
        assert bool(finite[:at].all()) and not bool(finite[at:n, :2].any())


@pytest.mark.parametrize("rows", [[3, 2, 4], [100, 70, 65]])
@pytest.mark.parametrize("bad", ["slot", "slot_below", "length", "offset_end", "offset_begin"])
def test_a_bad_sequence_is_left_out_and_reported(package, rows, bad):
    p = Problem(package, rows, earlier=[3, 3, 3], gated=True)
    slots, lengths, offsets = list(p.batch["slots"]), list(p.batch["lengths"]), list(p.batch["offsets"])
    untouched = slots[1]
    gone = [1]
    if bad == "slot":
        slots[1] = 5
    elif bad == "slot_below":
        slots[1] = -2
    elif bad == "length":
        lengths[1] = -1
    elif bad == "offset_end":
        offsets[3], gone, untouched = p.tokens + 1, [2], slots[2]
    else:
        offsets[0], gone, untouched = -1, [0], slots[0]
    good = [s for s in range(3) if s not in gone]
    batch = p.layer.batch(*(torch.tensor(slots, dtype=torch.int32, device="cuda"),), tokens=p.tokens,
                          lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                          row_offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"), max_new_tokens=max(rows))
    wanted = p.delta_wanted()
    conv_wanted = p.conv_wanted()
    before, conv_before = p.states[untouched].clone(), p.conv_states[untouched].clone()
    got = p.delta(batch=batch)
    with pytest.raises(package.AimaMoeError):
        p.layer.sync()
    p.layer.sync()                             # once
    conv = p.layer.conv(0, batch, p.x)
    with pytest.raises(package.AimaMoeError):
        p.layer.sync()
    assert torch.equal(p.states[untouched], before) and torch.equal(p.conv_states[untouched], conv_before)
    for s in good:
        part = slice(p.batch["offsets"][s], p.batch["offsets"][s + 1])
        slot = slice(p.batch["slots"][s], p.batch["slots"][s] + 1)
        check_delta(got[part], p.states[slot], {"out": wanted["out"][part], "out_error": wanted["out_error"][part], "reach": wanted["reach"][part],
                                                "states": wanted["states"][slot], "state_error": wanted["state_error"][slot]}, most(rows))
        p.check_conv(conv[part], p.conv_states[slot], (conv_wanted[0][part], conv_wanted[1][part], conv_wanted[2][slot]))


def test_many_sequences(package):
    """As many as a batch can have, some of them long."""
    rows = [1 + (i % 3) * (i % 7) for i in range(1024)]
    rows[500], rows[1023] = 90, 33
    p = Problem(package, rows, k_heads=1, v_heads=1, earlier=[i % 5 for i in range(1024)])
    wanted, conv_wanted = p.delta_wanted(), p.conv_wanted()
    got, conv = p.delta(), p.conv()
    p.layer.sync()
    check_delta(got, p.states, wanted, most(rows))
    p.check_conv(conv, p.conv_states, conv_wanted)


@pytest.mark.parametrize("rows", [[1, 1, 1], [4, 3, 2], [130, 70, 3]])
def test_captured_calls_follow_their_inputs(package, rows):
    """One capture of convolution and delta rule, replayed for other slots, lengths and rows."""
    p = Problem(package, rows, earlier=[4, 0, 9], gated=True)
    q, k, v = (p.k_heads, p.k_heads, p.v_heads)

    def step():
        y = p.conv().view(p.tokens, -1, DIM)
        parts = y.split([q, k, v], dim=1)
        return y, p.layer.delta(0, p.device_batch, *parts, p.a, p.b, gate=p.gate)

    first = (p.states.clone(), p.conv_states.clone())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y, out = step()
    torch.cuda.current_stream().wait_stream(stream)
    p.states.copy_(first[0])
    p.conv_states.copy_(first[1])
    for slots, lengths in (([0, 1, 2], [rows[0] + 1, rows[1], 1000]), ([4, 0, 3], [rows[0], rows[1] + 7, rows[2]])):
        p.batch["slots"], p.batch["lengths"] = slots, lengths
        p.device_batch.slots.copy_(torch.tensor(slots, dtype=torch.int32))
        p.device_batch.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        conv_wanted = p.conv_wanted()
        states = p.states.clone()
        graph.replay()
        torch.cuda.synchronize()
        p.check_conv(y.view(p.tokens, -1), p.conv_states, conv_wanted)
        parts = y.split([q, k, v], dim=1)
        wanted = linear_oracle.delta(*parts, p.a, p.b, p.a_log, p.dt_bias, states, p.batch, gate=p.gate, norm_weight=p.norm_weight,
                                     floor=constants(most(rows))[1])
        check_delta(out, p.states, wanted, most(rows))
    p.layer.sync()


@pytest.mark.parametrize("rows", [[1] * 5, [300, 200]])
def test_two_handles_on_two_streams(package, rows):
    """Each has its own workspace; the results are those of one after the other."""
    problems = [Problem(package, rows, k_heads=4, v_heads=8, earlier=[2] * len(rows), seed=s, gated=True) for s in (1, 2)]
    wanted = [p.delta_wanted() for p in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    outs = []
    for p, stream in zip(problems, streams):
        with torch.cuda.stream(stream):
            outs.append(p.delta())
    for p, out, want in zip(problems, outs, wanted):
        p.layer.sync()
        check_delta(out, p.states, want, most(rows))


@pytest.mark.parametrize("rows", [[3, 5], [200, 333], [1500]])
def test_a_call_gives_the_same_bits_every_time(package, rows):
    p = Problem(package, rows, earlier=[2, 0][:len(rows)], gated=True, k_heads=4, v_heads=8)
    before = p.states.clone()
    results = []
    for _ in range(3):
        p.states.copy_(before)
        results.append((p.delta(), p.states.clone()))
    for out, states in results[1:]:
        assert torch.equal(out, results[0][0]) and torch.equal(states, results[0][1])


def test_broadcast_inputs(package):
    """A stride of zero: one key for all tokens, one gate for all heads."""
    p = Problem(package, [20], earlier=[2], gated=True)
    p.k = p.k[:1].expand(20, -1, -1)
    p.gate = p.gate[:, :1].expand(-1, p.v_heads, -1)
    wanted = p.delta_wanted()
    check_delta(p.delta(), p.states, wanted, 20)


def test_refusals(package):
    p = Problem(package, [4, 4], earlier=[0, 0], gated=True)
    layer, batch = p.layer, p.device_batch
    call = (p.q, p.k, p.v, p.a, p.b)
    with pytest.raises(ValueError):
        layer.delta(0, batch, p.q.float(), *call[1:])
    with pytest.raises(ValueError):
        layer.delta(0, batch, p.q[:3], *call[1:])
    with pytest.raises(ValueError):
        layer.delta(0, batch, p.v, *call[1:])
    with pytest.raises(ValueError):
        layer.delta(0, batch, p.q, p.k, p.v, p.a[:, :2], p.b)
    with pytest.raises(ValueError):
        layer.delta(0, batch, p.q, p.k, p.v.cpu(), p.a, p.b)
    with pytest.raises(ValueError):
        layer.delta(0, batch, *call, out=torch.empty(8, p.v_heads, 2 * DIM, dtype=torch.bfloat16, device="cuda")[..., :DIM])
    with pytest.raises(package.AimaMoeError):
        layer.delta(1, batch, *call)
    with pytest.raises(ValueError):
        layer.conv(0, batch, p.x[:, :-DIM])
    with pytest.raises(ValueError):
        layer.batch(p.device_batch.slots.long(), tokens=8)
    with pytest.raises(ValueError):
        layer.batch(p.device_batch.slots, tokens=8, keep=torch.zeros(3, dtype=torch.int32, device="cuda"))
    flat = p.v.contiguous()
    with pytest.raises(package.AimaMoeError) as error:                 # values would be written over
        layer.delta(0, batch, p.q, p.k, flat, p.a, p.b, out=flat)
    assert error.value.status == -4
    x = p.x.contiguous()
    with pytest.raises(package.AimaMoeError) as error:
        layer.conv(0, batch, x, out=x)
    assert error.value.status == -4
    with pytest.raises(package.AimaMoeError) as error:                 # more than was prepared for
        layer.conv(0, layer.batch(p.device_batch.slots, tokens=10), torch.zeros(10, layer.channels, dtype=torch.bfloat16, device="cuda"))
    assert error.value.status == -8
    bare = package.LinearAttention(k_heads=2, v_heads=4, slots=4, max_sequences=2, max_tokens=8)
    with pytest.raises(package.AimaMoeError) as error:
        bare.delta(0, batch, *call)
    assert error.value.status == -3
    bare.bind_layer(0, states=p.states[:4], a_log=p.a_log, dt_bias=p.dt_bias)
    with pytest.raises(package.AimaMoeError) as error:                 # no weight for the gate's norm, none for the convolution
        bare.delta(0, batch, *call, gate=p.gate)
    assert error.value.status == -3
    with pytest.raises(package.AimaMoeError) as error:
        bare.conv(0, batch, p.x)
    assert error.value.status == -3
    for wrong in (dict(k_heads=3, v_heads=4), dict(k_heads=0, v_heads=4), dict(conv_width=5), dict(conv_width=1), dict(slots=0), dict(max_tokens=0)):
        with pytest.raises(package.AimaMoeError):
            package.LinearAttention(**{"k_heads": 2, "v_heads": 4, "slots": 4, **wrong})
    p.layer.sync()
