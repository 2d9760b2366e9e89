"""GPU tests of the attention of many row tiles, whose shares a launch of its own computes (more than 384 row tiles): with 128 query heads
for a key/value head a row tile is one token, so some hundred tokens are enough.  Tolerances as in test_kv_cache_gpu.py."""
from __future__ import annotations

import pytest
import torch

import kv_oracle
from test_kv_cache_gpu import Setup

pytestmark = pytest.mark.gpu


def _bound(want, spread):
    return want.abs() * 2.0 ** -8 + spread * (2.0 ** -8 + 2.0 ** -9)


def _oracle(setup, q, lengths=None):
    return kv_oracle.attention(*(t.float() for t in setup.gpu), setup.table.tolist(), setup.offsets, lengths or setup.lengths, q,
                               setup.heads[2] ** -0.5, setup.page)


def _run(setup, q, batch=None):
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    return setup.cache.attention(1, batch or setup.batch, q, out=out)


def _check(setup, q, out, lengths=None):
    want, spread = _oracle(setup, q, lengths)
    owned = setup.offsets[-1]
    assert (out[owned:] == 7.0).all() and torch.isfinite(out.float()).all()
    assert ((out.double() - want).abs() <= _bound(want, spread))[:owned].all()


PLANNED = [
    # lengths, new, heads, page
    ([500, 0, 100, 30, 260], [400, 0, 60, 50, 3], (128, 1, 64), 16),
    ([500, 0, 100, 30, 260], [400, 0, 60, 50, 3], (128, 1, 128), 32),
    ([500, 0, 100, 30, 260], [400, 0, 60, 50, 3], (128, 1, 256), 64),
    ([0, 7, 430], [300, 120, 430], (128, 1, 64), 128),          # most rows see nothing
    ([1300, 40], [1100, 40], (128, 1, 64), 64),                 # more row tiles than the planning block has threads
    ([900, 900, 1], [900, 700, 1], (128, 1, 256), 64),
    ([1] * 600, [1] * 600, (128, 1, 64), 16),
    ([0] * 500 + [70] * 100, [5] * 600, (128, 1, 64), 16),
    ([6300], [6200], (16, 2, 256), 64),
    ([3000, 2500], [2999, 2400], (12, 1, 128), 128),
    ([1700] * 4, [1600] * 4, (112, 8, 64), 64),
]


@pytest.mark.parametrize("lengths,new,heads,page", PLANNED)
def test_many_row_tiles(package, lengths, new, heads, page):
    setup = Setup(package, lengths, new, heads, page, 0, seed=sum(new) + page, gap=2)
    group = heads[0] // heads[1]
    assert setup.tokens // (128 // group) + len(lengths) > 384
    q = setup.randn(setup.tokens, heads[0], heads[2], std=1.5).cuda()
    out = _run(setup, q)
    setup.cache.sync()
    _check(setup, q, out)
    assert torch.equal(_run(setup, q), out)                     # the same bits every time


@pytest.mark.parametrize("heads", [(128, 1, 64), (128, 1, 128), (128, 1, 256)])
def test_one_call_gives_what_chunks_give(package, heads):
    """Chunks of few row tiles find their shares by themselves."""
    setup = Setup(package, [700], [600], heads, 64, 0, seed=3)
    q = setup.randn(600, heads[0], heads[2], std=1.5).cuda()
    whole = _run(setup, q)
    _check(setup, q, whole)
    table = setup.table.cuda()
    _, spread = _oracle(setup, q)
    for at in range(0, 600, 150):
        lengths = torch.tensor([100 + at + 150], dtype=torch.int32, device="cuda")
        part = _run(setup, q[at:at + 150], setup.cache.batch(table, lengths, tokens=150))
        difference = (part.double() - whole[at:at + 150].double()).abs()
        assert (difference <= 2 * _bound(whole[at:at + 150].double(), spread[at:at + 150])).all()
    setup.cache.sync()


def test_a_length_out_of_range_among_many_row_tiles(package):
    setup = Setup(package, [450, 200, 90], [400, 30, 90], (128, 1, 64), 64, 0, seed=5)
    q = setup.randn(setup.tokens, 128, 64, std=1.5).cuda()
    right = _run(setup, q)
    setup.cache.sync()
    for length in (64 * setup.columns + 1, -1):
        lengths = [450, length, 90]
        bad = setup.cache.batch(setup.table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), tokens=setup.tokens,
                                row_offsets=torch.tensor(setup.offsets, dtype=torch.int32, device="cuda"), max_new_tokens=400)
        out = _run(setup, q, bad)
        with pytest.raises(package.AimaMoeError) as error:
            setup.cache.sync()
        assert error.value.status == -1
        assert not out[400:430].any()
        _check(setup, q, out, [450, 0, 90])
        setup.cache.sync()
    table = setup.table.clone()
    table[1, 0] = -1
    bad = setup.cache.batch(table.cuda(), setup.batch.lengths, tokens=setup.tokens, row_offsets=setup.batch.row_offsets, max_new_tokens=400)
    out = _run(setup, q, bad)
    with pytest.raises(package.AimaMoeError):
        setup.cache.sync()
    want, spread = _oracle(setup, q)
    close = (out.double() - want).abs() <= _bound(want, spread)
    assert close[:400].all() and close[430:].all()
    assert torch.equal(_run(setup, q), right)


def test_many_row_tiles_in_a_captured_graph(package):
    """The shares come from the lengths of the replay."""
    setup = Setup(package, [500, 300], [400, 100], (128, 1, 64), 64, 0, seed=6)
    q = setup.randn(setup.tokens, 128, 64).cuda()
    out = _run(setup, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        setup.cache.attention(1, setup.batch, q, out=out)
    for lengths in ([500, 300], [410, 100], [300, 40], [0, 0], [512, 1]):
        setup.batch.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        setup.cache.sync()
        _check(setup, q, out, lengths)


@pytest.mark.parametrize("heads,new", [((16, 2, 256), 1), ((16, 2, 256), 3), ((8, 8, 64), 5), ((16, 2, 128), 4)])
def test_as_many_sequences_as_a_batch_can_have(package, heads, new):
    """1024 sequences, some of them empty, some with fewer positions than rows: few rows, and many with shares from a launch of their own."""
    g = torch.Generator().manual_seed(new)
    lengths = torch.randint(0, 260, (1024,), generator=g).tolist()
    lengths[0], lengths[500], lengths[1023] = 0, 1500, 2
    setup = Setup(package, lengths, [new] * 1024, heads, 64, 0, seed=new, gap=1)
    q = setup.randn(setup.tokens, heads[0], heads[2], std=1.5).cuda()
    out = _run(setup, q)
    setup.cache.sync()
    _check(setup, q, out)
