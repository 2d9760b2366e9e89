"""GPU tests of the attention's weights over their whole range, against oracle/kv_oracle.py in 64 bits.

The values are positive, so that an error that all weights of a size share shows in the output in full.  Tolerance: the output is rounded
to BF16 (2^-8), a weight may be held to 8 bits (2^-8 of itself), and 2^-9 is for scores, exponentials and sums in FP32."""
from __future__ import annotations

import math

import pytest
import torch

from test_kv_cache_gpu import Setup, _check_attention

pytestmark = pytest.mark.gpu


def _sink(package, length, new, heads, gaps, page=64, sink=3):
    """Keys that are zero but for one, whose score is `gaps` (log2 units, spread over the query heads) above all others; its
    value is zero, so that the output is what the small weights give."""
    q_heads, kv_heads, dim = heads
    setup = Setup(package, [length], [new], heads, page, 0, seed=length + new + dim)
    setup.gpu[2].fill_(2.0 ** -4)
    codes = torch.zeros(setup.gpu[0].shape)
    codes[int(setup.table[0, sink // page]), :, sink % page, 0] = 448.0
    setup.gpu[0].copy_(codes.to(torch.float8_e4m3fn).cuda())
    setup.gpu[1].copy_(setup.gpu[1].float().abs().clamp_min(1.0).to(torch.float8_e4m3fn))
    setup.gpu[1].view(torch.uint8)[int(setup.table[0, sink // page]), :, sink % page] = 0
    q = torch.zeros(new, q_heads, dim)
    low, high = gaps
    steps = torch.linspace(low, high, new * q_heads).view(new, q_heads)
    q[..., 0] = steps * math.log(2.0) * dim ** 0.5 / 28.0            # 448 / 16 = 28
    return setup, q.bfloat16()


@pytest.mark.parametrize("length", [60, 300, 1024])
@pytest.mark.parametrize("new", [1, 2, 5])
@pytest.mark.parametrize("heads", [(16, 2, 256), (16, 2, 128), (8, 1, 64), (8, 8, 64)])
def test_small_weights_of_few_rows_keep_their_bits(package, heads, new, length):
    """One position outweighs all others by 2^12 .. 2^27 and brings nothing."""
    for low, high in ((12.0, 16.0), (16.0, 20.0), (20.0, 24.0), (24.0, 27.0)):
        _check_attention(*_sink(package, length, new if new * heads[0] // heads[1] <= 16 else 1, heads, (low, high)))


@pytest.mark.parametrize("length", [60, 300, 1024])
@pytest.mark.parametrize("heads", [(16, 2, 256), (16, 2, 128), (8, 1, 64), (8, 8, 64)])
def test_small_weights_of_prompts_keep_their_bits(package, heads, length):
    """The same for many rows, up to where heads of 256 hold the weights beside the largest to 2^-8: 2^-22 of it."""
    for low, high in ((12.0, 16.0), (16.0, 19.0), (19.0, 22.0)) + (((22.0, 26.0),) if heads[2] < 256 else ()):
        _check_attention(*_sink(package, length, 40, heads, (low, high)))


def _scaled(package, lengths, new, heads, scales, scores=None, std=1.0, seed=7):
    """Pages whose value scales are `scales` in turn and whose keys lead to the scores `scores` (log2 units, by scale) above random
    ones; values between 1/2 and 1 times their scale."""
    q_heads, kv_heads, dim = heads
    setup = Setup(package, lengths, [min(new, n) for n in lengths], heads, 64, 0, seed=seed)
    codes = torch.randn(setup.gpu[0].shape, generator=setup.g) * 16
    codes[..., 0] = 0.0
    setup.gpu[2].fill_(2.0 ** -4)
    for row, length in zip(setup.table.tolist(), lengths):
        for column in range((length + 63) // 64):
            at = column % len(scales)
            setup.gpu[3][row[column]] = scales[at]
            if scores is not None:
                codes[row[column], :, :, 0] = scores[at]
    setup.gpu[0].copy_(codes.to(torch.float8_e4m3fn).cuda())
    setup.gpu[1].copy_((torch.rand(setup.gpu[1].shape, generator=setup.g) / 2 + 0.5).to(torch.float8_e4m3fn).cuda())
    q = setup.randn(setup.tokens, q_heads, dim, std=std).float()
    q[..., 0] = math.log(2.0) * dim ** 0.5 * 16                      # a code of 1 is a score of 1 in log2 units
    return setup, q.bfloat16()


FAR_APART = [
    [2.0 ** -64, 2.0 ** 63],                                         # a page of zeros beside one of values above 2e21
    [2.0 ** 63, 2.0 ** -64, 1.0],
    [2.0 ** 120, 2.0 ** -64],
    [2.0 ** -64, 2.0 ** -64, 2.0 ** -64, 2.0 ** 120, 1.0],
    [1.0] * 9 + [2.0 ** 100, 2.0 ** -60],
    [2.0 ** -33, 1.0, 2.0 ** 33],
    [2.0 ** -105], [2.0 ** -115], [3.0e-35], [2.0 ** 120], [3.0e35],
]
BATCHES = [([1000], 1), ([1000] * 40, 1), ([300] * 90, 2), ([700, 5, 64, 129], 5), ([1000], 40), ([1000] * 12, 40), ([200, 130, 64] * 6, 150)]


@pytest.mark.parametrize("heads", [(16, 2, 256), (16, 2, 128), (8, 8, 64)])
@pytest.mark.parametrize("lengths,new", BATCHES)
def test_value_scales_far_apart_and_far_from_one(package, lengths, new, heads):
    """The weights' sum counts every position alike, whatever its value's scale: in one block, and where several join their parts."""
    for scales in FAR_APART:
        _check_attention(*_scaled(package, lengths, new, heads, scales))


@pytest.mark.parametrize("heads", [(16, 2, 256), (8, 8, 64)])
@pytest.mark.parametrize("lengths,new", [([1000], 1), ([1000] * 40, 2), ([1000], 40), ([1000] * 12, 40)])
def test_small_values_that_the_scores_prefer_to_large_ones(package, lengths, new, heads):
    """The large values' scores are so low that the small ones decide the output, and the other way round."""
    for scales, scores in (([2.0 ** -64, 2.0 ** 60], [0.0, -208.0]), ([2.0 ** 60, 2.0 ** -64, 2.0 ** -50], [-208.0, 8.0, 0.0]),
                           ([2.0 ** -64, 2.0 ** 60], [104.0, 0.0]), ([2.0 ** 100, 2.0 ** -20], [-120.0, 0.0]), ([2.0 ** -64, 2.0 ** 100], [160.0, 0.0])):
        _check_attention(*_scaled(package, lengths, new, heads, scales, scores))


@pytest.mark.parametrize("new", [1, 40])
def test_a_page_of_zeros_beside_one_of_large_values(package, new):
    """As append leaves them: the least scale, and one above 2^100."""
    setup = Setup(package, [256], [256], seed=17, rotary=0)
    k, v = setup.randn(256, 2, 256, std=0.1), setup.randn(256, 2, 256)
    v[:64] = 0.0                                                     # scale 2^-64
    v[128:192] = (v[128:192].float().abs() * 2.0 ** 110).bfloat16()
    setup.cache.append(1, setup.batch, k.cuda(), v.cuda())
    q = setup.randn(256, 16, 256)[:new]
    setup.new, setup.offsets, setup.tokens = [new], [0, new], new
    setup.batch = setup.make_batch()
    _check_attention(setup, q)


@pytest.mark.parametrize("heads", [(16, 2, 256), (16, 2, 128), (8, 8, 64)])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("bad", ["too large", "negative"])
def test_positions_of_a_page_out_of_range_are_left_out(package, heads, new, bad):
    """Whatever the pages that exist hold: all that is of no sequence is NaN here, the first page among it."""
    setup = Setup(package, [150, 90], [new, new], heads, 64, 0, seed=33)
    spare = int(setup.unused[0])
    used = torch.arange(setup.columns)[None, :] < torch.tensor([[3], [2]])
    setup.table[used & (setup.table == 0)] = spare                    # the first page is nobody's
    nobody = torch.ones(len(setup.gpu[0]), dtype=torch.bool)
    nobody[setup.table[used].long()] = False
    for which in (0, 1):
        setup.gpu[which].view(torch.uint8)[nobody.cuda()] = 0x7F
    q = setup.randn(setup.tokens, heads[0], heads[2])
    table = setup.table.clone()
    table[0, 1] = len(setup.gpu[0]) if bad == "too large" else -1
    setup.table, whole = table, setup.table
    setup.batch = setup.make_batch()
    out = setup.cache.attention(1, setup.batch, q.cuda())
    with pytest.raises(package.AimaMoeError) as error:
        setup.cache.sync()
    assert error.value.status == -1
    # the same sequence without the page: its new rows lie behind it
    setup.table = whole.clone()
    setup.table[0, 1] = whole[0, 2]
    setup.lengths[0] -= 64
    setup.batch = setup.make_batch()
    _check_attention(setup, q)
    codes = [t.cpu().float() for t in setup.gpu]
    import kv_oracle

    want, spread = kv_oracle.attention(*codes, setup.table.tolist(), setup.offsets, setup.lengths, q, heads[2] ** -0.5, 64)
    assert ((out.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + spread * (2.0 ** -8 + 2.0 ** -9)).all()


@pytest.mark.parametrize("heads", [(16, 2, 256), (16, 2, 128), (8, 8, 64)])
@pytest.mark.parametrize("length,new", [(300, 1), (257, 2), (300, 30), (385, 140), (1030, 20)])
def test_no_position_is_dropped_or_added(package, heads, length, new):
    """Equal scores, and one position that has a value: a row that sees it returns its share of that value, the others return zero."""
    setup = Setup(package, [length, 130], [new, min(new, 20)], heads, 64, 0, seed=length)
    q = torch.zeros(setup.tokens, heads[0], heads[2]).bfloat16()
    last = length - 1
    for position in sorted({0, 1, 63, 64, 127, 128, 255, 256, last - new, last - new + 1, last - new // 2, last - 1, last} & set(range(length))):
        setup.gpu[1].zero_()
        setup.gpu[1][int(setup.table[0, position // 64]), :, position % 64] = 96.0
        _check_attention(setup, q)


@pytest.mark.parametrize("heads", [(16, 2, 256), (32, 8, 128), (8, 8, 64)])
@pytest.mark.parametrize("lengths,new", [([4000, 700, 33], 1), ([4000, 700, 33], 2), ([2500, 700], 40), ([900], 600)])
def test_distance_from_64_bits(package, heads, lengths, new):
    """Off by the output's rounding to BF16, 2^-9.2 of the norm, and by the weights', of at most 2^-8.7 / sqrt(3) each: by 0.0022 of the
    norm together where a row sees few positions, less where it sees many."""
    import kv_oracle

    setup = Setup(package, lengths, [min(new, n) for n in lengths], heads, 64, 0, seed=sum(lengths))
    q = setup.randn(setup.tokens, heads[0], heads[2], std=1.5).cuda()
    want, _ = kv_oracle.attention(*(t.float() for t in setup.gpu), setup.table.tolist(), setup.offsets, setup.lengths, q, heads[2] ** -0.5, 64)
    got = setup.cache.attention(1, setup.batch, q).double()
    setup.cache.sync()
    assert float((got - want).norm() / want.norm()) <= 0.0022
    # and not the same way everywhere: ties of the weights' last term go up, 2^-12.5 of a weight on the average
    assert abs(float((got * want).sum() / want.square().sum()) - 1.0) <= 2.0 ** -11.5
