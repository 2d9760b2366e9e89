"""GPU parity of the full-attention cache through the C ABI: what an append stores, scales and rotates, and the attention over
it, against oracle/kv_oracle.py in 64 bits.

Tolerances.  A stored element is one rounding of the rotated FP32 value to e4m3: half a step, 2^-4 of its magnitude or 2^-10 of
the scale, and 2^-22 for the FP32 rotation; where a page's scale grew, codes that fell below e4m3's normal range were rounded a
second time (another 2^-10 of the scale).  A rotated query is one rounding to BF16 (2^-8) of an FP32 value.  An attention output
is rounded to BF16 (2^-8); its weights may be held to 8 bits (2^-8 each), and 2^-9 is for scores, exponentials and sums in FP32."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import kv_oracle  # noqa: E402


def _rotation(positions: int, rotary: int) -> torch.Tensor:
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * (1.0e7 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1)))
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


class Setup:
    """A cache of random contents, with sequences of the given lengths (new tokens included) over shuffled pages."""

    def __init__(self, package, lengths, new, heads=(16, 2, 256), page=64, rotary=64, seed=0, spare=3, columns=None, gap=0, scale=0.0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.page, self.heads, self.rotary = g, page, heads, rotary
        q_heads, kv_heads, dim = heads
        counts = [(n + page - 1) // page for n in lengths]
        total = sum(counts) + spare
        order = torch.randperm(total, generator=g)
        self.columns = columns or max(max(counts), 1)
        table = torch.zeros(len(lengths), self.columns, dtype=torch.int32)
        at = 0
        for i, n in enumerate(counts):
            table[i, :n] = order[at:at + n].int()
            at += n
        self.unused = order[at:]
        self.table, self.lengths, self.new = table, list(lengths), list(new)
        self.offsets = [0]
        for n in new:
            self.offsets.append(self.offsets[-1] + n)
        self.tokens = self.offsets[-1] + gap                     # rows of nobody at the end
        codes = [(torch.randn(total, kv_heads, page, dim, generator=g) * 64).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.exp2(-torch.randint(5, 9, (total, kv_heads), generator=g).float()) for _ in range(2)]
        self.cpu = [codes[0], codes[1], scales[0], scales[1]]
        self.gpu = [t.cuda() for t in self.cpu]
        self.cache = package.KvCache(q_heads=q_heads, kv_heads=kv_heads, head_dim=dim, rotary_dim=rotary, page_tokens=page, pages=total,
                                     layers=2, max_sequences=len(lengths), softmax_scale=scale)
        self.cache.bind_layer(1, *self.gpu)
        self.rotation = _rotation(max(max(lengths), 1) + 3, rotary)
        if rotary:
            self.cache.set_rotation(self.rotation.cuda())
        self.batch = self.make_batch()

    def make_batch(self):
        return self.cache.batch(self.table.cuda(), torch.tensor(self.lengths, dtype=torch.int32, device="cuda"), tokens=self.tokens,
                                row_offsets=torch.tensor(self.offsets, dtype=torch.int32, device="cuda"), max_new_tokens=max(max(self.new), 1))

    def randn(self, *shape, std=1.0):
        return (torch.randn(*shape, generator=self.g) * std).bfloat16()

    def wide(self):
        return [t.double() for t in self.cpu]


def _check_append(setup, k, v, q=None, gpu_rows=None):
    want = setup.wide()
    before = [t.clone() for t in want]
    rotation = setup.rotation if setup.rotary else torch.zeros(setup.rotation.shape[0], 0)
    touched = kv_oracle.append(*want, setup.table.tolist(), setup.offsets, setup.lengths, k, v, rotation, setup.page)
    rows = gpu_rows or (k.cuda(), v.cuda(), None if q is None else q.cuda())
    q_out = setup.cache.append(1, setup.batch, rows[0], rows[1], q=rows[2])
    setup.cache.sync()
    got = [t.cpu().double() for t in setup.gpu]
    for which, (codes, scales) in enumerate(((0, 2), (1, 3)), start=1):
        for (page, h), entry in touched.items():
            have, wish, amax = float(got[scales][page, h]), float(want[scales][page, h]), entry["amax%d" % which]
            held = entry["first"] > 0 and float(before[scales][page, h]) >= have
            if which == 2 or have != wish:
                # values pass through untouched, so their scale is exact; a rotated key may sit within FP32 of a power's edge
                edge = 448.0 * max(have, wish) / 2
                assert have == wish or (which == 1 and abs(amax - edge) <= 2.0 ** -20 * edge and not held)
        assert torch.equal(torch.isnan(got[codes]), torch.isnan(want[codes]))
        scale = got[scales][..., None, None]
        have, wish = got[codes] * scale, want[codes] * want[scales][..., None, None]
        exact = torch.nan_to_num(wish)
        bound = torch.zeros_like(exact)
        for (page, h), entry in touched.items():
            for r in entry["rows"]:
                x = torch.nan_to_num(r[which], nan=0.0, posinf=0.0, neginf=0.0)
                if torch.isfinite(got[codes][page, h, r[0]]).all() and not torch.equal(wish[page, h, r[0]], torch.zeros_like(x)):
                    exact[page, h, r[0]] = x
                bound[page, h, r[0]] = torch.maximum(x.abs() * 2.0 ** -4, scale[page, h, 0] * 2.0 ** -10) + x.abs().max() * 2.0 ** -22
            older = before[codes][page, h, :entry["first"]] * before[scales][page, h]
            exact[page, h, :entry["first"]] = older
            grew = float(scale[page, h, 0, 0]) > float(before[scales][page, h])
            bound[page, h, :entry["first"]] = float(scale[page, h, 0, 0]) * 2.0 ** -10 if grew else 0.0
        assert ((torch.nan_to_num(have) - exact).abs() <= bound).all()
        # what no new token goes to stays, scales included
        rest = torch.ones(got[scales].shape, dtype=torch.bool)
        for page, h in touched:
            rest[page, h] = False
        assert torch.equal(got[scales][rest], before[scales][rest])
        assert torch.equal(torch.nan_to_num(got[codes][rest]), torch.nan_to_num(before[codes][rest]))
    if q is not None:
        out = q_out.cpu().double()
        for s, row, position in kv_oracle.rows_of(setup.lengths, setup.offsets):
            x = kv_oracle.rotate(q[row], rotation[position]) if position >= 0 else q[row].double()
            assert ((out[row] - x).abs() <= x.abs() * 2.0 ** -8 + q[row].double().abs().amax() * 2.0 ** -22).all()
    return touched


APPENDS = [
    # lengths with the new tokens, new tokens, heads, page, rotary
    ([1], [1], (16, 2, 256), 64, 64),
    ([64], [1], (16, 2, 256), 64, 64),
    ([65], [1], (16, 2, 256), 64, 256),
    ([68, 63, 5], [5, 5, 5], (16, 2, 256), 64, 64),
    ([137, 0, 16, 333], [130, 0, 16, 1], (4, 4, 128), 16, 128),
    ([300, 129], [300, 2], (8, 1, 64), 128, 0),
    ([31, 33, 32], [31, 2, 32], (6, 2, 128), 32, 48),
    ([1025], [1023], (16, 2, 256), 128, 64),
    ([3, 0, 2], [5, 1, 2], (16, 2, 256), 16, 64),          # rows before the first position are inactive
]


@pytest.mark.parametrize("lengths,new,heads,page,rotary", APPENDS)
def test_append(package, lengths, new, heads, page, rotary):
    setup = Setup(package, lengths, new, heads, page, rotary, seed=len(lengths) * 100 + page, gap=2)
    q_heads, kv_heads, dim = heads
    k, v, q = (setup.randn(setup.tokens, n, dim) for n in (kv_heads, kv_heads, q_heads))
    _check_append(setup, k, v, q)


def test_append_from_one_row_of_a_fused_projection(package):
    setup = Setup(package, [70, 40], [7, 40], seed=3)
    row = setup.randn(setup.tokens, 9216)
    q = row[:, :8192].view(setup.tokens, 16, 512)[:, :, :256]
    k, v = row[:, 8192:8704].view(-1, 2, 256), row[:, 8704:].view(-1, 2, 256)
    wide = row.cuda()
    rows = (wide[:, 8192:8704].view(-1, 2, 256), wide[:, 8704:].view(-1, 2, 256), wide[:, :8192].view(setup.tokens, 16, 512)[:, :, :256])
    _check_append(setup, k, v, q, rows)


@pytest.mark.parametrize("factor", [0.0, 2.0 ** -100, 2.0 ** -60, 2.0 ** -20, 1.0, 50.0, 2.0 ** 60, 2.0 ** 120])
def test_append_scales_from_nothing_to_the_largest(package, factor):
    """A page that holds small tokens has its scale raised by a larger one; zero and tiny pages keep the least scale."""
    setup = Setup(package, [17, 64], [1, 64], (2, 2, 64), 64, 64, seed=9)
    k, v = (setup.randn(setup.tokens, 2, 64) for _ in range(2))
    _check_append(setup, (k.float() * factor).bfloat16(), (v.float() * factor).bfloat16())


def test_append_exact_edges_of_a_scale(package):
    """448 * 2^e takes 2^e, the next BF16 number takes 2^(e+1)."""
    for value, exponent in ((448.0, 0), (450.0, 1), (1.75, -8), (1.7578125, -7), (2.0 ** -70, -64)):
        setup = Setup(package, [8], [8], (1, 1, 64), 16, 0, seed=1)
        v = torch.zeros(8, 1, 64).bfloat16()
        v[3, 0, 5] = -value
        _check_append(setup, v, v)
        assert setup.gpu[3].cpu()[int(setup.table[0, 0]), 0] == 2.0 ** exponent


def test_append_of_the_largest_values(package):
    """Above 448 * 2^119 (2.98e38) a page needs the scale 2^120; BF16 ends at 3.39e38."""
    setup = Setup(package, [40, 70], [5, 70], rotary=0, seed=8)
    k, v = (setup.randn(setup.tokens, 2, 256) for _ in range(2))
    largest = torch.finfo(torch.bfloat16).max
    k[3], v[3, 1], k[40, 0, 7], v[60, 0, 0] = largest, -largest, -3.0e38, 2.97e38
    _check_append(setup, k, v, gpu_rows=(k.cuda(), v.cuda(), None))


def test_append_token_by_token_stores_what_one_call_stores(package):
    """Powers of two: a page filled one token at a time ends with the scale, and up to codes below the normal range the codes, of
    a page filled at once."""
    lengths = [48]
    whole = Setup(package, lengths, [48], (2, 2, 128), 16, 64, seed=5)
    steps = Setup(package, lengths, [48], (2, 2, 128), 16, 64, seed=5)
    k, v = (whole.randn(48, 2, 128, std=3.0) for _ in range(2))
    whole.cache.append(1, whole.batch, k.cuda(), v.cuda())
    for i in range(48):
        batch = steps.cache.batch(steps.table.cuda(), torch.tensor([i + 1], dtype=torch.int32, device="cuda"), tokens=1)
        steps.cache.append(1, batch, k[i:i + 1].cuda(), v[i:i + 1].cuda())
    for a, b, scale in ((0, 0, 2), (1, 1, 3)):
        x, y = whole.gpu[a].cpu().float(), steps.gpu[b].cpu().float()
        pages = whole.table[0].long()
        assert torch.equal(whole.gpu[scale].cpu()[pages], steps.gpu[scale].cpu()[pages])
        assert ((x[pages] - y[pages]).abs() <= torch.where(x[pages].abs() < 2.0 ** -6, 2.0 ** -9, 0.0)).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_token_that_is_not_finite_reaches_only_the_rows_that_see_it(package, bad):
    setup = Setup(package, [40], [10], seed=11)
    k, v, q = setup.randn(10, 2, 256), setup.randn(10, 2, 256), setup.randn(10, 16, 256)
    k[4, 1, 200] = bad
    v[7, 0, 3] = bad
    _check_append(setup, k, v)
    out = setup.cache.attention(1, setup.batch, q.cuda()).cpu()
    setup.cache.sync()
    lost = torch.zeros(10, 16, dtype=torch.bool)
    lost[4:, 8:] = True
    lost[7:, :8] = True
    assert torch.equal(torch.isnan(out).all(-1), lost) and torch.equal(torch.isnan(out).any(-1), lost)


def _check_attention(setup, q, gpu_q=None):
    codes = [t.cpu().float() for t in setup.gpu]
    scale = setup.cache.config.softmax_scale or setup.heads[2] ** -0.5
    want, spread = kv_oracle.attention(*codes, setup.table.tolist(), setup.offsets, setup.lengths, q, scale, setup.page)
    out = torch.full((setup.tokens, *q.shape[1:]), 7.0, dtype=torch.bfloat16, device="cuda")
    setup.cache.attention(1, setup.batch, q.cuda() if gpu_q is None else gpu_q, out=out)
    setup.cache.sync()
    got = out.cpu().double()
    owned = setup.offsets[-1]
    assert (got[owned:] == 7.0).all()                            # rows of no sequence are not written
    assert torch.isfinite(got).all()
    bound = want.abs() * 2.0 ** -8 + spread * (2.0 ** -8 + 2.0 ** -9)
    worst = ((got - want).abs() - bound)[:owned].max()
    assert worst <= 0, f"beyond the bound by {float(worst)}"


ATTENTIONS = [
    # lengths, new, heads, page
    ([1], [1], (16, 2, 256), 64),
    ([2], [1], (16, 2, 256), 16),
    ([127, 128, 129, 1, 0, 500], [1, 1, 1, 1, 1, 1], (16, 2, 256), 64),
    ([4097], [1], (16, 2, 256), 128),
    ([5000, 3, 777], [1, 1, 1], (16, 2, 256), 16),
    ([1000, 130, 5], [5, 5, 5], (16, 2, 256), 64),
    ([700, 129, 8], [8, 3, 8], (16, 2, 256), 32),
    ([3, 0, 300], [5, 2, 4], (16, 2, 256), 64),                  # rows that see nothing
    ([333, 64], [1, 1], (5, 5, 128), 32),                        # one query head per key/value head
    ([333, 64, 1000], [2, 1, 2], (12, 4, 128), 64),
    ([1500, 90], [1, 1], (32, 1, 64), 16),
    ([260, 90], [3, 2], (24, 1, 64), 128),
    ([257], [9], (7, 1, 256), 64),
    ([200], [1], (128, 1, 128), 64),
    ([33], [33], (16, 2, 256), 64),
    ([700, 129, 0, 40], [300, 129, 0, 17], (16, 2, 256), 64),
    ([900, 513], [513, 100], (8, 8, 64), 16),
    ([1111], [257], (6, 2, 128), 128),
]


@pytest.mark.parametrize("lengths,new,heads,page", ATTENTIONS)
def test_attention(package, lengths, new, heads, page):
    setup = Setup(package, lengths, new, heads, page, 0, seed=sum(lengths) + page, gap=1)
    _check_attention(setup, setup.randn(setup.tokens, heads[0], heads[2], std=1.5))


@pytest.mark.parametrize("new", [1, 5, 40])
def test_attention_of_strided_queries(package, new):
    setup = Setup(package, [300, 77], [new, new], seed=21)
    wide = setup.randn(setup.tokens, 16, 512)
    _check_attention(setup, wide[:, :, :256], wide.cuda()[:, :, :256])


OTHER_HEADS = [(16, 2, 128), (24, 8, 128), (16, 2, 64), (8, 8, 64)]


@pytest.mark.parametrize("new", [1, 40, 150])
@pytest.mark.parametrize("heads", OTHER_HEADS)
def test_scores_and_values_of_other_head_sizes(package, heads, new):
    """Sharp scores, rising ones, a sink whose value is zero, NaN behind the sequences, and rows of every size."""
    setup = Setup(package, [400, 129, 200], [new, min(new, 100), new], heads, 64, 0, seed=new + heads[2])
    h, kv_heads, dim = heads
    q = setup.randn(setup.tokens, h, dim, std=8.0)
    for which in (0, 1):
        raw = setup.gpu[which].view(torch.uint8)
        for s, n in enumerate(setup.lengths):
            raw[int(setup.table[s, (n - 1) // 64]), :, n % 64 or 64:] = 0x7F
        raw[setup.unused.cuda()] = 0xFF
    _check_attention(setup, q)
    q[0, 0] *= 2.0 ** -100
    q[0, 1, 7] = 900.0
    q[0, 2] = 0.0
    _check_attention(setup, q)
    setup = Setup(package, [1024], [new], heads, 64, 0, seed=42)
    q = torch.zeros(new, h, dim).bfloat16()
    q[..., 0] = 4.0 * dim ** 0.5 / 16
    codes = setup.gpu[0].cpu().float()
    setup.gpu[2].fill_(2.0 ** -4)
    for i, page in enumerate(setup.table[0].tolist()):
        codes[page, :, :, 0] = torch.arange(64) * 0.5 + 32.0 * i - 256
    setup.gpu[0].copy_(codes.to(torch.float8_e4m3fn).cuda())
    _check_attention(setup, q)
    codes[..., :] = 0.0
    codes[int(setup.table[0, 0]), :, 3, 0] = 448.0
    setup.gpu[0].copy_(codes.to(torch.float8_e4m3fn).cuda())
    setup.gpu[1].view(torch.uint8)[int(setup.table[0, 0]), :, 3] = 0
    q[..., 0] = 8.0 * dim ** 0.5 / 16
    _check_attention(setup, q)


@pytest.mark.parametrize("heads", OTHER_HEADS)
@pytest.mark.parametrize("new", [3, 30])
def test_not_finite_tokens_and_queries_of_other_head_sizes(package, heads, new):
    h, kv_heads, dim = heads
    setup = Setup(package, [150], [new], heads, 64, 64, seed=12)
    k, v, q = setup.randn(new, kv_heads, dim), setup.randn(new, kv_heads, dim), setup.randn(new, h, dim)
    k[new - 2, 1, dim - 1] = math.nan
    v[new - 1, 0, 3] = math.inf
    q[0, h - 1, 5] = math.nan
    _check_append(setup, k, v)
    out = setup.cache.attention(1, setup.batch, q.cuda()).cpu()
    setup.cache.sync()
    lost = torch.zeros(new, h, dtype=torch.bool)
    lost[new - 2:, h // kv_heads:2 * h // kv_heads] = True
    lost[new - 1, :h // kv_heads] = True
    lost[0, h - 1] = True
    assert torch.equal(torch.isnan(out).all(-1), lost) and torch.equal(torch.isnan(out).any(-1), lost)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("heads", [(16, 2, 256), (6, 2, 128), (8, 8, 64)])
@pytest.mark.parametrize("layout", ["heads first", "one row for all", "one head for all", "rows that are no multiple of heads"])
def test_queries_of_any_strides(package, new, heads, layout):
    setup = Setup(package, [300, 77], [new, new], heads, seed=22)
    n, (h, _, dim) = setup.tokens, heads
    if layout == "heads first":
        gpu = setup.randn(h, n, dim).cuda().transpose(0, 1)
    elif layout == "one row for all":
        gpu = setup.randn(1, h, dim).cuda().expand(n, h, dim)
    elif layout == "one head for all":
        gpu = setup.randn(n, 1, dim).cuda().expand(n, h, dim)
    else:
        gpu = setup.randn(n, h * dim + 8).cuda()[:, :h * dim].unflatten(1, (h, dim))
    _check_attention(setup, gpu.cpu(), gpu)


def test_strides_of_a_single_row_or_head_are_not_looked_at(package):
    setup = Setup(package, [300], [1], seed=23)
    q = setup.randn(1, 16, 256)
    _check_attention(setup, q, torch.as_strided(q.cuda(), (1, 16, 256), (3, 256, 1)))
    setup = Setup(package, [300], [200], (1, 1, 128), seed=24)
    q = setup.randn(200, 1, 128)
    _check_attention(setup, q, torch.as_strided(q.cuda(), (200, 1, 128), (128, 3, 1)))


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("std", [0.0, 1.0e-3, 30.0])
def test_attention_of_flat_and_sharp_scores(package, std, new):
    setup = Setup(package, [1300], [new], seed=31)
    _check_attention(setup, setup.randn(setup.tokens, 16, 256, std=std))


@pytest.mark.parametrize("new", [1, 40])
def test_attention_of_rising_scores_and_a_sink(package, new):
    """The running maximum moves at every tile; then one early key outweighs everything by 2^20, and its value is zero, so the
    output is what the small weights give."""
    setup = Setup(package, [1024], [new], (16, 2, 256), 64, 0, seed=41)
    q = torch.zeros(new, 16, 256).bfloat16()
    q[..., 0] = 4.0
    codes = setup.gpu[0].cpu().float()
    pages = setup.table[0].long()
    setup.gpu[2].fill_(2.0 ** -4)
    for i, page in enumerate(pages.tolist()):
        codes[page, :, :, 0] = torch.arange(64) * 0.5 + 32.0 * i - 256
    setup.gpu[0].copy_(codes.to(torch.float8_e4m3fn).cuda())
    _check_attention(setup, q)
    codes[..., 0] = 0.0
    codes[int(pages[0]), :, 3, 0] = 448.0
    codes[..., 1:] = 0.0
    setup.gpu[0].copy_(codes.to(torch.float8_e4m3fn).cuda())
    setup.gpu[1].view(torch.uint8)[int(pages[0]), :, 3] = 0
    q[..., 0] = 8.0                                               # 448 / 16 * 8 / 16 = 14 nats
    _check_attention(setup, q)


@pytest.mark.parametrize("new", [1, 6, 40])
def test_attention_ignores_what_lies_behind_a_sequence(package, new):
    """Codes behind the length, in the last page and in unused ones, are NaN; scales of unused pages too."""
    setup = Setup(package, [70, 129, 200], [new, new, new], seed=51)
    q = setup.randn(setup.tokens, 16, 256)
    for which in (0, 1):
        raw = setup.gpu[which].view(torch.uint8)
        for s, n in enumerate(setup.lengths):
            raw[int(setup.table[s, (n - 1) // 64]), :, n % 64 or 64:] = 0x7F
        raw[setup.unused.cuda()] = 0xFF
        setup.gpu[which + 2][setup.unused.cuda()] = math.nan
    _check_attention(setup, q)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_takes_any_positive_scale(package, new):
    setup = Setup(package, [500, 60], [new, new], seed=61)
    for which in (2, 3):
        setup.gpu[which].copy_((torch.rand(setup.gpu[which].shape, generator=setup.g) * 0.03 + 1.0e-4).cuda())
    _check_attention(setup, setup.randn(setup.tokens, 16, 256))
    setup.gpu[3].mul_(2.0 ** torch.randint(-50, 50, setup.gpu[3].shape, generator=setup.g).float().cuda())
    _check_attention(setup, setup.randn(setup.tokens, 16, 256))


@pytest.mark.parametrize("new", [1, 40])
def test_queries_of_any_size(package, new):
    """Rows of 2^-100, 2^40 and with one element that dwarfs the rest; a NaN stays in its row."""
    setup = Setup(package, [400], [new], seed=71)
    q = setup.randn(new, 16, 256)
    q[0, 0] *= 2.0 ** -100
    q[0, 1, 7] = 900.0
    q[0, 2] = 0.0
    _check_attention(setup, q)
    q[0, 3, 5] = math.nan
    q[0, 9, 250] = math.inf
    out = setup.cache.attention(1, setup.batch, q.cuda()).cpu()
    lost = torch.isnan(out)
    assert lost[0, 3].all() and lost[0, 9].all() and int(lost.any(-1).sum()) == 2


@pytest.mark.parametrize("new", [1, 300])
def test_softmax_scale_and_repeatability(package, new):
    setup = Setup(package, [900, 333], [new, min(new, 33)], seed=81, scale=0.21)
    q = setup.randn(setup.tokens, 16, 256)
    _check_attention(setup, q)
    a = setup.cache.attention(1, setup.batch, q.cuda())
    b = setup.cache.attention(1, setup.batch, q.cuda())
    assert torch.equal(a, b)


def test_offsets_beyond_32_bits(package):
    """A pool of 5 GB per tensor whose last pages are in use."""
    page, kv_heads, dim = 128, 2, 256
    pages = 80000                                                 # 80000 * 2 * 128 * 256 B = 5.2e9
    g = torch.Generator().manual_seed(5)
    cache = package.KvCache(q_heads=16, kv_heads=2, head_dim=256, rotary_dim=64, page_tokens=page, pages=pages, max_sequences=2)
    tensors = cache.allocate_layer()
    cache.bind_layer(0, *tensors)
    rotation = _rotation(512, 64)
    cache.set_rotation(rotation.cuda())
    table = torch.tensor([[pages - 1, 0, pages - 3], [pages - 2, 1, pages - 4]], dtype=torch.int32)
    lengths, rows = [300, 257], 600
    offsets = [0, 300, 557]
    batch = cache.batch(table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), tokens=rows,
                        row_offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    k, v, q = (torch.randn(rows, n, dim, generator=g).bfloat16() for n in (2, 2, 16))
    turned = cache.append(0, batch, k.cuda(), v.cuda(), q=q.cuda())
    small = torch.unique(table.flatten().long())
    remap = {int(p): i for i, p in enumerate(small)}
    near = [[remap[int(p)] for p in row] for row in table]
    part = [t.view(torch.uint8)[small.cuda()].view(torch.float8_e4m3fn).cpu().float() if t.dtype == torch.float8_e4m3fn else t[small.cuda()].cpu() for t in tensors]
    want = [torch.zeros(t.shape, dtype=torch.float64) for t in part]
    kv_oracle.append(*want, near, offsets, lengths, k, v, rotation, page)
    assert torch.equal(part[3].double(), want[3])
    assert float((part[1].double() - want[1]).abs().max()) == 0.0  # values pass through untouched
    for n in (1, 40):
        last = torch.cat([turned[300 - n:300], turned[557 - n:557]])
        step = cache.batch(table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), tokens=2 * n)
        out = cache.attention(0, step, last).cpu().double()
        cache.sync()
        o, spread = kv_oracle.attention(*part, near, [0, n, 2 * n], lengths, last.cpu(), dim ** -0.5, page)
        assert ((out - o).abs() <= o.abs() * 2.0 ** -8 + spread * (2.0 ** -8 + 2.0 ** -9)).all()
    cache.release()


def test_another_stream_and_a_captured_graph(package):
    """The batch is read on the device: a graph replayed after the lengths moved attends to the new ones."""
    setup = Setup(package, [100, 260], [1, 1], seed=91)
    q = setup.randn(2, 16, 256).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(q)
    with torch.cuda.stream(stream):
        setup.cache.attention(1, setup.batch, q, out=out)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        setup.cache.attention(1, setup.batch, q, out=out)
    for lengths in ([100, 260], [64, 257], [1, 0]):
        setup.batch.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        codes = [t.cpu().float() for t in setup.gpu]
        want, spread = kv_oracle.attention(*codes, setup.table.tolist(), setup.offsets, lengths, q.cpu(), 1 / 16, 64)
        assert ((out.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + spread * (2.0 ** -8 + 2.0 ** -9)).all()


def test_a_handle_of_a_side_stream_and_its_release_with_work_under_way(package):
    """The workspace comes from the stream that is current at creation and goes back without a wait: what is still under way on
    another stream keeps it."""
    setup = Setup(package, [3000, 2000], [40, 40], seed=92)
    q = setup.randn(80, 16, 256).cuda()
    want = setup.cache.attention(1, setup.batch, q)
    torch.cuda.synchronize()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(first):
        scratch = [torch.full((1 << 24,), 0x7f7f7f7f, dtype=torch.int32, device="cuda") for _ in range(4)]
        del scratch                                              # memory that is written when the handle is made from it
        cache = package.KvCache(rotary_dim=0, pages=setup.cache.config.pages, layers=2, max_sequences=2)
        cache.bind_layer(1, *setup.gpu)
    with torch.cuda.stream(second):
        outs = [cache.attention(1, setup.batch, q) for _ in range(50)]
        cache.release()
    with torch.cuda.stream(first):
        scratch = [torch.full((1 << 24,), 0x7f7f7f7f, dtype=torch.int32, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)


def test_workspace_of_the_callers(package):
    import ctypes

    setup = Setup(package, [300, 77], [1, 1], seed=93)
    q = setup.randn(2, 16, 256).cuda()
    want = setup.cache.attention(1, setup.batch, q)
    lib, provider = setup.cache.lib, package.provider
    size, handle = ctypes.c_uint64(), ctypes.c_void_p()
    config = provider.KvConfig.from_buffer_copy(setup.cache.config)
    assert lib.aima_moe_kv_query_workspace(ctypes.byref(config), ctypes.byref(size)) == 0 and size.value == config.workspace_bytes
    memory = torch.full((size.value + 256,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for pointer, given in ((memory.data_ptr(), size.value - 1), (memory.data_ptr() + 16, size.value),
                           (torch.empty(64, dtype=torch.uint8).data_ptr() // 256 * 256, size.value)):
        config.workspace, config.workspace_bytes = pointer, given
        assert lib.aima_moe_kv_prepare(ctypes.byref(config), ctypes.byref(handle)) == -1 and not handle.value
    for pointer, given in ((memory.data_ptr(), size.value), (None, 0)):          # the caller's, and one that prepare allocates
        config.workspace, config.workspace_bytes = pointer, given
        lib.check(lib.aima_moe_kv_prepare(ctypes.byref(config), ctypes.byref(handle)))
        kept, setup.cache.handle = setup.cache.handle, handle
        setup.cache.bind_layer(1, *setup.gpu)
        out = setup.cache.attention(1, setup.batch, q)
        setup.cache.sync()
        setup.cache.handle = kept
        assert torch.equal(out, want)
        assert lib.aima_moe_kv_release(handle) == 0
    assert (memory[size.value:] == 255).all()


@pytest.mark.parametrize("new", [1, 40])
def test_device_data_out_of_range_is_reported_and_harmless(package, new):
    """Lengths, offsets and page numbers are only known on the device: each is held to its range there, the other sequences keep
    their results and the next call is clean."""
    setup = Setup(package, [200, 150], [new, new], seed=101)
    q, k, v = setup.randn(2 * new, 16, 256).cuda(), setup.randn(2 * new, 2, 256).cuda(), setup.randn(2 * new, 2, 256).cuda()
    right = setup.cache.attention(1, setup.batch, q).clone()
    before = [t.view(torch.uint8).clone() for t in setup.gpu]

    def refused():
        with pytest.raises(package.AimaMoeError) as error:
            setup.cache.sync()
        assert error.value.status == -1
        setup.cache.sync()

    for lengths in ([200, 64 * setup.columns + 1], [200, -1]):
        bad = setup.cache.batch(setup.table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), tokens=2 * new)
        out = setup.cache.attention(1, bad, q)
        assert torch.equal(out[:new], right[:new]) and not out[new:].any()
        refused()
    table = setup.table.clone()
    table[1, 1] = len(setup.gpu[0])
    bad = setup.cache.batch(table.cuda(), setup.batch.lengths, tokens=2 * new)
    assert torch.equal(setup.cache.attention(1, bad, q)[:new], right[:new])
    refused()
    offsets = torch.tensor([0, new, 2 * new + 1], dtype=torch.int32, device="cuda")
    bad = setup.cache.batch(setup.table.cuda(), setup.batch.lengths, tokens=2 * new, row_offsets=offsets, max_new_tokens=2 * new)
    assert torch.equal(setup.cache.attention(1, bad, q)[:new], right[:new])
    refused()
    bad = setup.cache.batch(setup.table.cuda(), torch.tensor([-5, 64 * setup.columns + 1], dtype=torch.int32, device="cuda"), tokens=2 * new)
    setup.cache.append(1, bad, k, v)
    refused()
    assert all(torch.equal(x, y.view(torch.uint8)) for x, y in zip(before, setup.gpu))
    assert torch.equal(setup.cache.attention(1, setup.batch, q), right)
    setup.cache.sync()


def test_refusals(package):
    setup = Setup(package, [200, 150], [1, 1], seed=111)
    cache, batch = setup.cache, setup.batch
    q, k, v = setup.randn(2, 16, 256).cuda(), setup.randn(2, 2, 256).cuda(), setup.randn(2, 2, 256).cuda()

    def status(call):
        with pytest.raises(package.AimaMoeError) as error:
            call()
        return error.value.status

    assert status(lambda: cache.attention(0, batch, q)) == -3     # layer 0 was never bound
    assert status(lambda: cache.attention(2, batch, q)) == -1
    assert status(lambda: cache.attention(1, batch, q, out=q)) == -4
    assert status(lambda: cache.append(1, batch, k, v, q=q, q_out=q)) == -4
    shifted = torch.empty(2 * 16 * 256 + 8, dtype=torch.bfloat16, device="cuda")[1:1 + 2 * 16 * 256].view(2, 16, 256)
    assert status(lambda: cache.attention(1, batch, shifted)) == -1
    assert status(lambda: cache.attention(1, batch, q, out=shifted)) == -1
    odd = torch.empty(2, 2, 260, dtype=torch.bfloat16, device="cuda")[:, :, :256]
    assert status(lambda: cache.append(1, batch, odd, v)) == -1
    three = cache.batch(torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), tokens=3)
    assert status(lambda: cache.attention(1, three, setup.randn(3, 16, 256).cuda())) == -8
    unrotated = package.KvCache(pages=4)
    unrotated.bind_layer(0, *unrotated.allocate_layer())
    assert status(lambda: unrotated.append(0, batch, k, v)) == -3
    with pytest.raises(package.AimaMoeError) as error:
        unrotated.bind_layer(0, *[t[:3] for t in unrotated.allocate_layer()])
    assert error.value.status == -1 and "bytes" in str(error.value)
    for wrong in (q.float(), q[:, :8], q[:1]):
        with pytest.raises(ValueError):
            cache.attention(1, batch, wrong)
    with pytest.raises(ValueError):
        cache.append(1, batch, k.transpose(1, 2).contiguous().transpose(1, 2), v)
    with pytest.raises(ValueError):
        cache.batch(setup.table.cuda().long(), setup.batch.lengths, tokens=2)
    for bad in (dict(head_dim=96), dict(page_tokens=48), dict(kv_heads=3), dict(rotary_dim=40), dict(max_sequences=0), dict(pages=1 << 30)):
        with pytest.raises(package.AimaMoeError):
            package.KvCache(**{"pages": 4, **bad})
