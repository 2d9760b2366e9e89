"""GPU tests of what ties an attention launch's blocks together: the join of a unit's parts against its formula in 64 bits, a part that
never comes, the status and counters after it, and two handles at work on two streams."""
from __future__ import annotations

import ctypes
import math
import shutil
import subprocess

import pytest
import torch

from conftest import PACKAGE_DIR, ROOT
from test_kv_cache_gpu import Setup, _check_attention

pytestmark = pytest.mark.gpu

BLOCKS, PART_ROWS = 160, 128


@pytest.fixture(scope="module")
def join(tmp_path_factory):
    path = tmp_path_factory.mktemp("join") / "libkv_join_probe.so"
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-std=c++17", "-O3", "-shared", "-Xcompiler", "-fPIC", "-gencode", "arch=compute_100a,code=sm_100a",
                    "-I", str(PACKAGE_DIR / "csrc"), "-o", str(path), str(ROOT / "tests" / "kv_join_probe.cu")], check=True)
    run = ctypes.CDLL(str(path)).run_join
    run.argtypes = [ctypes.c_void_p] * 5 + [ctypes.c_int] * 5 + [ctypes.c_uint64, ctypes.c_void_p]
    return run


class Parts:
    """A unit of `rows` rows in `parts` blocks, laid out as the attention kernels leave it."""

    def __init__(self, parts, rows, dim, group, tops, lows, seed=1):
        g = torch.Generator().manual_seed(seed)
        self.parts, self.rows, self.dim, self.group = parts, rows, dim, group
        self.o = torch.randn(parts, rows, dim, generator=g, dtype=torch.float64).float()
        self.d = (torch.rand(parts, rows, generator=g) + 0.5)
        self.tops, self.lows = tops.expand(parts, rows).contiguous().float(), lows.expand(parts, rows).contiguous().float()
        weights, sums = torch.zeros(2 * BLOCKS, PART_ROWS, 4), torch.zeros(2 * BLOCKS, dim // 4, PART_ROWS, 4)
        for p in range(parts):
            at = 2 * p + (1 if p == 0 else 0)
            weights[at, :rows, 0], weights[at, :rows, 1], weights[at, :rows, 2] = self.tops[p], self.d[p], self.lows[p]
            sums[at, :, :rows] = self.o[p].view(rows, dim // 4, 4).transpose(0, 1)
        self.weights, self.sums = weights.cuda(), sums.cuda()
        self.arrived = torch.zeros(2, dtype=torch.int32, device="cuda")
        self.status, self.verdict = (torch.full((1,), v, dtype=torch.int32, device="cuda") for v in (0, -1))
        self.out = torch.full((rows // group, group, dim), 7.0, dtype=torch.bfloat16, device="cuda")

    def run(self, join, mine, limit_ns=1_000_000):
        torch.cuda.synchronize()
        assert join(self.out.data_ptr(), self.status.data_ptr(), self.arrived.data_ptr(), self.weights.data_ptr(), self.sums.data_ptr(), self.dim,
                    self.group, self.rows, self.parts, mine, limit_ns, self.verdict.data_ptr()) == 0
        return int(self.verdict)

    def want(self):
        """sum O_p 2^top_p / sum D_p 2^low_p, and the same over |O_p|."""
        top, low = self.tops.double().amax(0), self.lows.double().amax(0)
        o = (self.o.double() * torch.exp2(self.tops.double() - top)[..., None]).sum(0)
        spread = (self.o.double().abs() * torch.exp2(self.tops.double() - top)[..., None]).sum(0)
        d = (self.d.double() * torch.exp2(self.lows.double() - low)).sum(0)
        back = torch.exp2(top - low)[:, None]
        shape = self.out.shape
        return (o / d[:, None] * back).view(shape), (spread / d[:, None] * back).view(shape)


@pytest.mark.parametrize("parts", [2, 3, 4, 5, 8, 9, 33, 74, 160])
@pytest.mark.parametrize("rows,group,dim", [(8, 8, 256), (40, 8, 256), (128, 1, 64), (3, 3, 64)])
def test_join(join, parts, rows, group, dim):
    """References near each other, far apart, and of parts that a row does not see."""
    g = torch.Generator().manual_seed(parts)
    near = torch.randn(parts, rows, generator=g) * 3
    far = torch.randn(parts, rows, generator=g) * 60
    unseen = near.clone()
    unseen[torch.rand(parts, rows, generator=g) < 0.4] = -math.inf
    unseen[0] = near[0]
    far -= far.amax(0)
    for tops, lows in ((near, near - 5), (near, near + 100), (near + 90, near), (far, near), (unseen, unseen + 7), (near, far)):
        parts_ = Parts(parts, rows, dim, group, tops, lows)
        parts_.d[parts_.tops == -math.inf] = 0.0
        parts_.o[parts_.tops == -math.inf] = 0.0
        parts_ = _relay(parts_)
        parts_.arrived[0] = parts
        for mine in range(parts):
            assert parts_.run(join, mine) == 1
        assert int(parts_.status) == 0 and parts_.arrived.tolist() == [0, 0]      # the last to leave put them back
        want, spread = parts_.want()
        # BF16's rounding; exponentials, products and sums in FP32, of up to 160 terms
        assert ((parts_.out.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + spread * 2.0 ** -16 + 2.0 ** -133).all()


def _relay(parts):
    """Lays changed sums out again."""
    for p in range(parts.parts):
        at = 2 * p + (1 if p == 0 else 0)
        parts.weights[at, :parts.rows, 1] = parts.d[p].cuda()
        parts.sums[at, :, :parts.rows] = parts.o[p].view(parts.rows, parts.dim // 4, 4).transpose(0, 1).cuda()
    return parts


@pytest.mark.parametrize("parts", [2, 6, 74])
def test_a_part_that_never_comes_ends_in_a_status(join, parts):
    level = torch.zeros(parts, 8)
    unit = Parts(parts, 8, 256, 8, level, level)
    unit.arrived[0] = parts - 1
    assert unit.run(join, 0, limit_ns=200_000) == 0
    assert int(unit.status) == 2 and unit.arrived.tolist() == [parts - 1, 0]
    assert (unit.out == 7.0).all()


def test_sync_after_a_wait_that_ran_out(package):
    """What such a launch leaves, a status and counters that are not zero, is reported once, and the next call is right."""
    setup = Setup(package, [3000, 500], [1, 1], seed=7)
    q = setup.randn(2, 16, 256)
    _check_attention(setup, q)
    want = setup.cache.attention(1, setup.batch, q.cuda())
    setup.cache.sync()
    words = setup.cache._workspace[:1024].view(torch.int32)
    words[0] = 2
    words[64:80] = 3
    torch.cuda.synchronize()
    with pytest.raises(package.AimaMoeError) as error:
        setup.cache.sync()
    assert error.value.status == -5
    assert not words.any()
    assert torch.equal(setup.cache.attention(1, setup.batch, q.cuda()), want)
    setup.cache.sync()


@pytest.mark.parametrize("new", [1, 40])
def test_two_handles_on_two_streams(package, new):
    """Each has a workspace of its own; what they compute does not depend on what runs beside them."""
    setups = [Setup(package, [3000, 700, 64], [new, new, min(new, 30)], seed=seed) for seed in (8, 9)]
    qs = [s.randn(s.tokens, 16, 256).cuda() for s in setups]
    want = [s.cache.attention(1, s.batch, q) for s, q in zip(setups, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in setups]
    outs = [[], []]
    for _ in range(20):
        for i, (s, q) in enumerate(zip(setups, qs)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(s.cache.attention(1, s.batch, q))
    for s in setups:
        s.cache.sync()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i in range(2) for out in outs[i])
