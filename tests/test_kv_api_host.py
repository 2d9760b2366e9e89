"""The full-attention cache's C ABI (csrc/kv_api.cu) over a CUDA runtime made for it, tests/kv_api_fake.cpp: what the entries check
and order by themselves, without a device."""
from __future__ import annotations

import ctypes
import shutil
import subprocess

import pytest

from conftest import PACKAGE_DIR, ROOT

BASE = 1 << 40                # of addresses that nothing reads


@pytest.fixture(scope="module")
def lib(package, tmp_path_factory):
    path = tmp_path_factory.mktemp("kv") / "libkv_api_fake.so"
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-std=c++17", "-O1", "-shared", "-cudart", "none", "-Xlinker", "-Bsymbolic", "-Xcompiler", "-fPIC", "-gencode", "arch=compute_100a,code=sm_100a",
                    "-I", str(PACKAGE_DIR / "csrc"), "-o", str(path), str(PACKAGE_DIR / "csrc" / "kv_api.cu"), str(ROOT / "tests" / "kv_api_fake.cpp")],
                   check=True)
    lib = ctypes.CDLL(str(path))
    for name, restype, argtypes in package.provider.EXPORTS:
        if name.startswith("aima_moe_kv_"):
            getattr(lib, name).restype, getattr(lib, name).argtypes = restype, argtypes
    lib.fake_leave.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]
    lib.fake_message.restype, lib.fake_cleared.restype = ctypes.c_char_p, ctypes.c_uint64
    return lib


class Handle:
    """A handle of one layer on the fake's device, with 4 query heads and 2 key/value heads of 64."""

    def __init__(self, package, lib, device=0):
        p, self.lib = package.provider, lib
        lib.fake_device(device)
        config = p.KvConfig(ctypes.sizeof(p.KvConfig), 4, 2, 64, 0, 16, 8, 1, 4, 0.0, None, 0)
        size = ctypes.c_uint64()
        assert lib.aima_moe_kv_query_workspace(ctypes.byref(config), ctypes.byref(size)) == 0
        self.memory = (ctypes.c_uint8 * (size.value + 256))()
        at = (ctypes.addressof(self.memory) + 255) // 256 * 256
        config.workspace, config.workspace_bytes = at, size.value
        self.handle = ctypes.c_void_p()
        owner = ctypes.c_void_p()
        lib.cudaMalloc(ctypes.byref(owner), ctypes.c_size_t(16))              # what follows is of this device
        lib.cudaFree(owner)
        assert lib.aima_moe_kv_prepare(ctypes.byref(config), ctypes.byref(self.handle)) == 0, lib.fake_message()
        self.status = ctypes.cast(at, ctypes.POINTER(ctypes.c_int))
        codes, scales = 8 * 2 * 16 * 64, 8 * 2 * 4
        layer = p.KvLayer(ctypes.sizeof(p.KvLayer), 0, BASE, codes, BASE, codes, BASE, scales, BASE, scales)
        assert lib.aima_moe_kv_bind_layer(self.handle, 0, ctypes.byref(layer)) == 0
        self.p = p

    def batch(self, tokens):
        return self.p.KvBatchStruct(ctypes.sizeof(self.p.KvBatchStruct), 1, tokens, tokens, 8, 0, BASE, None, BASE)

    def append(self, tokens, k, v, q, q_out, stream=None):
        """k, v, q: (offset in bytes, row stride, head stride); q_out: an offset."""
        rows = [self.p.KvRows(BASE + at, row, head) for at, row, head in (k, v, q)]
        return self.lib.aima_moe_kv_append_launch(self.handle, 0, ctypes.byref(self.batch(tokens)), *rows, BASE + q_out, stream)


ROW = 4 * 64 * 2              # bytes of a contiguous row of queries; of keys or values half of it


@pytest.mark.parametrize("tokens", [1, 5])
def test_rotated_queries_may_not_lie_over_any_input(package, lib, tokens):
    """Keys and values are read by the launch that writes the queries."""
    h = Handle(package, lib)
    size, half = tokens * ROW, tokens * ROW // 2
    k, v, q = (size, 128, 64), (size + half, 128, 64), (0, 256, 64)
    before = lib.fake_appends()
    assert h.append(tokens, k, v, q, 2 * size) == 0                           # behind all of them
    assert lib.fake_appends() == before + 1
    for q_out in (0, size - 16, size, size + 16, size + half, 2 * size - 16):
        assert h.append(tokens, k, v, q, q_out) == -4, q_out
        assert b"overlaps" in lib.fake_message()
    # before all of them, and one input at a time
    assert h.append(tokens, (3 * size, 128, 64), (4 * size, 128, 64), (2 * size, 256, 64), size) == 0
    assert h.append(tokens, (size, 128, 64), (4 * size, 128, 64), (3 * size, 256, 64), size) == -4
    assert h.append(tokens, (4 * size, 128, 64), (size, 128, 64), (3 * size, 256, 64), size) == -4
    # strided: the last row of a fused projection's keys
    wide = 4 * ROW
    rows = ((ROW, wide // 2, 64), (ROW + ROW // 2, wide // 2, 64), (0, wide // 2, 64))
    end = (tokens - 1) * wide + 2 * ROW
    assert h.append(tokens, *rows, end) == 0
    assert h.append(tokens, *rows, end - 16) == -4
    assert lib.fake_appends() == before + 3


@pytest.mark.parametrize("stream", [None, 4096])
@pytest.mark.parametrize("bits,status", [(1, -1), (2, -5), (3, -5), (0, 0)])
def test_sync_reports_a_handle_of_another_device(package, lib, stream, bits, status):
    """The default stream is that of the current device: what the handle's device has under way there is waited for all the same,
    and the caller's device stays current."""
    h = Handle(package, lib, device=1)
    rows = (4 * ROW, 128, 64), (6 * ROW, 128, 64), (0, 256, 64)
    assert h.append(1, *rows, 8 * ROW, stream) == 0
    lib.fake_leave(1, stream, ctypes.addressof(h.status.contents), bits)
    lib.fake_device(0)
    assert h.append(1, *rows, 8 * ROW, stream) == -1                          # launches want the handle's device
    assert lib.aima_moe_kv_sync(h.handle) == status
    assert lib.fake_current() == 0 and h.status[0] == 0
    assert lib.aima_moe_kv_sync(h.handle) == 0
    lib.fake_device(1)
    assert lib.aima_moe_kv_sync(h.handle) == 0 and lib.fake_current() == 1


@pytest.mark.parametrize("bits,left", [(1, 7), (2, 0), (3, 0)])
def test_sync_puts_the_joins_counters_back_only_after_a_wait_that_ran_out(package, lib, bits, left):
    """A launch under way on another stream counts on them; a length out of range does not touch them."""
    h = Handle(package, lib)
    h.status[0], h.status[64], h.status[64 + 511] = bits, 7, 7
    assert lib.aima_moe_kv_sync(h.handle) == (-1 if bits == 1 else -5)
    assert (h.status[0], h.status[64], h.status[64 + 511]) == (0, left, left)
