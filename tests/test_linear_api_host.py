"""The C ABI of the linear-attention layers and of the head norm (csrc/linear_api.cu) over a CUDA runtime made for it,
tests/linear_api_fake.cpp: what the entries check and choose by themselves, without a device."""
from __future__ import annotations

import ctypes
import shutil
import subprocess

import pytest

from conftest import PACKAGE_DIR, ROOT

BASE = 1 << 40                # of addresses that nothing reads
CHANNELS = (2 * 2 + 4) * 128


@pytest.fixture(scope="module")
def lib(package, tmp_path_factory):
    path = tmp_path_factory.mktemp("linear") / "liblinear_api_fake.so"
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-std=c++17", "-O1", "-shared", "-cudart", "none", "-Xlinker", "-Bsymbolic", "-Xcompiler", "-fPIC", "-gencode", "arch=compute_100a,code=sm_100a",
                    "-I", str(PACKAGE_DIR / "csrc"), "-o", str(path), str(PACKAGE_DIR / "csrc" / "linear_api.cu"), str(ROOT / "tests" / "linear_api_fake.cpp")],
                   check=True)
    lib = ctypes.CDLL(str(path))
    for name, restype, argtypes in package.provider.EXPORTS:
        if name.startswith(("aima_moe_linear_", "aima_moe_head_norm")):
            getattr(lib, name).restype, getattr(lib, name).argtypes = restype, argtypes
    lib.fake_message.restype = ctypes.c_char_p
    return lib


def config(p, **changes):
    c = p.LinearConfig(ctypes.sizeof(p.LinearConfig), 2, 4, 128, 4, 6, 1, 4, 4096, 0.0, None, 0)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


class Handle:
    """A handle of one layer on the fake's device, with 2 key and 4 value heads."""

    def __init__(self, package, lib, device=0, **changes):
        self.p, self.lib = package.provider, lib
        lib.fake_device(device)
        self.config = config(self.p, **changes)
        self.handle, owner = ctypes.c_void_p(), ctypes.c_void_p()
        lib.cudaMalloc(ctypes.byref(owner), ctypes.c_size_t(16))              # what follows is of this device
        lib.cudaFree(owner)
        assert lib.aima_moe_linear_prepare(ctypes.byref(self.config), ctypes.byref(self.handle)) == 0, lib.fake_message()

    def layer(self, **changes):
        p, slots = self.p, self.config.slots
        layer = p.LinearLayer(ctypes.sizeof(p.LinearLayer), 0)
        for name, size in (("conv_weight", CHANNELS * 4 * 2), ("conv_states", CHANNELS * 3 * 2 * slots), ("states", 128 * 128 * 4 * 4 * slots),
                           ("a_log", 16), ("dt_bias", 16), ("norm_weight", 256)):
            setattr(layer, name, BASE)
            setattr(layer, name + "_bytes", size)
        for name, value in changes.items():
            setattr(layer, name, value)
        return layer

    def bind(self, **changes):
        return self.lib.aima_moe_linear_bind_layer(self.handle, 0, ctypes.byref(self.layer(**changes)))

    def batch(self, tokens, sequences=1, most=None, offsets=BASE, **changes):
        p = self.p
        b = p.LinearBatchStruct(ctypes.sizeof(p.LinearBatchStruct), sequences, tokens, most or tokens, BASE, offsets, BASE, None)
        for name, value in changes.items():
            setattr(b, name, value)
        return b

    def call(self, tokens, out=1 << 41, **changes):
        p = self.p
        d = p.LinearDelta(ctypes.sizeof(p.LinearDelta), 0, p.KvRows(BASE, 256, 128), p.KvRows(BASE, 256, 128), p.KvRows(BASE, 512, 128), p.KvRows(),
                          BASE, BASE, 4, 4, out)
        for name, value in changes.items():
            setattr(d, name, value)
        return d

    def delta(self, batch, call, stream=None):
        return self.lib.aima_moe_linear_delta_launch(self.handle, 0, ctypes.byref(batch), ctypes.byref(call), stream)

    def conv(self, batch, x=BASE, stride=CHANNELS, out=1 << 41):
        return self.lib.aima_moe_linear_conv_launch(self.handle, 0, ctypes.byref(batch), x, stride, out, None)


@pytest.mark.parametrize("changes,status", [
    (dict(struct_bytes=8), -1), (dict(head_dim=64), -2), (dict(k_heads=0), -1), (dict(k_heads=3), -1), (dict(v_heads=512, k_heads=128), -1),
    (dict(conv_width=1), -2), (dict(conv_width=5), -2), (dict(slots=0), -1), (dict(slots=(1 << 20) + 1), -1), (dict(layers=0), -1), (dict(layers=65), -1),
    (dict(max_sequences=0), -1), (dict(max_sequences=1025), -1), (dict(max_tokens=0), -1), (dict(max_tokens=(1 << 20) + 1), -1),
    (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(eps=float("inf")), -1), (dict(workspace=BASE + 16, workspace_bytes=1 << 30), -1),
    (dict(workspace=BASE, workspace_bytes=100), -1)])
def test_configurations_that_are_refused(package, lib, changes, status):
    p = package.provider
    lib.fake_device(0)
    handle, size = ctypes.c_void_p(), ctypes.c_uint64()
    assert lib.aima_moe_linear_prepare(ctypes.byref(config(p, **changes)), ctypes.byref(handle)) == status
    assert not handle.value and lib.fake_message()
    if "workspace" not in changes:
        assert lib.aima_moe_linear_query_workspace(ctypes.byref(config(p, **changes)), ctypes.byref(size)) == status
    assert lib.aima_moe_linear_prepare(None, ctypes.byref(handle)) == -1 and lib.aima_moe_linear_query_workspace(ctypes.byref(config(p)), None) == -1


def test_the_workspace_is_what_its_query_says(package, lib):
    p = package.provider
    size = ctypes.c_uint64()
    assert lib.aima_moe_linear_query_workspace(ctypes.byref(config(p)), ctypes.byref(size)) == 0
    assert size.value == 256 + 16 * 4096
    assert lib.aima_moe_linear_query_workspace(ctypes.byref(config(p, max_tokens=28)), ctypes.byref(size)) == 0
    assert size.value == 256                         # never a chunk
    assert lib.aima_moe_linear_query_workspace(ctypes.byref(config(p, max_tokens=29)), ctypes.byref(size)) == 0
    assert size.value > 256


@pytest.mark.parametrize("changes,status", [
    ({}, 0), (dict(struct_bytes=8), -1), (dict(conv_weight_bytes=1), -1), (dict(states_bytes=1), -1), (dict(states=BASE + 8), -1), (dict(a_log=None), -1),
    (dict(conv_states=None), -1), (dict(conv_weight=None, conv_states=None), 0), (dict(states=None, a_log=None, dt_bias=None), 0), (dict(norm_weight=None), 0)])
def test_binding(package, lib, changes, status):
    h = Handle(package, lib)
    assert h.bind(**changes) == status
    assert lib.aima_moe_linear_bind_layer(h.handle, 1, ctypes.byref(h.layer())) == -1
    assert lib.aima_moe_linear_bind_layer(None, 0, ctypes.byref(h.layer())) == -1
    lib.aima_moe_linear_release(h.handle)


def test_what_is_not_bound_is_not_launched(package, lib):
    h = Handle(package, lib)
    before = lib.fake_launches()
    assert h.delta(h.batch(4), h.call(4)) == -3 and h.conv(h.batch(4)) == -3
    assert h.bind(conv_weight=None, conv_states=None, norm_weight=None) == 0
    assert h.conv(h.batch(4)) == -3 and h.delta(h.batch(4), h.call(4, gate=h.p.KvRows(BASE, 512, 128))) == -3
    assert lib.fake_launches() == before
    assert h.delta(h.batch(4), h.call(4)) == 0
    assert h.bind(states=None, a_log=None, dt_bias=None) == 0
    assert h.delta(h.batch(4), h.call(4)) == -3 and h.conv(h.batch(4)) == 0


@pytest.mark.parametrize("changes,status", [
    (dict(struct_bytes=8), -1), (dict(sequences=0), -8), (dict(sequences=5), -8), (dict(tokens=0), -8), (dict(tokens=4097), -8), (dict(max_new_tokens=0), -1),
    (dict(max_new_tokens=9), -1), (dict(slots=None), -1), (dict(row_offsets=None, sequences=3), -1)])
def test_batches_that_are_refused(package, lib, changes, status):
    h = Handle(package, lib)
    assert h.bind() == 0
    before = lib.fake_launches()
    batch = h.batch(8)
    for name, value in changes.items():
        setattr(batch, name, value)
    assert h.delta(batch, h.call(8)) == status and h.conv(batch) == status
    assert lib.fake_launches() == before


@pytest.mark.parametrize("tokens,sequences,most,offsets,launches", [
    (1, 1, 1, True, 10), (28, 1, 28, True, 10), (29, 1, 29, True, 100), (29, 1, 29, False, 100), (56, 2, 29, True, 110), (58, 2, 29, False, 100),
    (56, 2, 28, False, 10), (56, 2, 28, True, 10), (4096, 4, 1024, False, 100)])
def test_few_rows_go_token_by_token_and_many_in_chunks(package, lib, tokens, sequences, most, offsets, launches):
    """With offsets a batch may hold both kinds."""
    h = Handle(package, lib)
    assert h.bind() == 0
    before = lib.fake_launches()
    assert h.delta(h.batch(tokens, sequences, most, BASE if offsets else None), h.call(tokens)) == 0
    assert lib.fake_launches() == before + launches


def test_calls_that_are_refused(package, lib):
    h = Handle(package, lib)
    rows = h.p.KvRows
    assert h.bind() == 0
    before = lib.fake_launches()
    b = h.batch(8)
    for changes, status in ((dict(struct_bytes=8), -1), (dict(q=rows()), -1), (dict(k=rows(BASE + 8, 256, 128)), -1), (dict(v=rows(BASE, 516, 128)), -1),
                            (dict(v=rows(BASE, 512, 132)), -1), (dict(v=rows(BASE, 1 << 36, 128)), -1), (dict(a=None), -1), (dict(b=BASE + 1), -1),
                            (dict(a_row_stride=1 << 36), -1), (dict(out=BASE + (1 << 40) + 8), -1)):
        assert h.delta(b, h.call(8, **changes)) == status, changes
    assert lib.aima_moe_linear_delta_launch(h.handle, 0, ctypes.byref(b), None, None) == -1
    assert lib.aima_moe_linear_delta_launch(h.handle, 1, ctypes.byref(b), ctypes.byref(h.call(8)), None) == -1
    for x, stride, out in ((0, CHANNELS, 1 << 41), (BASE + 2, CHANNELS, 1 << 41), (BASE, CHANNELS + 4, 1 << 41), (BASE, CHANNELS, 0), (BASE, CHANNELS, (1 << 41) + 8)):
        assert h.conv(b, x, stride, out) == -1
    lib.fake_device(1)
    assert h.delta(b, h.call(8)) == -1 and h.conv(b) == -1                    # launches want the handle's device
    lib.fake_device(0)
    assert lib.fake_launches() == before
    # one row: its stride means nothing; a broadcast's is zero
    one = h.batch(1)
    assert h.delta(one, h.call(1, v=rows(BASE, 3, 128), a_row_stride=7)) == 0
    assert h.delta(b, h.call(8, k=rows(BASE, 0, 0), gate=rows(BASE, 512, 0))) == 0
    assert h.delta(b, h.call(8, out=None)) == 0


@pytest.mark.parametrize("name,heads", [("q", 2), ("k", 2), ("v", 4), ("gate", 4)])
def test_outputs_may_not_lie_over_any_input(package, lib, name, heads):
    h = Handle(package, lib)
    assert h.bind() == 0
    b, at = h.batch(3), 1 << 42
    row = heads * 128                                       # an input of its own, rows twice as far apart as they need be
    span = (2 * 2 * row + row) * 2
    out = 3 * 4 * 128 * 2
    for start, status in ((at + span, 0), (at + span - 16, -4), (at, -4), (at - out, 0), (at - out + 16, -4), (at + row * 2, -4)):
        assert h.delta(b, h.call(3, out=start, **{name: h.p.KvRows(at, 2 * row, 128)})) == status, start - at
    assert h.delta(b, h.call(3, out=at, a=at + out - 2)) == -4 and h.delta(b, h.call(3, out=at, b=at - 16)) == -4
    size = 3 * CHANNELS * 2
    for start, status in ((at + size, 0), (at + size - 16, -4), (at, -4), (at - size, 0), (at - size + 16, -4)):
        assert h.conv(b, at, CHANNELS, start) == status


@pytest.mark.parametrize("bits,status", [(1, -1), (2, -5), (3, -5), (0, 0)])
def test_sync_reports_once_and_for_a_handle_of_another_device(package, lib, bits, status):
    memory = (ctypes.c_uint8 * (256 + 16 * 4096 + 256))()
    at = (ctypes.addressof(memory) + 255) // 256 * 256
    h = Handle(package, lib, device=1, workspace=at, workspace_bytes=256 + 16 * 4096)
    word = ctypes.cast(at, ctypes.POINTER(ctypes.c_int))
    assert word[0] == 0
    word[0] = bits
    lib.fake_device(0)
    assert lib.aima_moe_linear_sync(h.handle) == status
    assert lib.fake_current() == 0 and word[0] == 0
    assert lib.aima_moe_linear_sync(h.handle) == 0
    assert lib.aima_moe_linear_sync(None) == -1 and lib.aima_moe_linear_release(None) == 0


def test_head_norm_calls(package, lib):
    p = package.provider
    lib.fake_device(0)

    def call(**changes):
        c = p.HeadNorm(ctypes.sizeof(p.HeadNorm), 5, 3, 128, 0, 1.0, 1.0e-6, 0, p.KvRows(BASE, 384, 128), p.KvRows(), BASE + (1 << 30), 1 << 41)
        for name, value in changes.items():
            setattr(c, name, value)
        return lib.aima_moe_head_norm_launch(ctypes.byref(c), None)

    before = lib.fake_launches()
    gate = p.KvRows(BASE, 384, 128)
    size = 5 * 384 * 2
    for changes, status in ((dict(struct_bytes=8), -1), (dict(tokens=0), -1), (dict(tokens=(1 << 24) + 1), -1), (dict(heads=0), -1), (dict(heads=1025), -1),
                            (dict(head_dim=96), -2), (dict(activation=3), -1), (dict(activation=1), -1), (dict(gate=gate), -1), (dict(weight=None), -1),
                            (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(weight_offset=float("inf")), -1), (dict(out=None), -1),
                            (dict(out=(1 << 41) + 8), -1), (dict(weight=BASE + 8), -1), (dict(x=p.KvRows()), -1), (dict(x=p.KvRows(BASE, 388, 128)), -1),
                            (dict(out=BASE + 16), -4), (dict(out=BASE, x=p.KvRows(BASE, 768, 256)), -4), (dict(out=BASE + size - 16), -4),
                            (dict(out=1 << 41, gate=p.KvRows((1 << 41) + 256, 384, 128), activation=1), -4), (dict(weight=(1 << 41) + size - 16), -4)):
        assert call(**changes) == status, changes
    assert lib.aima_moe_head_norm_launch(None, None) == -1
    assert lib.fake_launches() == before
    for changes in ({}, dict(out=BASE), dict(out=BASE + size), dict(weight=None, gate=gate, activation=2), dict(gate=p.KvRows(BASE, 0, 0), activation=1),
                    dict(tokens=1, x=p.KvRows(BASE, 3, 128)), dict(heads=1, x=p.KvRows(BASE, 128, 1), out=BASE)):
        assert call(**changes) == 0, changes
