"""The full-attention cache and the verification without a device: structure sizes, configurations that are refused, and the
oracle's own statements checked against independent ones."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import kv_oracle


def _config(package, **changes):
    c = dict(q_heads=16, kv_heads=2, head_dim=256, rotary_dim=64, page_tokens=64, pages=8, layers=1, max_sequences=4,
             softmax_scale=0.0, workspace=None, workspace_bytes=0)
    c.update(changes)
    return package.provider.KvConfig(ctypes.sizeof(package.provider.KvConfig), *c.values())


def test_struct_sizes_match_the_header(package):
    p = package.provider
    assert ctypes.sizeof(p.KvConfig) == 10 * 4 + 16
    assert ctypes.sizeof(p.KvLayer) == 8 + 4 * 16
    assert ctypes.sizeof(p.KvBatchStruct) == 6 * 4 + 3 * 8
    assert ctypes.sizeof(p.KvRows) == 3 * 8
    assert ctypes.sizeof(p.VerifyDrafts) == 4 * 4 + 2 * 3 * 8 + 7 * 8


@pytest.mark.parametrize("change,status", [
    (dict(head_dim=96), -2), (dict(page_tokens=48), -2), (dict(page_tokens=256), -2), (dict(kv_heads=3), -1), (dict(kv_heads=0), -1),
    (dict(q_heads=0), -1), (dict(q_heads=258), -1), (dict(rotary_dim=40), -1), (dict(rotary_dim=272), -1), (dict(pages=0), -1),
    (dict(pages=1 << 24), -1), (dict(layers=0), -1), (dict(layers=65), -1), (dict(max_sequences=0), -1), (dict(max_sequences=1025), -1),
    (dict(softmax_scale=-1.0), -1), (dict(softmax_scale=math.inf), -1), (dict(softmax_scale=math.nan), -1)])
def test_configurations_that_are_refused(package, built_library, change, status):
    lib = package.load_library()
    size, handle = ctypes.c_uint64(), ctypes.c_void_p(1)
    config = _config(package, **change)
    assert lib.aima_moe_kv_query_workspace(ctypes.byref(config), ctypes.byref(size)) == status
    assert lib.aima_moe_kv_prepare(ctypes.byref(config), ctypes.byref(handle)) == status
    assert not handle.value and b"kv" in lib.aima_moe_last_error_string()


def test_workspace_depends_on_the_head_size_alone(package, built_library):
    lib = package.load_library()

    def need(**changes):
        size = ctypes.c_uint64()
        assert lib.aima_moe_kv_query_workspace(ctypes.byref(_config(package, **changes)), ctypes.byref(size)) == 0
        return size.value

    assert need() == need(pages=1 << 20, layers=64, max_sequences=1024, page_tokens=16) == need(q_heads=4, kv_heads=4)
    assert need(head_dim=64) < need(head_dim=128) < need()
    assert need() % 16 == 0


def test_arguments_are_checked_before_a_device_is_needed(package, built_library):
    lib, p = package.load_library(), package.provider
    wrong = _config(package)
    wrong.struct_bytes = 4
    size, handle = ctypes.c_uint64(), ctypes.c_void_p()
    assert lib.aima_moe_kv_query_workspace(ctypes.byref(wrong), ctypes.byref(size)) == -1
    assert b"size mismatch" in lib.aima_moe_last_error_string()
    assert lib.aima_moe_kv_query_workspace(None, ctypes.byref(size)) == -1
    assert lib.aima_moe_kv_query_workspace(ctypes.byref(_config(package)), None) == -1
    assert lib.aima_moe_kv_prepare(ctypes.byref(_config(package)), None) == -1
    rows, batch, layer = p.KvRows(), p.KvBatchStruct(), p.KvLayer()
    assert lib.aima_moe_kv_bind_layer(None, 0, ctypes.byref(layer)) == -1
    assert lib.aima_moe_kv_set_rotation(None, None, 1) == -1
    assert lib.aima_moe_kv_append_launch(None, 0, ctypes.byref(batch), rows, rows, None, None, None) == -1
    assert lib.aima_moe_kv_attention_launch(None, 0, ctypes.byref(batch), rows, None, None) == -1
    assert lib.aima_moe_kv_sync(None) == -1
    assert lib.aima_moe_kv_release(None) == 0
    if not torch.cuda.is_available():
        assert lib.aima_moe_kv_prepare(ctypes.byref(_config(package)), ctypes.byref(handle)) == -7 and not handle.value
        with pytest.raises(RuntimeError):
            package.KvCache(pages=4)


@pytest.mark.parametrize("change", [dict(struct_bytes=8), dict(sequences=0), dict(sequences=65536), dict(max_drafts=65), dict(vocabulary=0),
                                    dict(vocabulary=(1 << 22) + 1), dict(target=None), dict(target=18), dict(draft=18), dict(uniforms=None),
                                    dict(accepted=None), dict(tokens=None), dict(draft_tokens=None), dict(cache_lengths=64), dict(new_lengths=64)])
def test_verification_arguments_that_are_refused(package, built_library, change):
    lib, p = package.load_library(), package.provider
    call = p.VerifyDrafts(ctypes.sizeof(p.VerifyDrafts), 1, 2, 8, 64, 24, 8, None, 0, 0, 64, None, 64, None, 64, 64, None)
    for name, value in change.items():
        setattr(call, name, value)
    assert lib.aima_moe_verify_drafts_launch(call, None) == -1
    assert b"mismatch" in lib.aima_moe_last_error_string() or b"verify" in lib.aima_moe_last_error_string()
    assert lib.aima_moe_verify_drafts_launch(None, None) == -1


def test_the_oracles_rounding_is_that_of_the_type():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    every = every[torch.isfinite(every)]
    g = torch.Generator().manual_seed(1)
    x = torch.cat([every, (every[:, None] + every[None, :]).flatten() / 2, torch.randn(5000, generator=g) * 2.0 ** torch.randint(-12, 9, (5000,), generator=g)])
    x = x[x.abs() <= 448]
    assert torch.equal(kv_oracle.e4m3(x), x.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("amax", [2.0 ** -120, 1e-20, 0.3, 447.9, 448.0, 448.1, 1e5, 3e38])
def test_the_oracles_scale_is_the_least(amax):
    e = kv_oracle.exponent_for(amax)
    assert amax <= 448.0 * 2.0 ** e and (e == kv_oracle.MIN_EXPONENT or amax > 448.0 * 2.0 ** (e - 1))


def test_the_oracles_rotation_keeps_lengths_and_turns_by_the_angle():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 64, generator=g, dtype=torch.float64)
    angle = torch.rand(16, generator=g, dtype=torch.float64) * 6.0
    y = kv_oracle.rotate(x, torch.cat([angle.cos(), angle.sin()]))
    turned = torch.complex(x[:, :16], x[:, 16:32]) * torch.polar(torch.ones(16, dtype=torch.float64), angle)
    assert torch.allclose(torch.complex(y[:, :16], y[:, 16:32]), turned, rtol=0, atol=1e-14) and torch.equal(y[:, 32:], x[:, 32:])


def test_the_oracles_attention_is_that_of_dense_tensors():
    g = torch.Generator().manual_seed(3)
    page, heads, dim, length, rows = 16, 2, 64, 45, 7
    keys, values = (torch.randn(6, heads, page, dim, generator=g).to(torch.float8_e4m3fn).float() for _ in range(2))
    scales = [torch.rand(6, heads, generator=g) + 0.5 for _ in range(2)]
    table = torch.tensor([[4, 1, 3]])
    q = torch.randn(rows, 4, dim, generator=g)
    out, _ = kv_oracle.attention(keys, values, *scales, table, [0, rows], [length], q, 0.125, page)
    k, v = ((x.double() * s.double()[..., None, None])[table[0]].transpose(0, 1).flatten(1, 2)[:, :length].repeat_interleave(2, 0)
            for x, s in zip((keys, values), scales))
    mask = torch.ones(rows, length, dtype=torch.bool).tril(length - rows)
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k, v, attn_mask=mask, scale=0.125)
    assert torch.allclose(out, want.transpose(0, 1), rtol=0, atol=1e-12)


def test_the_oracles_verification_leaves_the_targets_distribution():
    """Over a grid of uniform numbers a draft drawn from q and verified against p leaves tokens distributed as p."""
    p, q = torch.tensor([0.5, 0.25, 0.125, 0.125]), torch.tensor([0.125, 0.5, 0.375, 0.0])
    grid, share = 64, torch.zeros(4, dtype=torch.float64)
    for x in range(4):
        uniforms = torch.cartesian_prod((torch.arange(grid) + 0.5) / grid, (torch.arange(grid) + 0.5) / grid).float()
        n = uniforms.shape[0]
        target = p.expand(n, 2, 4)
        accepted, tokens = kv_oracle.verify(target, torch.full((n, 1), x, dtype=torch.int32), uniforms, q.expand(n, 1, 4))
        first = torch.tensor([t[0] for t in tokens])
        share += torch.bincount(first, minlength=4).double() / n * float(q[x])
    assert (share - p.double()).abs().max() <= 2.0 / grid
