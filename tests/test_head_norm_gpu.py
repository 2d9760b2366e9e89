"""The norm of each head with its gate against the 64-bit oracle."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import linear_oracle  # noqa: E402

HALF_STEP = 2.0 ** -8


def check(got, want):
    """The sum of squares, a root, four products and a logistic function in FP32: below 2^-18; then one rounding to BF16."""
    assert bool(((got.double() - want).abs() <= want.abs() * (HALF_STEP + 2.0 ** -18) + 2.0 ** -133).all())


@pytest.mark.parametrize("activation", ["none", "silu", "sigmoid"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 16), (3, 5), (257, 2), (64, 31), (1000, 32), (9001, 32)])
def test_head_norm(package, tokens, heads, dim, activation):
    g = torch.Generator(device="cuda").manual_seed(tokens + heads + dim)
    row = torch.randn(tokens, heads, 2 * dim, generator=g, device="cuda").bfloat16()
    x, gate = row[..., :dim], row[..., dim:] if activation != "none" else None
    weight = (torch.randn(dim, generator=g, device="cuda") * 0.3).bfloat16()
    for offset, w in ((0.0, weight), (1.0, weight)) + (((0.0, None),) if gate is not None else ()):
        check(package.head_norm(x, w, offset=offset, gate=gate, activation=activation), linear_oracle.head_norm(x, w, offset, gate, activation))
    flat, flat_gate = x.contiguous(), None if gate is None else gate.contiguous()
    want = linear_oracle.head_norm(flat, weight, 1.0, flat_gate, activation)
    out = torch.empty_like(flat)
    assert package.head_norm(flat, weight, offset=1.0, gate=flat_gate, activation=activation, out=out) is out
    check(out, want)
    package.head_norm(flat, weight, offset=1.0, gate=flat_gate, activation=activation, out=flat)          # in place
    assert torch.equal(flat, out)


def test_rows_of_any_order(package):
    """Heads before tokens, broadcast gates, a single row with strides that mean nothing."""
    x = torch.randn(6, 50, 128, device="cuda").bfloat16().transpose(0, 1)
    gate = torch.randn(50, 1, 128, device="cuda").bfloat16().expand(-1, 6, -1)
    weight = torch.randn(128, device="cuda").bfloat16()
    check(package.head_norm(x, weight, gate=gate, activation="silu"), linear_oracle.head_norm(x, weight, 0.0, gate, "silu"))
    one = torch.randn(1, 3, 64, device="cuda").bfloat16().as_strided((1, 3, 64), (7, 64, 1))
    check(package.head_norm(one, weight[:64]), linear_oracle.head_norm(one, weight[:64]))


def test_extreme_numbers(package):
    x = torch.randn(8, 4, 128, device="cuda").bfloat16()
    gate = torch.randn(8, 4, 128, device="cuda").bfloat16()
    x[0] = 0.0
    x[1] *= 1.0e15
    x[2] *= 1.0e-15
    x[3, 1, 7] = float("nan")
    x[4, 2, 9] = float("inf")
    gate[5], gate[6] = 80.0, -80.0
    gate[7, :, :3] = torch.tensor([float("inf"), 0.0, float("nan")], device="cuda").bfloat16()
    weight = torch.randn(128, device="cuda").bfloat16()
    for activation in ("silu", "sigmoid"):
        want = linear_oracle.head_norm(x, weight, 0.0, gate, activation)
        got = package.head_norm(x, weight, gate=gate, activation=activation).double()
        fine = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool((got[0][torch.isfinite(gate[0])] == 0.0).all())
        assert bool(((got - want).abs() <= want.abs() * (HALF_STEP + 2.0 ** -18) + 2.0 ** -126)[fine].all())


def test_captured_and_on_another_stream(package):
    x = torch.randn(33, 16, 256, device="cuda").bfloat16()
    weight = torch.randn(256, device="cuda").bfloat16()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        package.head_norm(x, weight)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = package.head_norm(x, weight)
    torch.cuda.current_stream().wait_stream(stream)
    x.copy_(torch.randn(33, 16, 256, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    check(out, linear_oracle.head_norm(x, weight))


def test_refusals(package):
    x = torch.randn(4, 2, 128, device="cuda").bfloat16()
    weight = torch.ones(128, device="cuda").bfloat16()
    for wrong in (dict(x=x.float()), dict(x=x[0]), dict(x=x.cpu()), dict(weight=weight[:64]), dict(weight=weight.float()), dict(activation="tanh"),
                  dict(gate=x[:3], activation="silu"), dict(out=torch.empty(4, 2, 256, device="cuda", dtype=torch.bfloat16)[..., ::2]),
                  dict(x=torch.randn(4, 2, 256, device="cuda").bfloat16()[..., ::2])):
        with pytest.raises(ValueError):
            package.head_norm(**{"x": x, "weight": weight, **wrong})
    for wrong, status in ((dict(activation="silu"), -1), (dict(gate=x), -1), (dict(weight=None), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1),
                          (dict(offset=float("inf")), -1), (dict(gate=x, activation="silu", out=x.clone(), x=x), None)):
        if status is None:
            package.head_norm(**{"weight": weight, **wrong})
            continue
        with pytest.raises(package.AimaMoeError) as error:
            package.head_norm(**{"x": x, "weight": weight, **wrong})
        assert error.value.status == status
    with pytest.raises(package.AimaMoeError) as error:
        package.head_norm(torch.randn(4, 2, 32, device="cuda").bfloat16(), weight[:32].clone())
    assert error.value.status == -2
    flat = torch.randn(16 * 256 + 64, device="cuda").bfloat16()
    with pytest.raises(package.AimaMoeError) as error:                # shifted by a part of a row
        package.head_norm(flat[:16 * 256].view(16, 2, 128), weight, out=flat[64:].view(16, 2, 128))
    assert error.value.status == -4
    gate = torch.randn(4, 2, 128, device="cuda").bfloat16()
    with pytest.raises(package.AimaMoeError) as error:
        package.head_norm(x, weight, gate=gate, activation="silu", out=gate)
    assert error.value.status == -4
    with pytest.raises(package.AimaMoeError) as error:                # rows that are not 16-byte aligned
        package.head_norm(torch.randn(4, 2, 136, device="cuda").bfloat16()[..., 4:132], weight)
    assert error.value.status == -1
