"""The operators together, as experiments.moe_layer runs them; weights beyond 32-bit offsets."""
import numpy as np
import pytest
import torch

from mxq import nn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["MXFP8_E4M3", "MXFP4"])
def test_layer_command(cuda, fmt):
    """The layer in bfloat16 against float32 on the dequantized weights: three roundings to bfloat16 (2^-8 each, at most)
    of rows of norm, on their way through products that keep relative error."""
    from experiments import moe_layer
    found = moe_layer.main(["--tokens", "40", "--width", "96", "--hidden", "80", "--experts", "5", "--shared", "64", "--fmt", fmt])
    assert found["relative"] < 4 * 2.0 ** -8


def test_layer_router_gradient(cuda):
    """Against differences of the layer itself along the router's weight, every expert chosen so that no choice changes on the
    way: in float32, with steps whose quotient is off by the outputs' float32 rounding over the step."""
    from experiments.moe_layer import MoELayer
    g = torch.Generator("cuda").manual_seed(4)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")
    layer = MoELayer.from_weights(normal(4, 32) * 0.3, normal(4, 96, 32) * 0.2, normal(4, 32, 48) * 0.2, top_k=4)
    x, dy = normal(12, 32), normal(12, 32)
    grad = layer.router_gradient(x, dy)
    way = normal(4, 32)
    step = 2.0 ** -8
    start, values = layer.router, []
    for sign in (1, -1):
        layer.router = start + sign * step * way
        values.append(float((layer(x).double() * dy.double()).sum()))
    layer.router = start
    size = float((layer(x).double().abs() * dy.double().abs()).sum())
    want = float((grad.double() * way.double()).sum())
    # rounding: 2^-20 of the sum's size a value (32 and 48 products, in float32); the third derivative's share step^2
    assert abs((values[0] - values[1]) / (2 * step) - want) < size * 2.0 ** -19 / (2 * step) + 40 * step ** 2 * size


def test_offsets_beyond_32_bits(cuda):
    """The last rows of a weight of more than 2^32 bytes: the same as of their own copy."""
    N, K = 66000, 65536 + 128
    codes = torch.randint(0, 120, (1, K), dtype=torch.uint8, device="cuda").expand(N, K).contiguous()
    codes[-8:] = torch.randint(0, 120, (8, K), dtype=torch.uint8, device="cuda")
    scales = torch.full((N, K // 32), 120, dtype=torch.uint8, device="cuda")
    assert codes.numel() > 1 << 32
    for M in (2, 40):
        x = torch.randn(M, K, device="cuda", dtype=torch.bfloat16)
        whole = nn.packed_linear(x, codes, scales, "MXFP8_E4M3", out_dtype=torch.float32)[:, -8:]
        alone = nn.packed_linear(x, codes[-8:].clone(), scales[-8:], "MXFP8_E4M3", out_dtype=torch.float32)
        size = x.float().abs().sum(1, keepdim=True) * 448 * 2.0 ** -7
        assert ((whole - alone).abs() <= 2 * K * 2.0 ** -24 * size).all()
        assert not torch.equal(whole[:, 0], whole[:, 1])


def test_experts_offsets_beyond_32_bits(cuda):
    E, N, K = 40, 2048, 54272
    codes = torch.zeros(E, N, K, dtype=torch.uint8, device="cuda")
    codes[-1] = torch.randint(0, 120, (N, K), dtype=torch.uint8, device="cuda")
    scales = torch.full((E, N, K // 32), 120, dtype=torch.uint8, device="cuda")
    assert codes.numel() > 1 << 32
    for T in (3, 40 * 20):
        plan = nn.dispatch(torch.full((T, 1), E - 1, device="cuda"), E)
        x = torch.randn(T, K, device="cuda", dtype=torch.bfloat16)
        y = nn.expert_linear(x, codes, scales, "MXFP8_E4M3", plan, out_dtype=torch.float32)
        alone = nn.packed_linear(x, codes[-1].clone(), scales[-1].clone(), "MXFP8_E4M3", out_dtype=torch.float32)
        size = x.float().abs().sum(1, keepdim=True) * 448 * 2.0 ** -7
        assert ((y - alone).abs() <= 2 * K * 2.0 ** -24 * size).all()
