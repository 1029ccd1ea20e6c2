"""Weights and activations past 32-bit offsets: sums of small whole numbers, which float32 holds exactly in any order, so
that every result has to be equal."""
import pytest
import torch

from mxq import nn

pytestmark = pytest.mark.gpu
# E4M3's codes of 1, 2, 3, -1; a scale byte of 1
ONES = torch.tensor([0x38, 0x40, 0x44, 0xB8], dtype=torch.uint8)
VALUES = torch.tensor([1.0, 2.0, 3.0, -1.0])


@pytest.fixture(autouse=True)
def _memory(cuda):
    yield
    torch.cuda.empty_cache()


def _whole(rows, K, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-2, 3, (rows, K), generator=gen, device="cuda").to(dtype)


def _codes(rows, K, seed=0):
    """Codes and their values."""
    gen = torch.Generator("cuda").manual_seed(seed)
    kind = torch.randint(0, 4, (rows, K), generator=gen, device="cuda", dtype=torch.uint8)
    codes, values = torch.zeros_like(kind), torch.zeros(rows, K, device="cuda")
    for i in range(4):
        codes[kind == i], values[kind == i] = int(ONES[i]), float(VALUES[i])
    return codes, values


def test_last_rows_of_a_weight_past_2_32_bytes(cuda):
    N, K, last = 66000, 65536 + 128, 300
    codes = torch.full((N, K), 0x40, dtype=torch.uint8, device="cuda")            # 2 in every place
    codes[-last:], values = _codes(last, K)
    scales = torch.full((N, K // 32), 127, dtype=torch.uint8, device="cuda")
    assert (N - last) * K > 1 << 32
    for M in (2, 40, 700, 1100):                                                  # few rows, and every tile
        x = _whole(M, K, seed=M)
        y = nn.packed_linear(x, codes, scales, "MXFP8_E4M3", out_dtype=torch.float32)
        want, other = x.float() @ values.t(), 2 * x.float().sum(1, keepdim=True)
        assert (want != other).float().mean() > 0.9 and (want != 0).float().mean() > 0.9 and \
            (want[:, 1:] != want[:, :-1]).float().mean() > 0.9                    # another row, or zeros, would show
        assert torch.equal(y[:, -last:], want) and torch.equal(y[:, :-last], other.expand(M, N - last))
    codes[-2 * last:-last] = codes[-last:]
    gated = nn.packed_linear(x, codes, scales, "MXFP8_E4M3", activation="relu", gated=True, out_dtype=torch.float32)
    assert torch.equal(gated[:, -last:], other.clamp_min(0) * want)


def test_last_expert_past_2_32_bytes(cuda):
    E, N, K = 40, 2048, 54272
    codes = torch.full((E, N, K), 0x40, dtype=torch.uint8, device="cuda")
    codes[-1], values = _codes(N, K)
    scales = torch.full((E, N, K // 32), 127, dtype=torch.uint8, device="cuda")
    assert (E - 1) * N * K > 1 << 32
    for T in (3, 800, 24000):                                                     # few rows an expert, 20, 600
        x = _whole(T, K, seed=T)
        plan = nn.dispatch(torch.full((T, 1), E - 1, device="cuda"), E)
        y = nn.expert_linear(x, codes, scales, "MXFP8_E4M3", plan, out_dtype=torch.float32)
        rows = torch.arange(0, T, max(1, T // 64), device="cuda")
        want, other = x[rows].float() @ values.t(), 2 * x[rows].float().sum(1, keepdim=True)
        assert (want != other).float().mean() > 0.9 and (want != 0).float().mean() > 0.9 and \
            (want[:, 1:] != want[:, :-1]).float().mean() > 0.9
        assert torch.equal(y[rows], want)


def test_x_past_2_32_bytes(cuda):
    """Rows of x that lie past 2^32 bytes, and experts' rows found there by their slots."""
    T, K, N = 40000, 54272, 130
    assert (T - 300) * K * 2 > 1 << 32
    codes, values = _codes(N, K)
    scales = torch.full((N, K // 32), 127, dtype=torch.uint8, device="cuda")
    x = torch.ones(T, K, dtype=torch.bfloat16, device="cuda")
    x[-300:] = _whole(300, K)
    want = x[-300:].float() @ values.t()
    assert (want != values.sum(1)).float().mean() > 0.9
    y = nn.packed_linear(x, codes, scales, "MXFP8_E4M3", out_dtype=torch.float32)
    assert torch.equal(y[-300:], want) and torch.equal(y[:-300], values.sum(1).expand(T - 300, N))
    picks = torch.full((T, 1), -1, device="cuda")
    picks[-300:] = 1
    for few in (5, 300):
        picks[:-few] = -1
        found = nn.expert_linear(x, codes.expand(2, N, K), scales.expand(2, N, K // 32), "MXFP8_E4M3", nn.dispatch(picks, 2),
                                 out_dtype=torch.float32)
        assert torch.equal(found[:few], want[-few:]) and (found[few:] == 0).all()
        picks[-300:] = 1
