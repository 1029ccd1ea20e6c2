"""Which values the products with packed weights take, on the kernel of few rows and on every tile: every code under every
scale byte, weights past float32's range, float16's products bit for bit, activations
below bfloat16's smallest step."""
import numpy as np
import pytest
import torch

from mxq import nn
from oracle import moe as om
from oracle.packed import FORMATS

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = torch.finfo(torch.float32).eps / 2
# rows of x that take the kernel of few rows and each tile there is
ROWS = [3, 20, 600, 1001]


def _pairs(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _as_float32(W):
    """Weights of 2^128 and more are infinite, as they are in float32: a code's few bits never lie between its largest value
    and 2^128."""
    return torch.where(W.abs() >= 2.0 ** 128, torch.copysign(torch.full_like(W, np.inf), W), W)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt, pairs", [(f, False) for f in FORMATS] + [("MXFP4", True)])
def test_every_code_and_scale(cuda, fmt, pairs, dtype):
    """One code a row, at every place of a block in turn, the other columns zeros: a power of two times the weight, exactly,
    and a weight below 2^-126 within half a step of bfloat16's subnormals."""
    e, m = FORMATS[fmt]
    kinds, K = 2 ** (1 + e + m), 128
    N = kinds * 256
    n = torch.arange(N)
    code, scale, block = (n // 256).to(torch.uint8), (n % 256).to(torch.uint8), n % 4
    codes, scales = torch.zeros(N, K, dtype=torch.uint8), torch.full((N, 4), 127, dtype=torch.uint8)
    column = block * 32 + n // 4 % 32
    codes[n, column], scales[n, block] = code, scale
    W = torch.from_numpy(om.weight(code[:, None].numpy(), scale[:, None].numpy(), fmt, 1))[:, 0].cuda()
    w = _as_float32(W)
    codes, scales = (_pairs(codes) if pairs else codes).cuda(), scales.cuda()
    for M in ROWS:
        powers = torch.tensor((15.0, 0.0, -14.0) if dtype == "f16" else (100.0, 0.0, -100.0)).exp2().double()
        x = powers[torch.arange(M) % 3][:, None].expand(M, K).to(DTYPES[dtype]).cuda()
        y = nn.packed_linear(x, codes, scales, fmt, out_dtype=torch.float32)
        for i, power in enumerate(powers.tolist()):
            want, got = w * power, y[i].double()
            rows = y[i::3].nan_to_num(0.375, np.inf, -np.inf)         # every row the same, wherever a tile has it
            assert torch.equal(rows, rows[:1].expand_as(rows)), (M, i)
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (M, i)
            large = want.abs() >= 2.0 ** 128                        # the product is, or the weight already
            assert torch.equal(got[large], torch.copysign(torch.full_like(want, np.inf), want)[large]), (M, i)
            small = w.abs() < 2.0 ** -126
            exact = ~small & ~large & (want.abs() >= 2.0 ** -126) & ~torch.isnan(want)
            assert torch.equal(got[exact], want[exact]), (M, i)
            rounded = small & (want.abs() >= 2.0 ** -110)            # sums of them are no subnormals
            assert ((got - want).abs()[rounded] <= 2.0 ** -134 * power).all(), (M, i)
            tiny = want.abs() < 2.0 ** -126
            assert (got.abs()[tiny] <= 2.0 ** -126).all(), (M, i)
            assert int(exact.sum()) > N // 3 and (int(rounded.sum()) > 0 or dtype == "f16" or i > 0), (M, i)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt, pairs", [(f, False) for f in FORMATS] + [("MXFP4", True)])
def test_weights_past_float32(cuda, fmt, pairs, dtype):
    """Finite codes under the largest scales: a weight of 2^128 or more is an infinity for every type of x, whatever bits
    x has, and makes NaN of a zero only."""
    rng = np.random.default_rng(7)
    e, m = FORMATS[fmt]
    N, K = 96, 160
    # the largest code, and the scale byte from which it is 2^128 or more
    top, first = {"MXFP8_E4M3": (0x7E, 247), "MXFP8_E5M2": (0x7B, 240), "MXFP6_E3M2": (0x1F, 251), "MXFP6_E2M3": (0x1F, 253),
                  "MXFP4": (7, 253)}[fmt]
    codes = torch.from_numpy(rng.integers(0, top + 1, (N, K)).astype(np.uint8)) & (top >> 1)      # halved exponents: finite
    scales = torch.from_numpy(rng.integers(first - 4, 255, (N, K // 32)).astype(np.uint8))
    scales[::2] = torch.from_numpy(rng.integers(100, 130, (N // 2, K // 32)).astype(np.uint8))
    for n in range(1, N, 2):                                         # odd rows: the largest code in one block
        codes[n, rng.integers(0, K)] = top
    codes = codes | torch.from_numpy((rng.integers(0, 2, (N, K)) << (e + m)).astype(np.uint8))
    w = _as_float32(torch.from_numpy(om.weight(codes.numpy(), scales.numpy(), fmt, K)))
    past = torch.isinf(w).any(1)
    assert 4 < past[1::2].sum() < 44 and not past[::2].any()
    sent = (_pairs(codes) if pairs else codes).cuda()
    for M in ROWS:
        x = torch.from_numpy(rng.standard_normal((M, K)) * 2.0 ** -12).to(DTYPES[dtype])
        x[0] = (x[0].double() != 0).to(x.dtype) * 2.0 ** -12        # no bits for a lower plane
        x[1, ::3] = 0
        x[2] = torch.from_numpy(np.exp2(rng.integers(-14, -8, K))).to(x.dtype)
        y = nn.packed_linear(x.cuda(), sent, scales.cuda(), fmt, out_dtype=torch.float32).double().cpu()
        want = x.double() @ w.t()
        assert torch.equal(torch.isnan(y), torch.isnan(want)), M
        inf = torch.isinf(want)
        assert torch.equal(y[inf], want[inf]) and inf.any()
        finite = torch.isfinite(want)
        size = x.double().abs() @ torch.where(past[:, None], 0.0, w).abs().t()
        near = finite & (size < 2.0 ** 127)                          # no partial sum leaves float32
        assert ((y - want).abs()[near] <= ((K + 2) * HALF * size)[near]).all(), M
        assert near[:, ::2].all()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_float16_products_are_exact(cuda, fmt):
    """One product an output: 11 bits by 4 fit float32, and so do two sums of an 8-bit part and the rest."""
    rng = np.random.default_rng(3)
    e, m = FORMATS[fmt]
    codes = torch.from_numpy(rng.integers(0, 2 ** (e + m) - (4 if e > 3 else 0), (80, 128)).astype(np.uint8))
    codes |= torch.from_numpy((rng.integers(0, 2, (80, 128)) << (e + m)).astype(np.uint8))
    scales = torch.from_numpy(rng.integers(112, 130, (80, 4)).astype(np.uint8))
    W = torch.from_numpy(om.weight(codes.numpy(), scales.numpy(), fmt, 128))
    lost = 0
    for M in ROWS:
        x = torch.zeros(M, 128, dtype=torch.float16)
        at = torch.from_numpy(rng.integers(0, 128, M))
        x[torch.arange(M), at] = torch.from_numpy(rng.standard_normal(M) * np.exp2(rng.integers(-20, 10, M))).half()
        y = nn.packed_linear(x.cuda(), codes.cuda(), scales.cuda(), fmt, out_dtype=torch.float32).double().cpu()
        assert torch.equal(y, x.double() @ W.t())
        lost += int((x.bfloat16().double() @ W.t() != y).sum())
    assert lost > 1000                                               # one plane alone would not pass


@pytest.mark.parametrize("M", ROWS)
def test_small_float32_activations(cuda, M):
    """The part of a float32 activation below 2^-133, bfloat16's smallest step, is left out; above 2^-110 there is none."""
    rng = np.random.default_rng(11)
    codes = torch.from_numpy((rng.integers(0, 0x7F, (64, 128)) | rng.integers(0, 2, (64, 128)) << 7).astype(np.uint8))
    scales = torch.from_numpy(rng.integers(200, 220, (64, 4)).astype(np.uint8))
    W = torch.from_numpy(om.weight(codes.numpy(), scales.numpy(), "MXFP8_E4M3", 128))
    for low, high, part in ((-149, -109, 2.0 ** -133), (-110, -90, 0.0)):
        x = torch.from_numpy(rng.standard_normal((M, 128)) * np.exp2(rng.integers(low, high, (M, 128)))).float()
        if not part:
            x = torch.where(x.abs() < 2.0 ** -110, 0.0, x)
        y = nn.packed_linear(x.cuda(), codes.cuda(), scales.cuda(), "MXFP8_E4M3").double().cpu()
        size = x.double().abs() @ W.abs().t()
        bound = 130 * HALF * size + part * W.abs().sum(1) + 2.0 ** -126
        assert ((y - x.double() @ W.t()).abs() <= bound).all()
