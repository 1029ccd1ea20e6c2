"""Products with packed weights against 64 bits, within the bound that one float32 sum and one rounding allow
(oracle.moe.linear): formats, types, epilogues, ragged sizes, strides, special codes and scales, the experts' rows."""
import numpy as np
import pytest
import torch

from mxq import nn, packed
from oracle import moe as om

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOP = {"MXFP8_E4M3": 0x7F, "MXFP8_E5M2": 0x7C, "MXFP6_E3M2": 0x20, "MXFP6_E2M3": 0x20, "MXFP4": 0x8}
SIGN = {"MXFP8_E4M3": 0x80, "MXFP8_E5M2": 0x80, "MXFP6_E3M2": 0x20, "MXFP6_E2M3": 0x20, "MXFP4": 0x8}


def _weight(rng, shape, fmt, scales=(112, 130)):
    """Finite codes of all kinds, scales over a range."""
    codes = rng.integers(0, TOP[fmt], shape) | SIGN[fmt] * rng.integers(0, 2, shape)
    return (torch.from_numpy(codes.astype(np.uint8)),
            torch.from_numpy(rng.integers(*scales, (*shape[:-1], -(-shape[-1] // 32))).astype(np.uint8)))


def _pairs(codes):
    codes = torch.nn.functional.pad(codes, (0, codes.shape[-1] % 2))
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _matrix(codes, scales, fmt, K):
    return torch.from_numpy(om.weight(codes.numpy(), scales.numpy(), fmt, K)).cuda()


def _check(got, want, bound, what=""):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - bound
    assert not torch.isnan(off).any(), what
    past = want.abs() + bound > torch.finfo(got.dtype).max                  # may round to infinity
    off = torch.where(past & (got == torch.copysign(torch.full_like(want, np.inf), want)), 0.0, off)
    assert not (off > 0).any(), (what, float(off.max()), float((off / bound).max()))


def _run(rng, M, N, K, fmt, dtype=torch.bfloat16, bias=False, activation=None, gated=False, residual=False, pairs=False, **more):
    rows = 2 * N if gated else N
    codes, scales = _weight(rng, (rows, K), fmt)
    x = torch.from_numpy(rng.standard_normal((M, K))).to(dtype).cuda()
    b = torch.from_numpy(rng.standard_normal(rows)).to(dtype).cuda() if bias else None
    r = torch.from_numpy(rng.standard_normal((M, N))).to(dtype).cuda() if residual else None
    y = nn.packed_linear(x, (_pairs(codes) if pairs else codes).cuda(), scales.cuda(), fmt, bias=b, activation=activation,
                         gated=gated, residual=r, **more)
    assert y.dtype == more.get("out_dtype", dtype)
    want, bound = om.linear(x, _matrix(codes, scales, fmt, K), b, activation, gated, r, y.dtype)
    _check(y, want, bound, (M, N, K, fmt, dtype, activation, gated))


@pytest.mark.parametrize("fmt", list(TOP))
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M", [1, 17, 70, 300])
def test_formats_and_types(cuda, M, dtype, fmt):
    rng = np.random.default_rng(M)
    _run(rng, M, 96, 256, fmt, DTYPES[dtype])
    if fmt == "MXFP4":
        _run(rng, M, 96, 256, fmt, DTYPES[dtype], pairs=True)


@pytest.mark.parametrize("K", [1, 2, 31, 32, 33, 63, 64, 95, 127, 128, 129, 160, 255, 257, 511, 1000, 2057])
@pytest.mark.parametrize("M, N", [(1, 5), (19, 130), (129, 67)])
def test_contractions(cuda, M, N, K):
    rng = np.random.default_rng(K)
    for fmt, dtype, pairs in (("MXFP8_E4M3", torch.bfloat16, False), ("MXFP8_E5M2", torch.float16, False), ("MXFP4", torch.bfloat16, True),
                              ("MXFP6_E2M3", torch.float32, False)):
        _run(rng, M, N, K, fmt, dtype, bias=True, residual=True, pairs=pairs)


@pytest.mark.parametrize("M, N", [(1, 1), (2, 16), (15, 17), (16, 64), (31, 63), (32, 65), (33, 1), (48, 200), (64, 128), (65, 257),
                                  (127, 255), (128, 256), (256, 256), (257, 129), (500, 40), (1, 5000), (1030, 520)])
def test_outputs(cuda, M, N):
    rng = np.random.default_rng(M + N)
    _run(rng, M, N, 192, "MXFP8_E4M3", bias=True)
    _run(rng, M, N, 256, "MXFP8_E4M3", activation="silu", gated=True, residual=True)
    _run(rng, M, N, 128, "MXFP6_E3M2", torch.float16)


@pytest.mark.parametrize("M, N, K", [(2049, 6180, 96), (4096, 4096, 64), (1100, 2050, 128), (130, 70, 4128), (200, 700, 1090)])
def test_many_outputs_and_long_contractions(cuda, M, N, K):
    """The large tiles, whole and cut off, and contractions shared among workgroups."""
    rng = np.random.default_rng(M)
    _run(rng, M, N, K, "MXFP8_E4M3", bias=True, activation="gelu", residual=True)
    _run(rng, M, N, K, "MXFP8_E5M2", torch.float16, bias=True, residual=True)
    _run(rng, M, N // 2, K, "MXFP4", bias=True, activation="silu", gated=True, residual=True, pairs=True)
    _run(rng, M, N // 2, K + 3, "MXFP6_E2M3", torch.float32, bias=True, gated=True)


def test_experts_of_many_rows(cuda):
    rng = np.random.default_rng(21)
    _experts(rng, 1500, 2, 4, 1030, 128, "MXFP8_E4M3", bias=True, activation="silu", gated=True)
    _experts(rng, 1500, 2, 4, 2100, 70, "MXFP4", torch.float16, pairs=True, sorted_rows=True)
    _experts(rng, 900, 4, 30, 516, 192, "MXFP8_E5M2", sorted_rows=True)


def test_largest_scales_of_narrow_codes(cuda):
    """Scale bytes up to 254 of formats that are put into wider fields first."""
    for fmt, K in (("MXFP6_E3M2", 64), ("MXFP6_E2M3", 64), ("MXFP4", 64)):
        codes = torch.full((6, K), {"MXFP6_E3M2": 1, "MXFP6_E2M3": 1, "MXFP4": 1}[fmt], dtype=torch.uint8)
        scales = torch.tensor([[0, 1], [127, 247], [248, 249], [250, 251], [252, 253], [254, 255]], dtype=torch.uint8)
        for M in (3, 100):
            x = torch.zeros(M, K)
            x[:, 0], x[:, 40] = 2.0 ** -3, 2.0 ** -4
            y = nn.packed_linear(x.cuda(), codes.cuda(), scales.cuda(), fmt).double().cpu()
            want = x.double() @ _matrix(codes, scales, fmt, K).cpu().t()
            assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.isnan(y[:, 5]).all()
            assert torch.equal(y[:, 1:5], want[:, 1:5]), fmt
            assert ((y[:, 0] - want[:, 0]).abs() <= 2.0 ** -133).all()          # a weight below 2^-126: bfloat16's subnormals


@pytest.mark.parametrize("activation", [None, "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [3, 40, 290])
def test_epilogues(cuda, M, gated, activation):
    rng = np.random.default_rng(M)
    for bias in (False, True):
        for residual in (False, True):
            _run(rng, M, 72, 96, "MXFP8_E4M3", torch.float32, bias, activation, gated, residual)
    _run(rng, M, 72, 96, "MXFP8_E5M2", torch.bfloat16, True, activation, gated, True, out_dtype=torch.float32)
    _run(rng, M, 72, 96, "MXFP8_E5M2", torch.float32, True, activation, gated, True, out_dtype=torch.float16)


@pytest.mark.parametrize("M", [1, 50, 200])
def test_strides_and_leading_axes(cuda, M):
    """Rows apart from each other, addresses off every alignment, transposed and higher-dimensional inputs: the same bits."""
    rng = np.random.default_rng(M)
    N, K = 80, 320
    codes, scales = (t.cuda() for t in _weight(rng, (N, K), "MXFP8_E4M3"))
    x = torch.from_numpy(rng.standard_normal((M, K))).to(torch.bfloat16).cuda()
    r = torch.from_numpy(rng.standard_normal((M, N))).to(torch.bfloat16).cuda()
    want = nn.packed_linear(x, codes, scales, "MXFP8_E4M3", residual=r)

    def apart(t, by):
        wide = torch.full((t.shape[0], t.shape[1] + 9), 0x7F if t.dtype == torch.uint8 else float("nan"), dtype=t.dtype, device="cuda")
        wide[:, by:by + t.shape[1]] = t
        return wide[:, by:by + t.shape[1]]

    for by in (1, 3, 8):
        assert torch.equal(nn.packed_linear(apart(x, by), apart(codes, by), apart(scales, by), "MXFP8_E4M3", residual=apart(r, by)), want)
    t = nn.packed_linear(x.t().contiguous().t(), codes.t().contiguous().t(), scales, "MXFP8_E4M3", residual=r.t().contiguous().t())
    assert torch.equal(t, want)
    lead = nn.packed_linear(x.reshape(M, 1, 1, K), codes, scales, "MXFP8_E4M3", residual=r.reshape(M, 1, 1, N))
    assert lead.shape == (M, 1, 1, N) and torch.equal(lead.reshape(M, N), want)
    cpu = nn.packed_linear(x.cpu(), codes.cpu(), scales.cpu(), "MXFP8_E4M3", residual=r.cpu())
    assert cpu.device.type == "cpu" and torch.equal(cpu, want.cpu())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = nn.packed_linear(x, codes, scales, "MXFP8_E4M3", residual=r)
    side.synchronize()
    assert torch.equal(there, want)


@pytest.mark.parametrize("M", [1, 40, 200])
def test_empty_sizes(cuda, M):
    codes, scales = torch.zeros(8, 64, dtype=torch.uint8, device="cuda"), torch.zeros(8, 2, dtype=torch.uint8, device="cuda")
    assert nn.packed_linear(torch.zeros(0, 64, device="cuda"), codes, scales, "MXFP8_E4M3").shape == (0, 8)
    assert nn.packed_linear(torch.zeros(M, 64, device="cuda"), codes[:0], scales[:0], "MXFP8_E4M3").shape == (M, 0)
    b, r = torch.randn(8, device="cuda"), torch.randn(M, 8, device="cuda")
    y = nn.packed_linear(torch.zeros(M, 0, device="cuda"), codes[:, :0], scales[:, :0], "MXFP8_E4M3", bias=b, residual=r)
    assert torch.equal(y, b + r)


@pytest.mark.parametrize("M", [2, 40, 200])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_special_values(cuda, M, dtype):
    """A NaN or an infinity reaches the outputs that use it and no other; NaN and Inf codes and the NaN scale likewise."""
    rng = np.random.default_rng(M)
    N, K = 70, 160
    codes, scales = _weight(rng, (N, K), "MXFP8_E5M2")
    x = torch.from_numpy(rng.standard_normal((M, K))).to(DTYPES[dtype])
    x[1, 3], x[0, 5] = float("nan"), float("inf")
    codes[:, 5] = 0x3C
    codes[7, 100], codes[9, 10] = 0x7E, 0x7C                                # NaN, +Inf
    scales[20, 4] = 255
    x[0, 10] = 2.0
    W = _matrix(codes, scales, "MXFP8_E5M2", K)
    y = nn.packed_linear(x.cuda(), codes.cuda(), scales.cuda(), "MXFP8_E5M2").double().cpu()
    want = x.double() @ W.cpu().t()
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.isnan(y[1]).all() and torch.isnan(y[:, 7]).all() and torch.isnan(y[:, 20]).all()
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(y) & inf, inf) and torch.equal(y[inf], want[inf]) and inf[0].sum() > 40


@pytest.mark.parametrize("M", [1, 33, 200])
def test_scale_range(cuda, M):
    """Scales from the smallest to those whose products still fit."""
    rng = np.random.default_rng(M)
    for fmt in TOP:
        codes, scales = _weight(rng, (64, 128), fmt, (20, 220))
        x = torch.from_numpy(rng.standard_normal((M, 128))).cuda()
        y = nn.packed_linear(x.float(), codes.cuda(), scales.cuda(), fmt)
        want, bound = om.linear(x.float(), _matrix(codes, scales, fmt, 128))
        _check(y, want, bound, fmt)


def test_float32_products_are_exact(cuda):
    """One product an output, 24-bit activations times codes: off by less than the one step that a single rounding of the
    whole product, in whatever direction, can take."""
    rng = np.random.default_rng(1)
    for fmt in TOP:
        codes, scales = _weight(rng, (40, 64), fmt)
        for M in (4, 50, 200):
            x = torch.zeros(M, 64)
            at = torch.from_numpy(rng.integers(0, 64, M))
            x[torch.arange(M), at] = torch.from_numpy(rng.standard_normal(M)).float()
            y = nn.packed_linear(x.cuda(), codes.cuda(), scales.cuda(), fmt)
            want = x.double() @ _matrix(codes, scales, fmt, 64).cpu().t()
            _check(y.cpu(), want, torch.finfo(torch.float32).eps * want.abs(), fmt)


def test_codes_of_the_library(cuda):
    """packed.quantize's bytes along the last axis, against its own dequantized values."""
    W = torch.randn(200, 352, device="cuda") * 0.05
    x = torch.randn(50, 352, device="cuda")
    for fmt in TOP:
        codes, scales = packed.quantize(W, fmt, axis=-1)
        y = nn.packed_linear(x, codes, scales, fmt)
        want, bound = om.linear(x, packed.dequantize(codes, scales, fmt, axis=-1).double())
        _check(y, want, bound, fmt)


# ---------------------------------------------------------------------------------------------- experts

def _experts(rng, T, k, E, N, K, fmt, dtype=torch.bfloat16, bias=False, activation=None, gated=False, sorted_rows=False, pairs=False,
             picks=None):
    rows = 2 * N if gated else N
    codes, scales = _weight(rng, (E, rows, K), fmt)
    e = torch.from_numpy(rng.integers(0, E, (T, k))) if picks is None else picks
    plan = nn.dispatch(e.cuda(), E)
    x = torch.from_numpy(rng.standard_normal((T * k if sorted_rows else T, K))).to(dtype).cuda()
    b = torch.from_numpy(rng.standard_normal((E, rows))).to(dtype).cuda() if bias else None
    y = nn.expert_linear(x, (_pairs(codes) if pairs else codes).cuda(), scales.cuda(), fmt, plan, bias=b, activation=activation,
                         gated=gated, sorted_rows=sorted_rows)
    assert y.shape == (T * k, N) and y.dtype == dtype
    order, offsets, _ = om.dispatch(e.numpy(), E)
    rows_of = torch.arange(T * k) if sorted_rows else torch.from_numpy(order) // k
    for i in range(E):
        mine = slice(int(offsets[i]), int(offsets[i + 1]))
        if mine.stop > mine.start:
            want, bound = om.linear(x[rows_of[mine].cuda()], _matrix(codes[i], scales[i], fmt, K), None if b is None else b[i], activation,
                                    gated, None, dtype)
            _check(y[mine], want, bound, (i, mine))
    assert (y[int(offsets[E]):] == 0).all()


@pytest.mark.parametrize("sorted_rows", [False, True])
@pytest.mark.parametrize("T, k, E", [(1, 1, 1), (1, 8, 16), (5, 2, 3), (64, 2, 8), (200, 6, 64), (700, 2, 4), (40, 3, 200)])
def test_experts(cuda, T, k, E, sorted_rows):
    rng = np.random.default_rng(T + E)
    _experts(rng, T, k, E, 48, 96, "MXFP8_E4M3", sorted_rows=sorted_rows)
    _experts(rng, T, k, E, 40, 65, "MXFP4", torch.float16, True, "silu", True, sorted_rows, pairs=True)


def test_experts_of_unlike_loads(cuda):
    """All rows with one expert, experts without rows, slots of no expert, and nobody with any."""
    rng = np.random.default_rng(5)
    one = torch.full((300, 2), 6)
    some = torch.from_numpy(rng.integers(-3, 12, (300, 2)))
    none = torch.full((30, 2), -1)
    for picks in (one, some, none):
        for sorted_rows in (False, True):
            _experts(rng, len(picks), 2, 9, 130, 128, "MXFP8_E4M3", bias=True, sorted_rows=sorted_rows, picks=picks)
    _experts(rng, 3000, 1, 2, 264, 64, "MXFP6_E3M2", picks=torch.from_numpy(rng.integers(0, 2, (3000, 1))))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt", list(TOP))
def test_experts_formats_and_types(cuda, fmt, dtype):
    rng = np.random.default_rng(9)
    for T in (6, 150):
        _experts(rng, T, 2, 4, 100, 200, fmt, DTYPES[dtype], True, "gelu", False)


def test_expert_strides(cuda):
    rng = np.random.default_rng(12)
    codes, scales = (t.cuda() for t in _weight(rng, (4, 96, 128), "MXFP8_E4M3"))
    plan = nn.dispatch(torch.from_numpy(rng.integers(0, 4, (90, 2))).cuda(), 4)
    x = torch.randn(90, 128, device="cuda", dtype=torch.bfloat16)
    want = nn.expert_linear(x, codes, scales, "MXFP8_E4M3", plan)
    assert torch.equal(nn.expert_linear(x, codes.transpose(0, 2).contiguous().transpose(0, 2), scales, "MXFP8_E4M3", plan), want)
    wide = torch.zeros(90, 150, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:131] = x
    every = torch.zeros(8, 100, 140, device="cuda", dtype=torch.uint8)
    every[::2, 2:98, 5:133] = codes
    assert torch.equal(nn.expert_linear(wide[:, 3:131], every[::2, 2:98, 5:133], scales, "MXFP8_E4M3", plan), want)
    cpu = nn.expert_linear(x.cpu(), codes.cpu(), scales.cpu(), "MXFP8_E4M3", nn.dispatch(torch.zeros(90, 2, dtype=torch.int64), 4))
    assert cpu.device.type == "cpu" and cpu.shape == (180, 96)


def test_layer_captured_in_a_graph(cuda):
    """A whole layer replayed on new inputs, eager calls between: each replay equals the eager result."""
    rng = np.random.default_rng(3)
    E, D, F = 8, 128, 96
    up, down = _weight(rng, (E, 2 * F, D), "MXFP8_E4M3", (118, 122)), _weight(rng, (E, D, F), "MXFP8_E4M3", (118, 122))
    up, down = [t.cuda() for t in up], [t.cuda() for t in down]
    for T in (3, 150):
        x, l = torch.randn(T, D, device="cuda", dtype=torch.bfloat16), torch.randn(T, E, device="cuda")

        def layer():
            w, e = nn.route(l, 2)
            plan = nn.dispatch(e, E)
            h = nn.expert_linear(x, *up, "MXFP8_E4M3", plan, activation="silu", gated=True)
            return nn.combine(nn.expert_linear(h, *down, "MXFP8_E4M3", plan, sorted_rows=True), w, plan, residual=x)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer()
        for _ in range(4):
            x.normal_()
            l.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, layer())


def _far(t, stride):
    """t's rows `stride` elements apart."""
    there = torch.empty((t.shape[0] - 1) * stride + t.shape[1], dtype=t.dtype, device="cuda").as_strided(t.shape, (stride, 1))
    return there.copy_(t)


def test_rows_2_32_bytes_apart(cuda):
    """Tiles whose rows' offsets need more than 32 bits: the same bits as of neighbouring rows."""
    rng = np.random.default_rng(30)
    for K in (256, 200):
        codes, scales = (t.cuda() for t in _weight(rng, (150, K), "MXFP8_E4M3"))
        x = torch.from_numpy(rng.standard_normal((130, K))).to(torch.bfloat16).cuda()
        want = nn.packed_linear(x, codes, scales, "MXFP8_E4M3")
        assert torch.equal(nn.packed_linear(x, _far(codes, 1 << 25), scales, "MXFP8_E4M3"), want)
        assert torch.equal(nn.packed_linear(_far(x, 1 << 24), codes, scales, "MXFP8_E4M3"), want)
        gated = nn.packed_linear(x, codes, scales, "MXFP8_E4M3", activation="silu", gated=True)
        assert torch.equal(nn.packed_linear(x, _far(codes, 1 << 25), scales, "MXFP8_E4M3", activation="silu", gated=True), gated)
        experts, es = (t.cuda() for t in _weight(rng, (3, 96, K), "MXFP8_E4M3"))
        plan = nn.dispatch(torch.from_numpy(rng.integers(0, 3, (130, 2))).cuda(), 3)
        want = nn.expert_linear(x, experts, es, "MXFP8_E4M3", plan)
        assert torch.equal(nn.expert_linear(_far(x, 1 << 24), experts, es, "MXFP8_E4M3", plan), want)
