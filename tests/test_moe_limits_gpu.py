"""Sizes at which a launch would pass 2^32 threads, of which a part would run: sums of small whole numbers, which float32
holds exactly in any order, so that every result has to be equal."""
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


@pytest.mark.parametrize("T", [2 ** 22 + 1, 2 ** 24 + 3])
def test_combine_of_many_tokens(cuda, T):
    y = _whole(T, 2, torch.float32)
    w = _whole(T, 1, torch.float32, 1)
    plan = nn.Dispatch(torch.zeros(T, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"),
                       torch.arange(T - 1, -1, -1, dtype=torch.int32, device="cuda")[:, None])
    g = _whole(T, 2, torch.float32, 2)
    back = y.flip(0)
    out = nn.combine(y.requires_grad_(), w.requires_grad_(), plan)
    assert torch.equal(out, w * back)
    dy, dw = torch.autograd.grad(out, (y, w), g)
    assert torch.equal(dy, (w * g).flip(0)) and torch.equal(dw, (g * back).sum(1, keepdim=True))


def test_combine_of_many_groups(cuda):
    """More 16-byte groups than threads in the largest launch."""
    T = 2 ** 29 + 1000
    y = torch.empty(T, 9, dtype=torch.bfloat16, device="cuda")
    for part in y.split(1 << 26):
        part.copy_(torch.randint(-2, 3, part.shape, device="cuda", dtype=torch.int8))
    plan = nn.Dispatch(torch.zeros(T, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"),
                       torch.arange(T, dtype=torch.int32, device="cuda")[:, None])
    out = nn.combine(y, torch.full((T, 1), -2.0, device="cuda"), plan)
    for a, b in zip(out.split(1 << 26), y.split(1 << 26)):
        assert torch.equal(a, b * -2)


def test_route_of_many_tokens(cuda):
    T = 2 ** 28 + 5
    logits = torch.zeros(T, 2, dtype=torch.bfloat16, device="cuda")
    second = torch.randint(0, 2, (T,), device="cuda", dtype=torch.uint8)
    logits[:, 1] = second * 2.0 - 1.0
    logits.requires_grad_()
    w, e = nn.route(logits, 1, score="sigmoid", renormalize=False)
    assert torch.equal(e[:, 0], second.int())
    top = torch.stack([torch.tensor(0.5), torch.sigmoid(torch.tensor(1.0, dtype=torch.float64)).float()]).cuda()
    assert torch.equal(w[:, 0], top[second.int()])
    grad = torch.autograd.grad(w, logits, torch.ones_like(w))[0]
    for a, s in zip(grad.split(1 << 26), second.split(1 << 26)):
        assert (a.gather(1, s.long()[:, None]) > 0.19).all() and (a.gather(1, 1 - s.long()[:, None]) == 0).all()


def test_route_of_many_tokens_and_experts(cuda):
    """A wave a token."""
    T, E = 2 ** 26 + 3, 513
    if torch.cuda.mem_get_info()[0] < 110 * 2 ** 30:
        pytest.skip("less than 110 GiB free")
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device="cuda")
    at = torch.randint(0, E, (T, 1), device="cuda")
    logits.scatter_(1, at, 2.0)
    _, e = nn.route(logits, 1)
    assert torch.equal(e.long(), at)


@pytest.mark.parametrize("M", [1, 17])
def test_weight_rows_laid_out(cuda, M):
    """More rows of a weight than workgroups of 256 threads fit a launch."""
    N, K = 2 ** 24 + 5, 33
    codes, values = _codes(N, K)
    x = _whole(M, K)
    y = nn.packed_linear(x, codes, torch.full((N, 2), 127, dtype=torch.uint8, device="cuda"), "MXFP8_E4M3", out_dtype=torch.float32)
    assert torch.equal(y, x.float() @ values.t())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_x_laid_out(cuda, dtype):
    M, N, K = 2 ** 24 + 9, 2, 3
    codes, values = _codes(N, K)
    x = _whole(M, K, dtype)
    y = nn.packed_linear(x, codes, torch.full((N, 1), 127, dtype=torch.uint8, device="cuda"), "MXFP8_E4M3", out_dtype=torch.float32)
    assert torch.equal(y, x.float() @ values.t())


def test_outputs_past_a_launch_are_refused(cuda):
    N = 2 ** 28 + 17
    codes, scales = (torch.zeros(N, 1, dtype=torch.uint8, device="cuda") for _ in range(2))
    with pytest.raises(RuntimeError, match="too many outputs"):
        nn.packed_linear(torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16), codes, scales, "MXFP8_E4M3")
    fits = nn.packed_linear(torch.ones(1, 1, device="cuda", dtype=torch.bfloat16), torch.full_like(codes, 0x38)[:2 ** 28 - 16],
                            torch.full_like(scales, 127)[:2 ** 28 - 16], "MXFP8_E4M3")
    assert (fits == 1).all()
