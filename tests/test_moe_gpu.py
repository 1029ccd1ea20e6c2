"""Routing, the slots' order and the weighted sum against 64 bits.  Experts, orders and positions have to be equal;
weights are within two of float32's half steps (the 64-bit value rounded, times a float32 scale), sums within k + 1 of
them and the output's rounding."""
import numpy as np
import pytest
import torch

from mxq import nn
from oracle import moe as om

pytestmark = pytest.mark.gpu
HALF = torch.finfo(torch.float32).eps / 2
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _logits(rng, T, E, dtype, masked=0.0):
    l = torch.from_numpy(rng.standard_normal((T, E)) * 2).to(dtype)
    if masked:
        l[torch.from_numpy(rng.random((T, E)) < masked)] = -np.inf
        l[0] = -np.inf                                                     # a row with nothing open
    return l


def _close(got, want, bound, what=""):
    got, want, bound = (torch.as_tensor(t).double().cpu() for t in (got, want, bound))
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    off = (got - want).abs() - bound
    assert not (off[~nan] > 0).any(), (what, float(off[~nan].max()))


SHAPES = [(1, 1, 1), (1, 64, 8), (5, 2, 2), (33, 7, 3), (17, 65, 6), (9, 128, 4), (40, 160, 8), (3, 512, 64), (7, 1000, 16),
          (130, 1024, 2)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T, E, k", SHAPES)
def test_route(cuda, T, E, k, dtype, score):
    rng = np.random.default_rng(T * 1000 + E)
    for masked, with_bias, renormalize in ((0.0, False, True), (0.3, True, False), (0.9, False, True)):
        l = _logits(rng, T, E, DTYPES[dtype], masked)
        bias = torch.from_numpy(rng.standard_normal(E) * 0.2).float() if with_bias else None
        w, e = nn.route(l.cuda(), k, score=score, bias=None if bias is None else bias.cuda(), renormalize=renormalize, scale=2.5)
        ww, we, _ = om.route(l.double().numpy(), k, score, None if bias is None else bias.double().numpy(), renormalize=renormalize, scale=2.5)
        assert w.dtype == torch.float32 and e.dtype == torch.int32
        assert np.array_equal(e.cpu().numpy(), we), (masked, with_bias)
        _close(w, ww, 2 * HALF * np.abs(ww) + 2.0 ** -149)


@pytest.mark.parametrize("E, groups, top_groups, k", [(8, 8, 3, 2), (64, 4, 1, 8), (256, 8, 4, 8), (96, 6, 2, 30), (1024, 64, 5, 16)])
def test_route_groups(cuda, E, groups, top_groups, k):
    rng = np.random.default_rng(E + groups)
    for score in ("softmax", "sigmoid"):
        for masked in (0.0, 0.95):
            l = _logits(rng, 29, E, torch.float32, masked)
            bias = rng.standard_normal(E).astype(np.float32) * 0.3
            args = dict(score=score, groups=groups, top_groups=top_groups)
            w, e = nn.route(l.cuda(), k, bias=torch.from_numpy(bias).cuda(), **args)
            ww, we, _ = om.route(l.double().numpy(), k, bias=bias, **args)
            assert np.array_equal(e.cpu().numpy(), we)
            _close(w, ww, 2 * HALF * np.abs(ww) + 2.0 ** -149)


def test_route_ties_go_to_the_lowest_index(cuda):
    l = torch.zeros(3, 200, device="cuda")
    l[1, 100:] = 1.0
    l[2, ::7] = -1.0
    l[0, 5] = -0.0
    for score in ("softmax", "sigmoid"):
        _, e = nn.route(l, 4, score=score)
        assert e.tolist() == [[0, 1, 2, 3], [100, 101, 102, 103], [1, 2, 3, 4]]


def test_route_close_scores(cuda):
    """Neighbouring float32 logits: the scores differ by less than float32 resolves near 1, the experts do not."""
    base = torch.full((64, 128), 4.0)
    step = torch.randperm(128, generator=torch.Generator().manual_seed(3))
    l = (base.view(torch.int32) + step.int()).view(torch.float32)
    for score in ("softmax", "sigmoid"):
        _, e = nn.route(l.cuda(), 16, score=score)
        assert torch.equal(e.cpu(), step.argsort(descending=True)[:16].int().expand(64, 16))


def test_route_far_and_special_logits(cuda):
    inf, nan = np.inf, np.nan
    l = torch.tensor([[0, 1, nan, 2], [0, 1, inf, 2], [-inf, -inf, -inf, -inf], [-inf, 3, -inf, -inf],
                      [3e38, -3e38, 0, 0], [-3e38, -3e38, -3e38, -3e38], [-800, -700, -750, 0]])
    bias = torch.tensor([0.0, 0.0, 9.0, 0.0])
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            w, e = nn.route(l.cuda(), 3, score=score, bias=None if b is None else b.cuda())
            ww, we, _ = om.route(l.double().numpy(), 3, score, None if b is None else b.numpy())
            assert np.array_equal(e.cpu().numpy(), we), (score, b)
            _close(w, ww, 2 * HALF * np.abs(ww) + 2.0 ** -149, score)
    w, e = nn.route(torch.zeros(2, 4).cuda(), 2, bias=torch.tensor([0, nan, 0, 0]).cuda())
    assert torch.isnan(w).all() and (e == -1).all()


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T, E, k, dtype", [(1, 1, 1, "f32"), (37, 64, 6, "bf16"), (9, 300, 16, "f32"), (5, 1024, 64, "f16"), (70, 8, 8, "f32")])
def test_route_gradient(cuda, T, E, k, dtype, score, renormalize):
    """Against the formula; and the formula against differences, in 64 bits."""
    rng = np.random.default_rng(E)
    l = _logits(rng, T, E, DTYPES[dtype], 0.2)
    g = torch.from_numpy(rng.standard_normal((T, k))).float()
    args = dict(score=score, renormalize=renormalize, scale=1.5)
    leaf = l.cuda().requires_grad_()
    w, e = nn.route(leaf, k, **args)
    assert not e.requires_grad
    w.backward(g.cuda())
    _, we, s = om.route(l.double().numpy(), k, **args)
    want = om.route_grad(s, we, g.numpy(), **args)
    eps = torch.finfo(DTYPES[dtype])
    _close(leaf.grad, want, (eps.eps / 2 + 2.0 ** -40) * np.abs(want) + 2.0 ** -40 + eps.smallest_normal * eps.eps)
    t, e0 = min(1, T - 1), int(we[min(1, T - 1), 0])
    if e0 >= 0:
        far = []
        for d in (1e-6, -1e-6):
            moved = l.double().numpy().copy()
            moved[t, e0] += d
            far.append((om.route(moved, k, **args)[0][t] * g[t].double().numpy()).sum())
        assert abs((far[0] - far[1]) / 2e-6 - want[t, e0]) < 1e-6


def test_route_gradient_of_a_row_without_scores(cuda):
    l = torch.zeros(3, 4, device="cuda")
    l[1, 2] = np.nan
    l[2] = -np.inf
    l.requires_grad_()
    w, _ = nn.route(l, 2)
    w.sum().backward()
    assert torch.isnan(l.grad[1]).all() and (l.grad[2] == 0).all() and torch.isfinite(l.grad[0]).all()


def test_route_layouts_devices_streams(cuda):
    rng = np.random.default_rng(4)
    l = _logits(rng, 48, 96, torch.float32)
    w, e = nn.route(l.cuda(), 5)
    for other in (l, l.t().contiguous().t().cuda(), torch.stack([l, l], 1).cuda()[:, 1], l.reshape(6, 8, 96).cuda()):
        w2, e2 = nn.route(other, 5)
        assert w2.device == other.device and w2.shape == (*other.shape[:-1], 5)
        assert torch.equal(w2.reshape(48, 5).cpu(), w.cpu()) and torch.equal(e2.reshape(48, 5).cpu(), e.cpu())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w2, _ = nn.route(l.cuda(), 5)
    side.synchronize()
    assert torch.equal(w2, w)
    w0, e0 = nn.route(torch.zeros(0, 8, device="cuda"), 2)
    assert w0.shape == e0.shape == (0, 2)


@pytest.mark.parametrize("T, k, E", [(0, 2, 4), (1, 1, 1), (1, 8, 64), (7, 3, 5), (100, 2, 1024), (1000, 3, 17), (2048, 8, 256), (40000, 2, 1000)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_dispatch(cuda, T, k, E, dtype):
    rng = np.random.default_rng(T + E)
    for high in (E, min(E, 2)):
        e = rng.integers(0, high, (T, k))
        if T > 1:
            e[rng.random((T, k)) < 0.1] = -1
            e[0, 0], e[-1, -1] = E, (1 << 40 if dtype == torch.int64 else 1 << 30)
        plan = nn.dispatch(torch.from_numpy(e).to(dtype).cuda(), E)
        key = np.where((e >= 0) & (e < E), e, E).reshape(-1)
        order = np.argsort(key, kind="stable")
        assert plan.num_experts == E and plan.top_k == k
        assert np.array_equal(plan.order.cpu().numpy(), order)
        assert np.array_equal(plan.offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])]))
        place = np.empty(T * k, dtype=np.int64)
        place[order] = np.arange(T * k)
        assert np.array_equal(plan.positions.cpu().numpy().reshape(-1), np.where(key < E, place, -1 - place))


def _combine_case(rng, T, k, D, E, dtype, dropped=0.2):
    e = torch.from_numpy(rng.integers(0, E, (T, k)))
    e[torch.from_numpy(rng.random((T, k)) < dropped)] = -1
    y = torch.from_numpy(rng.standard_normal((T * k, D))).to(dtype)
    w = torch.from_numpy(rng.random((T, k))).float()
    r = torch.from_numpy(rng.standard_normal((T, D))).to(dtype)
    return e, y, w, r


def _combine_64(e, y, w, r, E):
    order, offsets, place = om.dispatch(e.numpy(), E)
    place = torch.from_numpy(place)
    rows = y.double()[place.clamp_min(0)] * (place >= 0)[..., None]
    terms = rows * w.double()[..., None]
    out, size = terms.sum(1), terms.abs().sum(1)
    if r is not None:
        out, size = out + r.double(), size + r.double().abs()
    return out, size, place


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T, k, D, E", [(1, 1, 1, 1), (1, 2, 4096, 8), (7, 3, 33, 5), (19, 8, 1030, 64), (130, 4, 264, 9), (3, 64, 72, 70)])
def test_combine(cuda, T, k, D, E, dtype):
    rng = np.random.default_rng(T * D)
    e, y, w, r = _combine_case(rng, T, k, D, E, DTYPES[dtype])
    eps = torch.finfo(DTYPES[dtype])
    plan = nn.dispatch(e.cuda(), E)
    for res in (None, r):
        out = nn.combine(y.cuda(), w.cuda(), plan, residual=None if res is None else res.cuda())
        want, size, _ = _combine_64(e, y, w, res, E)
        _close(out, want, eps.eps / 2 * want.abs() + (k + 2) * HALF * size + eps.smallest_normal * eps.eps)
        assert torch.equal(out, nn.combine(y.cuda(), w.cuda(), plan, residual=None if res is None else res.cuda()))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T, k, D, E", [(1, 1, 1, 1), (7, 3, 33, 5), (19, 8, 1030, 64), (130, 4, 264, 9), (2, 5, 4096, 3)])
def test_combine_gradients(cuda, T, k, D, E, dtype):
    """dy = w g, dw = <g, y>, the residual's is g: the formulas in 64 bits, and differences of a linear function, exact."""
    rng = np.random.default_rng(T + D)
    e, y, w, r = _combine_case(rng, T, k, D, E, DTYPES[dtype])
    g = torch.from_numpy(rng.standard_normal((T, D))).to(DTYPES[dtype])
    eps = torch.finfo(DTYPES[dtype])
    leaves = [t.cuda().requires_grad_() for t in (y, w, r)]
    out = nn.combine(leaves[0], leaves[1], nn.dispatch(e.cuda(), E), residual=leaves[2])
    dy, dw, dr = torch.autograd.grad(out, leaves, g.cuda())
    assert torch.equal(dr.cpu(), g)
    _, _, place = _combine_64(e, y, w, None, E)
    live = place >= 0
    want_dy = torch.zeros(T * k, D, dtype=torch.float64)
    want_dy[place[live]] = (w.double()[..., None] * g.double()[:, None])[live]
    _close(dy, want_dy, (eps.eps / 2 + HALF) * want_dy.abs() + eps.smallest_normal * eps.eps)
    terms = g.double()[:, None] * y.double()[place.clamp_min(0)] * live[..., None]
    _close(dw, terms.sum(-1), (D + 2) * HALF * terms.abs().sum(-1) + 2.0 ** -149)
    moved = y.double().clone()
    moved[0, 0] += 1.0
    far = (_combine_64(e, moved, w, r, E)[0] - _combine_64(e, y, w, r, E)[0]) * g.double()
    assert abs(float(far.sum()) - float(want_dy[0, 0])) < 1e-9
    only = nn.combine(y.cuda(), leaves[1], nn.dispatch(e.cuda(), E))
    assert torch.equal(torch.autograd.grad(only, leaves[1], g.cuda())[0], dw)


def test_combine_leaves_out_rows_of_no_expert(cuda):
    """NaN and infinities in rows that no slot has do not come through, a NaN weight does."""
    e = torch.tensor([[0, -1], [-1, -1], [1, 0]])
    plan = nn.dispatch(e.cuda(), 2)
    y = torch.ones(6, 40)
    y[3:] = float("nan")
    w = torch.full((3, 2), 0.5)
    out = nn.combine(y.cuda(), w.cuda(), plan)
    assert out.cpu().tolist() == [[0.5] * 40, [0.0] * 40, [1.0] * 40]
    w[1, 0] = float("nan")
    out = nn.combine(y.cuda(), w.cuda(), plan)
    assert torch.isnan(out[1]).all() and not torch.isnan(out[0]).any() and not torch.isnan(out[2]).any()
    out = nn.combine(torch.zeros(0, 8).cuda(), torch.zeros(0, 2).cuda(), nn.dispatch(torch.zeros(0, 2, dtype=torch.int32).cuda(), 3))
    assert out.shape == (0, 8)
    assert nn.combine(torch.zeros(6, 0).cuda(), w.cuda(), plan).shape == (3, 0)


def test_combine_strides_and_devices(cuda):
    rng = np.random.default_rng(8)
    e, y, w, r = _combine_case(rng, 21, 3, 50, 6, torch.bfloat16)
    plan = nn.dispatch(e.cuda(), 6)
    want = nn.combine(y.cuda(), w.cuda(), plan, residual=r.cuda()).cpu()
    wide = torch.zeros(63, 101, dtype=torch.bfloat16)
    wide[:, 1:51] = y
    assert torch.equal(nn.combine(wide.cuda()[:, 1:51], w.t().contiguous().cuda().t(), plan, residual=r.cuda()).cpu(), want)
    cpu = nn.combine(y, w, nn.dispatch(e, 6), residual=r)
    assert cpu.device.type == "cpu" and torch.equal(cpu, want)


def test_route_to_combine_captured_in_a_graph(cuda):
    """Routing, order and sum replayed with new inputs between eager calls: each replay equals the eager result."""
    rng = np.random.default_rng(2)
    l = _logits(rng, 64, 32, torch.float32).cuda()
    y = torch.randn(64 * 4, 96, device="cuda", dtype=torch.bfloat16)

    def step():
        w, e = nn.route(l, 4)
        return nn.combine(y, w, nn.dispatch(e, 32))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        l.copy_(torch.randn(64, 32))
        y.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


def test_second_derivatives_are_refused(cuda):
    """Not taken for zero: a graph of the gradient can be asked for, a derivative through it cannot."""
    l = torch.randn(4, 8, device="cuda", requires_grad=True)
    w, _ = nn.route(l, 2)
    g = torch.autograd.grad(w.square().sum(), l, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    y = torch.randn(8, 5, device="cuda", requires_grad=True)
    out = nn.combine(y, torch.rand(4, 2, device="cuda"), nn.dispatch(torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 1))
    g = torch.autograd.grad(out.square().sum(), y, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_forward_and_backward_captured_in_a_graph(cuda):
    """A step with its gradients captured with no eager graph of its leaves alive; each replay equals an eager step."""
    rng = np.random.default_rng(6)
    l = _logits(rng, 40, 16, torch.float32).cuda().requires_grad_()
    y = torch.randn(80, 24, device="cuda", requires_grad=True)
    g = torch.randn(40, 24, device="cuda")

    def step():
        w, e = nn.route(l, 2)
        out = nn.combine(y, w, nn.dispatch(e, 16))
        return (out.detach(), *torch.autograd.grad(out, (l, y), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(4):
        with torch.no_grad():
            l.normal_()
            y.normal_()
            g.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T, k, D", [(3, 2, 40), (5, 7, 33)])
def test_combine_holds_positions_to_the_rows(cuda, T, k, D, dtype):
    """Positions past the last row, in a plan that is not dispatch's: as slots of no expert, and nothing outside y and dy is
    read or written."""
    from mxq import _lib
    rng = np.random.default_rng(D)
    n, dt = T * k, _lib.DTYPE_CODE[DTYPES[dtype]]
    place = torch.from_numpy(rng.permutation(n).astype(np.int32)).reshape(T, k)
    far = torch.from_numpy(rng.integers(0, 3, (T, k))) == 0
    far[0, 0], far[0, 1] = True, False
    held = torch.where(far, torch.tensor(-1, dtype=torch.int32), place).cuda()
    wild = torch.tensor([n, n + 1, 2 ** 31 - 1, n + 5], dtype=torch.int32)[torch.from_numpy(rng.integers(0, 4, (T, k)))]
    place = torch.where(far, wild, place)
    place[far & (torch.from_numpy(rng.integers(0, 2, (T, k))) == 0)] = -2 ** 31          # a slot of none, its row far away too
    around = torch.full((n + 8, D), float("nan"), dtype=DTYPES[dtype], device="cuda")
    around[:n] = torch.from_numpy(rng.standard_normal((n, D)))
    y, g = around[:n], torch.from_numpy(rng.standard_normal((T, D))).to(DTYPES[dtype]).cuda()
    w = torch.from_numpy(rng.random((T, k))).float().cuda()
    offsets = torch.zeros(2, dtype=torch.int32, device="cuda")
    plan = nn.Dispatch(torch.zeros(n, dtype=torch.int32, device="cuda"), offsets, place.cuda())
    assert torch.equal(nn.combine(y, w, plan), nn.combine(y, w, plan._replace(positions=held)))
    dy, dw = torch.full_like(around, 7), torch.empty(T, k, device="cuda")
    _lib.run("mxq_combine_grad", g.data_ptr(), dt, y.data_ptr(), w.data_ptr(), plan.positions.data_ptr(), dy.data_ptr(), dw.data_ptr(), T, k, D,
             _lib.stream(torch.device("cuda", 0)))
    named = torch.zeros(n + 8, dtype=torch.bool)
    named[place[~far].long()] = True
    assert (dy[~named.cuda()] == 7).all()
    _, want = torch.autograd.grad(nn.combine(y.requires_grad_(), w.requires_grad_(), plan._replace(positions=held)), (y, w), g)
    assert torch.equal(dw, want) and (dw.cpu()[far] == 0).all() and (dw.cpu()[~far] != 0).all()
    eps = torch.finfo(DTYPES[dtype])
    for t, j in torch.nonzero(~far).tolist():
        row = w[t, j].detach().double() * g[t].double()
        _close(dy[place[t, j].item()], row, (eps.eps / 2 + HALF) * row.abs() + eps.smallest_normal * eps.eps)
