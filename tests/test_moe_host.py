"""Refusals of the mixture-of-experts operators, on the CPU: every check runs before any device work.  And without a
GPU a valid call fails loudly."""
import ctypes

import pytest
import torch

from mxq import _lib, nn


def _plan(T=3, k=2, E=4):
    n = T * k
    return nn.Dispatch(torch.zeros(n, dtype=torch.int32), torch.zeros(E + 1, dtype=torch.int32),
                       torch.zeros(T, k, dtype=torch.int32))


def _u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


@pytest.mark.parametrize("kwargs, error, text", [
    (dict(top_k=0), ValueError, "top_k must be an integer from 1 to 8"),
    (dict(top_k=9), ValueError, "top_k must be an integer from 1 to 8"),
    (dict(top_k=True), ValueError, "top_k must be an integer"),
    (dict(top_k=2, groups=3), ValueError, "groups 3 must divide the 8 experts"),
    (dict(top_k=2, groups=2, top_groups=3), ValueError, "top_groups must be an integer from 1 to 2"),
    (dict(top_k=2, score="tanh"), ValueError, "score must be one of"),
    (dict(top_k=2, bias=torch.zeros(7)), ValueError, "bias must hold 8 values"),
])
def test_route_refuses(kwargs, error, text):
    with pytest.raises(error, match=text):
        nn.route(torch.zeros(3, 8), **kwargs)


def test_route_refuses_types_and_sizes():
    with pytest.raises(TypeError, match="logits must be float32"):
        nn.route(torch.zeros(3, 8, dtype=torch.float64), 2)
    with pytest.raises(ValueError, match="number of experts must be an integer from 1 to 1024"):
        nn.route(torch.zeros(1, 1025), 2)
    with pytest.raises(ValueError, match="experts axis"):
        nn.route(torch.zeros(()), 1)


def test_dispatch_and_combine_refuse():
    with pytest.raises(TypeError, match="experts must be int32 or int64"):
        nn.dispatch(torch.zeros(3, 2), 4)
    with pytest.raises(ValueError, match="tokens x top_k"):
        nn.dispatch(torch.zeros(3, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="num_experts must be an integer from 1 to 1024"):
        nn.dispatch(torch.zeros(3, 2, dtype=torch.int32), 0)
    plan, w = _plan(), torch.zeros(3, 2)
    with pytest.raises(TypeError, match="plan must be dispatch's"):
        nn.combine(torch.zeros(6, 4), w, (1, 2, 3))
    with pytest.raises(ValueError, match="plan does not hold"):
        nn.combine(torch.zeros(6, 4), w, plan._replace(order=plan.order[:5]))
    with pytest.raises(ValueError, match="y must have 6 rows"):
        nn.combine(torch.zeros(5, 4), w, plan)
    with pytest.raises(TypeError, match="y must be float32"):
        nn.combine(torch.zeros(6, 4, dtype=torch.float64), w, plan)
    with pytest.raises(ValueError, match="weights must be 3 x 2"):
        nn.combine(torch.zeros(6, 4), torch.zeros(2, 3), plan)
    with pytest.raises(ValueError, match="residual must be 3 x 4"):
        nn.combine(torch.zeros(6, 4), w, plan, residual=torch.zeros(3, 4, dtype=torch.float16))


@pytest.mark.parametrize("change, error, text", [
    (dict(fmt="FP32"), ValueError, "fmt must name one of"),
    (dict(fmt="MXFP9"), ValueError, "Unknown format"),
    (dict(codes=_u8(6, 63)), ValueError, "do not hold 64 columns"),
    (dict(codes=_u8(6, 32)), ValueError, "do not hold 64 columns"),          # pairs, but not of MXFP4
    (dict(codes=_u8(2, 3, 64)), ValueError, "codes must have 2 axes"),
    (dict(codes=torch.zeros(6, 64)), TypeError, "must be uint8"),
    (dict(scales=_u8(6, 3)), ValueError, "scales must be"),
    (dict(x=torch.zeros(5, 64, dtype=torch.float64)), TypeError, "x must be float32"),
    (dict(x=torch.zeros(5, 64, requires_grad=True)), RuntimeError, "torch.no_grad"),
    (dict(bias=torch.zeros(5)), ValueError, "bias must have shape"),
    (dict(bias=torch.zeros(6, dtype=torch.int32)), TypeError, "bias must be float32"),
    (dict(activation="tanh"), ValueError, "activation must be one of"),
    (dict(residual=torch.zeros(5, 5)), ValueError, "residual must have shape"),
    (dict(out_dtype=torch.int8), TypeError, "out_dtype must be"),
    (dict(codes=_u8(5, 64), scales=_u8(5, 2), gated=True), ValueError, "even number of rows"),
])
def test_packed_linear_refuses(change, error, text):
    args = {**dict(x=torch.zeros(5, 64), codes=_u8(6, 64), scales=_u8(6, 2), fmt="MXFP8_E4M3"), **change}
    with pytest.raises(error, match=text):
        nn.packed_linear(**args)


@pytest.mark.parametrize("change, error, text", [
    (dict(x=torch.zeros(6, 64)), ValueError, "x must have 3 rows"),
    (dict(sorted_rows=True), ValueError, "x must have 6 rows"),
    (dict(codes=_u8(3, 6, 64), scales=_u8(3, 6, 2)), ValueError, "codes of 3 experts, plan has 4"),
    (dict(plan=None), TypeError, "plan must be dispatch's"),
    (dict(bias=torch.zeros(6)), ValueError, "bias must have shape"),
])
def test_expert_linear_refuses(change, error, text):
    args = {**dict(x=torch.zeros(3, 64), codes=_u8(4, 6, 64), scales=_u8(4, 6, 2), fmt="MXFP8_E4M3", plan=_plan()), **change}
    with pytest.raises(error, match=text):
        nn.expert_linear(**args)


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is visible")
def test_no_gpu_fails_loudly():
    with pytest.raises(RuntimeError, match="no GPU is visible"):
        nn.route(torch.zeros(3, 8), 2)
    with pytest.raises(RuntimeError, match="no GPU is visible"):
        nn.dispatch(torch.zeros(3, 2, dtype=torch.int64), 4)
    with pytest.raises(RuntimeError, match="no GPU is visible"):
        nn.combine(torch.zeros(6, 4), torch.zeros(3, 2), _plan())
    with pytest.raises(RuntimeError, match="no GPU is visible"):
        nn.packed_linear(torch.zeros(5, 64), _u8(6, 64), _u8(6, 2), "MXFP8_E4M3")
    with pytest.raises(RuntimeError, match="no GPU is visible"):
        nn.expert_linear(torch.zeros(3, 64), _u8(4, 6, 64), _u8(4, 6, 2), "MXFP8_E4M3", _plan())


def test_c_entries_refuse():
    """Bad sizes, specs and NULL arguments come back as MXQ_EINVAL with a message, before any HIP call."""
    lib = _lib.load()
    buf = ctypes.cast((ctypes.c_uint8 * 4096)(), ctypes.c_void_p)

    def refused(text, name, *args):
        assert getattr(lib, name)(*args) == 1, (name, args)
        assert text in lib.mxq_last_error().decode(), lib.mxq_last_error()

    good = dict(score=0, top_k=2, groups=1, top_groups=1, renormalize=1, scale=1.0)
    for change, text in ((dict(score=2), "score"), (dict(top_k=0), "top_k"), (dict(top_k=9), "top_k"),
                         (dict(groups=3), "groups"), (dict(groups=0), "groups"), (dict(top_groups=2), "top_groups")):
        spec = _lib.RouteSpec(**{**good, **change})
        refused(text, "mxq_route", buf, 0, 0, 4, 8, spec, buf, buf, 0)
        refused(text, "mxq_route_grad", buf, 0, buf, buf, 4, 8, spec, buf, 0)
    spec = _lib.RouteSpec(**good)
    refused("NULL", "mxq_route", 0, 0, 0, 4, 8, spec, buf, buf, 0)
    refused("experts", "mxq_route", buf, 0, 0, 4, 1025, spec, buf, buf, 0)
    refused("dtype", "mxq_route", buf, 3, 0, 4, 8, spec, buf, buf, 0)
    refused("out of range", "mxq_route", buf, 0, 0, -1, 8, spec, buf, buf, 0)
    refused("out of range", "mxq_dispatch", buf, -1, 8, buf, buf, buf, 0)
    refused("experts", "mxq_dispatch", buf, 4, 0, buf, buf, buf, 0)
    refused("NULL", "mxq_dispatch", buf, 4, 8, buf, 0, buf, 0)
    refused("top_k", "mxq_combine", buf, 0, buf, buf, 0, buf, 4, 65, 8, 0)
    refused("slots", "mxq_combine", buf, 0, buf, buf, 0, buf, 1 << 30, 4, 8, 0)
    refused("NULL", "mxq_combine", 0, 0, buf, buf, 0, buf, 4, 2, 8, 0)
    refused("NULL", "mxq_combine_grad", buf, 0, buf, buf, 0, buf, 0, 4, 2, 8, 0)
    lin = _lib.LinearSpec(ld_x=64, ld_y=8, ld_codes=64, ld_scales=2)
    for field, value, text in (("x_dtype", 3, "dtype"), ("y_dtype", -1, "dtype"), ("format", 6, "format"),
                               ("activation", 5, "activation")):
        bad = _lib.LinearSpec(ld_x=64, ld_y=8, ld_codes=64, ld_scales=2)
        setattr(bad, field, value)
        refused(text, "mxq_packed_linear", buf, buf, buf, 0, 0, buf, 4, 8, 64, bad, 0, 0)
    refused("NULL", "mxq_packed_linear", buf, 0, buf, 0, 0, buf, 4, 8, 64, lin, 0, 0)
    refused("size", "mxq_packed_linear", buf, buf, buf, 0, 0, buf, 4, -8, 64, lin, 0, 0)
    refused("experts", "mxq_expert_linear", buf, buf, buf, 0, buf, 4, 8, 64, 0, buf, buf, lin, 0, 0)
    refused("NULL", "mxq_expert_linear", buf, buf, buf, 0, buf, 4, 8, 64, 2, buf, 0, lin, 0, 0)
    lin.top_k = 65
    refused("top_k", "mxq_expert_linear", buf, buf, buf, 0, buf, 4, 8, 64, 2, buf, buf, lin, 0, 0)


def test_specs_are_remembered_by_value():
    """A scale held in a tensor is read in every call: a tensor's hash is its identity, which a change in place keeps."""
    from mxq.nn._moe import _route_spec
    scale = torch.tensor(2.5)
    assert _route_spec(8, 2, "softmax", 1, 1, True, scale).scale == 2.5
    scale.mul_(2)
    assert _route_spec(8, 2, "softmax", 1, 1, True, scale).scale == 5.0
    assert _route_spec(8, 2, "softmax", 1, 1, True, 2.5) is _route_spec(8, 2, "softmax", 1, 1, True, 2.5)
    from mxq.block import mxgemmini
    from mxq.element_quant.formats import get
    f, floor = get("MXFP8_E4M3"), torch.tensor(0.5)
    assert mxgemmini.spec(f, "ties_away", floor, None).scale_floor == 0.5
    floor.fill_(0.25)
    assert mxgemmini.spec(f, "ties_away", floor, None).scale_floor == 0.25
    assert mxgemmini.spec(f, "ties_away", 0.5, None) is mxgemmini.spec(f, "ties_away", 0.5, None)


def test_forward_mode_tangents_are_refused():
    """An input of forward-mode differentiation does not ask for a gradient; its tangent must not be taken for zero."""
    from torch.autograd import forward_ad

    dual = lambda *shape: forward_ad.make_dual(torch.zeros(shape), torch.ones(shape))
    packed = dict(codes=_u8(6, 64), scales=_u8(6, 2), fmt="MXFP8_E4M3")
    experts = dict(codes=_u8(4, 6, 64), scales=_u8(4, 6, 2), fmt="MXFP8_E4M3", plan=_plan())
    plain = torch.zeros
    with forward_ad.dual_level():
        for call in (lambda: nn.route(dual(3, 8), 2),
                     lambda: nn.combine(dual(6, 4), plain(3, 2), _plan()),
                     lambda: nn.combine(plain(6, 4), dual(3, 2), _plan()),
                     lambda: nn.combine(plain(6, 4), plain(3, 2), _plan(), residual=dual(3, 4)),
                     lambda: nn.packed_linear(dual(5, 64), **packed),
                     lambda: nn.packed_linear(plain(5, 64), **packed, bias=dual(6)),
                     lambda: nn.packed_linear(plain(5, 64), **packed, residual=dual(5, 6)),
                     lambda: nn.expert_linear(dual(3, 64), **experts),
                     lambda: nn.expert_linear(plain(3, 64), **experts, bias=dual(4, 6))):
            for grad in (True, False):                 # torch.no_grad does not end forward mode
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    call()


def test_layer_refuses_an_input_that_asks_for_a_gradient(monkeypatch):
    """The experts' products have no gradient of x: the router's share of it alone must not pass for the whole."""
    from experiments import moe_layer
    monkeypatch.setattr(moe_layer.nn, "route", lambda l, k: (torch.zeros(3, k), torch.zeros(3, k, dtype=torch.int32)))
    monkeypatch.setattr(moe_layer.nn, "dispatch", lambda e, n: _plan(3, 2, n))
    layer = moe_layer.MoELayer(torch.zeros(4, 64), (_u8(4, 12, 64), _u8(4, 12, 2)), (_u8(4, 64, 6), _u8(4, 64, 1)))
    with pytest.raises(RuntimeError, match="torch.no_grad"):
        layer(torch.zeros(3, 64, requires_grad=True))
