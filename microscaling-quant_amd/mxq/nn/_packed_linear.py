"""Products with packed MX weights: codes and scales as mxq.packed writes them, activations and outputs in the model's
own dtype.  Not in the reference, whose products take float32 codes of both operands and round inside the sum.

    codes, scales = mxq.packed.quantize(W, fmt, axis=-1)                 W: out x in
    y = packed_linear(x, codes, scales, fmt, bias=b, activation="gelu", residual=r)
    h = expert_linear(x, codes, scales, fmt, plan, activation="silu", gated=True)     codes: E x 2 out x in

y = act(x W^T + bias) + residual; gated: act(x G^T + b) * (x U^T + c) + residual, where the weight's first half of rows
is G and the second U (bias likewise).  Each product of an activation and a weight is exact, sums are float32, and y
is rounded once.  A weight is its code times its scale; below 2^-126 it is rounded to bfloat16's subnormals, from 2^128 on
it is infinite, as in packed.dequantize's float32.  The part of a float32 activation below 2^-133 is left out (only
one below 2^-110 has any).

For inference: codes have no gradient, and an input that asks for one is refused.
"""
from typing import Optional, Union

import torch

from .. import _lib
from ..element_quant.formats import Format, get
from ._moe import MAX_EXPERTS, Dispatch, _check_plan, _dtype, _no_tangent

__all__ = ["packed_linear", "expert_linear", "ACTIVATIONS"]

ACTIVATIONS = (None, "silu", "gelu", "gelu_tanh", "relu")
_FORMATS = {"MXFP8_E4M3": 0, "MXFP8_E5M2": 1, "MXFP6_E3M2": 2, "MXFP6_E2M3": 3, "MXFP4": 4}
_PAIRS = 5
BLOCK = 32


@_lib.memo_spec
def _weight(fmt, codes_shape, codes_dtype, scales_shape, scales_dtype, K, ndim, who):
    """The format code of a weight of K columns, its types and shapes checked."""
    f = get(fmt)
    code = None if f is None else _FORMATS.get(f.name)
    if code is None:
        raise ValueError(f"mxq.nn.{who}: fmt must name one of {tuple(_FORMATS)}, got {fmt!r}")
    if codes_dtype != torch.uint8 or scales_dtype != torch.uint8:
        raise TypeError(f"mxq.nn.{who}: codes and scales must be uint8, got {codes_dtype} and {scales_dtype}")
    if len(codes_shape) != ndim:
        raise ValueError(f"mxq.nn.{who}: codes must have {ndim} axes, got shape {tuple(codes_shape)}")
    if codes_shape[-1] != K:
        if code != _FORMATS["MXFP4"] or codes_shape[-1] != (K + 1) // 2:
            raise ValueError(f"mxq.nn.{who}: codes of shape {tuple(codes_shape)} do not hold {K} columns")
        code = _PAIRS
    if tuple(scales_shape) != (*codes_shape[:-1], -(-K // BLOCK)):
        raise ValueError(f"mxq.nn.{who}: scales must be {(*codes_shape[:-1], -(-K // BLOCK))}, got "
                         f"{tuple(scales_shape)}")
    return code


def _no_grad(who: str, *tensors) -> None:
    _no_tangent(who, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"mxq.nn.{who}: packed weights are for inference; call it under torch.no_grad()")


def _rows(t: Optional[torch.Tensor], dev) -> Optional[torch.Tensor]:
    """t on dev, its last axis's elements next to each other."""
    if t is None:
        return None
    t = _lib.to_device(t, dev)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _outputs(rows: int, gated: bool, who: str) -> int:
    if gated and rows % 2:
        raise ValueError(f"mxq.nn.{who}: a gated weight has an even number of rows, got {rows}")
    return rows // 2 if gated else rows


def _checked(x, bias, bias_shape, activation, out_dtype, who):
    _dtype(x, who, "x")
    if activation not in ACTIVATIONS:
        raise ValueError(f"mxq.nn.{who}: activation must be one of {ACTIVATIONS}, got {activation!r}")
    if bias is not None:
        _dtype(bias, who, "bias")
        if tuple(bias.shape) != bias_shape:
            raise ValueError(f"mxq.nn.{who}: bias must have shape {bias_shape}, got {tuple(bias.shape)}")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"mxq.nn.{who}: out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    return out_dtype


def _spec(x, bias, residual, y, codes, scales, code, activation, gated, top_k=0):
    dt = _lib.DTYPE_CODE
    batched = codes.ndim == 3
    return _lib.LinearSpec(
        dt[x.dtype], 0 if bias is None else dt[bias.dtype], 0 if residual is None else dt[residual.dtype], dt[y.dtype],
        code, ACTIVATIONS.index(activation), int(gated), top_k, x.stride(0), 0 if residual is None else
        residual.stride(0), y.stride(0), codes.stride(-2), scales.stride(-2), codes.stride(0) if batched else 0,
        scales.stride(0) if batched else 0, bias.stride(0) if batched and bias is not None else 0)


def _workspace(name: str, rows: int, each: int, dev, *args) -> Optional[torch.Tensor]:
    """What the kernels of this call need; nothing where a matrix has at most 16 rows of x."""
    if rows <= 16 * each:
        return None
    size = _lib.call(name, *args)
    return torch.empty(size, dtype=torch.uint8, device=dev) if size else None


def packed_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, fmt: Union[str, Format], *,
                  bias: Optional[torch.Tensor] = None, activation: Optional[str] = None, gated: bool = False,
                  residual: Optional[torch.Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x (... x K) by a packed weight (codes rows x K, scales rows x ceil(K / 32)): ... x N in out_dtype (x's dtype).

    MXFP4's codes may lie two to a byte, rows x ceil(K / 2), the even column in the low nibble.  N is the number of
    rows, half of it where gated.  bias: one value a row.  residual: the output's shape.  x, bias, residual and
    out_dtype are float32, bfloat16 or float16, each on its own."""
    who = "packed_linear"
    _no_grad(who, x, bias, residual)
    if x.ndim < 1:
        raise ValueError("mxq.nn.packed_linear: x must have a last axis to contract")
    K = x.shape[-1]
    code = _weight(fmt, codes.shape, codes.dtype, scales.shape, scales.dtype, K, 2, who)
    N = _outputs(codes.shape[0], gated, who)
    out_dtype = _checked(x, bias, (codes.shape[0],), activation, out_dtype, who)
    shape = (*x.shape[:-1], N)
    if residual is not None:
        _dtype(residual, who, "residual")
        if tuple(residual.shape) != shape:
            raise ValueError(f"mxq.nn.packed_linear: residual must have shape {shape}, got {tuple(residual.shape)}")
    dev = _lib.compute_device(x, codes)
    M = _lib.numel(shape[:-1])
    xd = _rows(x if x.ndim == 2 else x.reshape(M, K), dev)
    cd, sd, bd = _rows(codes, dev), _rows(scales, dev), _rows(bias, dev)
    rd = residual if residual is None or residual.ndim == 2 else residual.reshape(M, N)
    rd = _rows(rd, dev)
    y = torch.empty((M, N), dtype=out_dtype, device=dev)
    spec = _spec(xd, bd, rd, y, cd, sd, code, activation, gated)
    xp, cp, sp = xd.data_ptr(), cd.data_ptr(), sd.data_ptr()
    with _lib.on(dev):
        work = _workspace("mxq_packed_linear_workspace", M, 1, dev, xp, cp, sp, M, N, K, spec)
        _lib.run("mxq_packed_linear", xp, cp, sp, _lib.ptr(bd), _lib.ptr(rd), y.data_ptr(), M, N, K, spec,
                 _lib.ptr(work), _lib.stream(dev))
    return _lib.back(y if x.ndim == 2 else y.reshape(shape), x)


def expert_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, fmt: Union[str, Format], plan: Dispatch,
                  *, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None, gated: bool = False,
                  sorted_rows: bool = False, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """packed_linear with a weight an expert (codes E x rows x K, scales E x rows x ceil(K / 32), bias E x rows): a row
    for each of plan's slots, in the experts' order, n x N.

    x: tokens x K, each slot taking its token's row; sorted_rows: n x K, a row for each slot in the experts' order
    already, as a first product returns them.  Rows of no expert (plan's last) are zeros."""
    who = "expert_linear"
    _no_grad(who, x, bias)
    _check_plan(plan, who)
    T, k = plan.positions.shape
    n, E = T * k, plan.num_experts
    if x.ndim != 2 or x.shape[0] != (n if sorted_rows else T):
        raise ValueError(f"mxq.nn.expert_linear: x must have {n if sorted_rows else T} rows, got shape "
                         f"{tuple(x.shape)}")
    K = x.shape[1]
    code = _weight(fmt, codes.shape, codes.dtype, scales.shape, scales.dtype, K, 3, who)
    if codes.shape[0] != E or E > MAX_EXPERTS:
        raise ValueError(f"mxq.nn.expert_linear: codes of {codes.shape[0]} experts, plan has {E}")
    N = _outputs(codes.shape[1], gated, who)
    out_dtype = _checked(x, bias, tuple(codes.shape[:2]), activation, out_dtype, who)
    dev = _lib.compute_device(x, codes)
    xd, cd, sd, bd = (_rows(t, dev) for t in (x, codes, scales, bias))
    order, offsets = (_lib.to_device(t, dev).contiguous() for t in (plan.order, plan.offsets))
    y = torch.empty((n, N), dtype=out_dtype, device=dev)
    spec = _spec(xd, bd, None, y, cd, sd, code, activation, gated, 0 if sorted_rows else k)
    xp, cp, sp = xd.data_ptr(), cd.data_ptr(), sd.data_ptr()
    with _lib.on(dev):
        work = _workspace("mxq_expert_linear_workspace", n, E, dev, xp, cp, sp, n, N, K, E, spec)
        _lib.run("mxq_expert_linear", xp, cp, sp, _lib.ptr(bd), y.data_ptr(), n, N, K, E, order.data_ptr(),
                 offsets.data_ptr(), spec, _lib.ptr(work), _lib.stream(dev))
    return _lib.back(y, x)
