"""A paged key and value cache in MX formats, and the attention that reads it.  Not in the reference, whose attention core
(mxq.nn.attend) emulates an accelerator's products on whole float32 tensors.

    cache = packed_cache(pages, page_size, kv_heads, head_dim, "MXFP4")
    cache_write(k, v, cache, slots)                        k, v: T x kv_heads x head_dim, quantized into the slots' rows
    out = cache_attend(q, cache, table, lengths)           q: B x n x heads x head_dim, n tokens a sequence
    out = cache_attend(q, cache, table, lengths, starts)   q: T x heads x head_dim, sequence b's from starts[b] on
    k, v = cache_read(cache, slots, torch.bfloat16)        the rows as values

Slot s is row s % page_size of page s // page_size.  Rows are quantized in blocks of 32 columns by the OCP rule, scale
2^(floor(log2 amax) - emax), elements to the nearest: the bytes of mxq.packed.quantize(x, fmt, "ocp", axis=-1), MXFP4's codes
two to a byte.  For inference: codes have no gradient, and an input that asks for one is refused.
"""
import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from .. import _lib
from ..element_quant.formats import Format, get
from ._moe import _dtype, _no_tangent, _whole
from ._packed_linear import BLOCK

__all__ = ["PackedCache", "packed_cache", "cache_write", "cache_read", "cache_attend"]

_FORMATS = {"MXFP8_E4M3": (0, 32), "MXFP8_E5M2": (1, 32), "MXFP4": (5, 16)}      # MXQ_FMT_* and a block's bytes
MAX_HEAD_DIM = 256
_MOST = 2 ** 31 - 1


class PackedCache(NamedTuple):
    """Codes pages x kv_heads x page_size x bytes and scales pages x kv_heads x page_size x blocks (E8M0), uint8, of keys
    and of values.  A row is a vector of head_dim columns in blocks of 32, the last filled up with zeros; a block is 32
    bytes, 16 of MXFP4, the even column in the low nibble.  Rows have their bytes next to each other; the other axes'
    strides are free."""
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    fmt: Union[str, Format]
    head_dim: int

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]


@_lib.memo_spec
def _format(fmt, who):
    f = get(fmt)
    found = None if f is None else _FORMATS.get(f.name)
    if found is None:
        raise ValueError(f"mxq.nn.{who}: a cache's fmt must name one of {tuple(_FORMATS)}, got {fmt!r}")
    return found


def packed_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, fmt: Union[str, Format] = "MXFP4", *,
                 device=None) -> PackedCache:
    """An empty cache (zeros) on `device`, the current GPU by default."""
    for what, value, high in (("pages", pages, _MOST), ("page_size", page_size, _MOST), ("kv_heads", kv_heads, 65535),
                              ("head_dim", head_dim, MAX_HEAD_DIM)):
        _whole(value, "packed_cache", what, 1, high)
    if pages * page_size > _MOST:
        raise ValueError(f"mxq.nn.packed_cache: {pages} pages of {page_size} rows are more than {_MOST} slots")
    each = _format(fmt, "packed_cache")[1]
    if device is None:
        device = _lib.compute_device()
    blocks = -(-head_dim // BLOCK)
    new = lambda last: torch.zeros((pages, kv_heads, page_size, last), dtype=torch.uint8, device=device)  # noqa: E731
    return PackedCache(new(blocks * each), new(blocks), new(blocks * each), new(blocks), fmt, head_dim)


@_lib.memo_spec
def _spec(fmt, head_dim, shapes, strides, who):
    """The cache's spec, its shapes checked."""
    code, each = _format(fmt, who)
    _whole(head_dim, who, "the cache's head_dim", 1, MAX_HEAD_DIM)
    blocks = -(-head_dim // BLOCK)
    if any(len(s) != 4 for s in shapes):
        raise ValueError(f"mxq.nn.{who}: a cache's tensors must be pages x kv_heads x page_size x bytes, got {shapes}")
    lead = shapes[0][:3]
    for s, last in zip(shapes, (blocks * each, blocks) * 2):
        if s != (*lead, last):
            raise ValueError(f"mxq.nn.{who}: a cache of head_dim {head_dim} in {fmt} must have codes {(*lead, blocks * each)} "
                             f"and scales {(*lead, blocks)}, got {shapes}")
    if 0 in lead or lead[0] * lead[2] > _MOST or lead[1] > 65535:
        raise ValueError(f"mxq.nn.{who}: a cache must have 1 to {_MOST} slots and 1 to 65535 heads, got {lead}")
    spec = _lib.CacheSpec(code, head_dim, lead[0], lead[2], lead[1])
    for i, s in enumerate(strides):
        if shapes[i][3] > 1 and s[3] != 1:
            raise ValueError(f"mxq.nn.{who}: a cache's rows must have their bytes next to each other, strides are {s}")
        if who == "cache_write" and any(n > 1 and t == 0 for n, t in zip(shapes[i], s)):
            raise ValueError(f"mxq.nn.{who}: a cache to be written must not be expanded, strides are {s}")
        spec.page_stride[i], spec.head_stride[i], spec.row_stride[i] = s[:3]
    return spec


def _parts(cache, who) -> Tuple[torch.Tensor, ...]:
    if not isinstance(cache, PackedCache):
        raise TypeError(f"mxq.nn.{who}: cache must be a PackedCache, got {type(cache).__name__}")
    parts = cache[:4]
    for t in parts:
        if t.dtype != torch.uint8:
            raise TypeError(f"mxq.nn.{who}: a cache's codes and scales must be uint8, got {t.dtype}")
        if t.device != parts[0].device:
            raise ValueError(f"mxq.nn.{who}: a cache's tensors must be on one device, got {[p.device for p in parts]}")
    return parts


def _checked(cache, parts, who):
    return _spec(cache.fmt, cache.head_dim, tuple(tuple(t.shape) for t in parts), tuple(t.stride() for t in parts), who)


def _no_grad(who: str, *tensors) -> None:
    _no_tangent(who, *tensors)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"mxq.nn.{who}: a cache's bytes have no gradient; call it under torch.no_grad()")


def _slots(slots, who):
    if slots.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"mxq.nn.{who}: slots must be int32 or int64, got {slots.dtype}")
    if slots.ndim != 1 or slots.shape[0] > _MOST:
        raise ValueError(f"mxq.nn.{who}: slots must have one axis, got shape {tuple(slots.shape)}")
    return slots.shape[0]


def _columns(t, dev):
    """t on dev, its last axis's elements next to each other."""
    t = _lib.to_device(t, dev)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def cache_write(k: torch.Tensor, v: torch.Tensor, cache: PackedCache, slots: torch.Tensor) -> None:
    """Quantizes k and v (T x kv_heads x head_dim; float32, bfloat16 or float16) into the rows of `slots` (T whole numbers).

    A token whose slot is not in the cache (-1, say) is left out; where several have one slot the last one's row stays.  A
    block with an infinity or a NaN reads back as NaN."""
    who = "cache_write"
    parts = _parts(cache, who)
    spec = _checked(cache, parts, who)
    T = _slots(slots, who)
    shape = (T, parts[0].shape[1], cache.head_dim)
    for what, t in (("k", k), ("v", v)):
        _dtype(t, who, what)
        if tuple(t.shape) != shape:
            raise ValueError(f"mxq.nn.cache_write: {what} must have shape {shape}, got {tuple(t.shape)}")
    if k.dtype != v.dtype:
        raise TypeError(f"mxq.nn.cache_write: k and v must have one dtype, got {k.dtype} and {v.dtype}")
    _no_grad(who, k, v)
    dev = _lib.compute_device(parts[0], k)
    if parts[0].device != dev:                                   # a cache in host memory: written on the GPU, copied back
        there = PackedCache(*(t.to(dev).contiguous() for t in parts), cache.fmt, cache.head_dim)
        cache_write(k, v, there, slots)
        for t, new in zip(parts, there):
            t.copy_(new)
        return
    kd, vd = _columns(k, dev), _columns(v, dev)
    sd = _lib.to_device(slots, dev).contiguous()
    with _lib.on(dev):
        _lib.run("mxq_cache_write", kd.data_ptr(), vd.data_ptr(), _lib.DTYPE_CODE[k.dtype], T, kd.stride(0), kd.stride(1),
                 vd.stride(0), vd.stride(1), sd.data_ptr(), int(sd.dtype == torch.int64), *(t.data_ptr() for t in parts),
                 spec, _lib.stream(dev))


def cache_read(cache: PackedCache, slots: torch.Tensor,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v), T x kv_heads x head_dim each, of the rows of `slots`: code times scale, rounded once to dtype (float32,
    bfloat16 or float16); zeros for a slot that is not in the cache."""
    who = "cache_read"
    parts = _parts(cache, who)
    spec = _checked(cache, parts, who)
    T = _slots(slots, who)
    code = _lib.DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError(f"mxq.nn.cache_read: dtype must be float32, bfloat16 or float16, got {dtype}")
    dev = _lib.compute_device(parts[0], slots)
    if parts[0].device != dev:
        parts = tuple(t.to(dev).contiguous() for t in parts)
        spec = _checked(cache, parts, who)
    sd = _lib.to_device(slots, dev).contiguous()
    k = torch.empty((T, parts[0].shape[1], cache.head_dim), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    with _lib.on(dev):
        _lib.run("mxq_cache_read", *(t.data_ptr() for t in parts), spec, sd.data_ptr(), int(sd.dtype == torch.int64), T,
                 k.data_ptr(), v.data_ptr(), code, _lib.stream(dev))
    return _lib.back(k, cache.k_codes), _lib.back(v, cache.k_codes)


def _indices(t, who, what, shape):
    if t.dtype != torch.int32:
        raise TypeError(f"mxq.nn.{who}: {what} must be int32, got {t.dtype}")
    if len(t.shape) != len(shape) or any(n is not None and m != n for m, n in zip(t.shape, shape)):
        raise ValueError(f"mxq.nn.{who}: {what} must have shape {shape}, got {tuple(t.shape)}")


def cache_attend(q: torch.Tensor, cache: PackedCache, table: torch.Tensor, lengths: torch.Tensor,
                 starts: Optional[torch.Tensor] = None, *, scale: Optional[float] = None, causal: bool = True,
                 window: Optional[int] = None, return_lse: bool = False):
    """softmax(scale q k^T) v over the cache: a tensor like q, and with return_lse the float32 logarithm of each query's sum
    of exp(scale q k^T), q's shape without its last axis.

    q: B x n x heads x head_dim, or with starts (B + 1 ascending int32) T x heads x head_dim, sequence b's queries being
    [starts[b], starts[b + 1]); float32, bfloat16 or float16.  heads is a multiple of the cache's; neighbouring heads share
    one.  table (B x pages, int32) names each sequence's pages and lengths (B, int32) says how many keys it has, its newest
    tokens', written before, among them.  The last query is at the last key; query j of n is at position
    p = lengths[b] - n + j.  causal: it sees keys up to p; window: from p - window + 1 on.  scale (head_dim ** -0.5 by default)
    must be positive.

    Lengths are held to the table's pages and starts to T.  A key on a page that the cache does not have (-1, say) is not
    there.  A query that sees no key, or that belongs to no sequence, gets zeros and an lse of -inf; so does one whose every
    score is -inf.  Sums are float32, and the weights exp(scale q k^T - max) of bfloat16 queries are rounded to bfloat16."""
    who = "cache_attend"
    parts = _parts(cache, who)
    spec = _checked(cache, parts, who)
    _dtype(q, who, "q")
    _no_grad(who, q)
    G, D = parts[0].shape[1], cache.head_dim
    if q.ndim != (4 if starts is None else 3):
        raise ValueError(f"mxq.nn.cache_attend: q must be B x n x heads x head_dim, or T x heads x head_dim with starts, got "
                         f"shape {tuple(q.shape)}")
    H = q.shape[-2]
    if q.shape[-1] != D or H % G or not H:
        raise ValueError(f"mxq.nn.cache_attend: q must have a multiple of {G} heads of {D} columns, got shape {tuple(q.shape)}")
    _indices(table, who, "table", (None, None))
    B = table.shape[0]
    _indices(lengths, who, "lengths", (B,))
    if starts is not None:
        _indices(starts, who, "starts", (B + 1,))
    elif q.shape[0] != B:
        raise ValueError(f"mxq.nn.cache_attend: q must have {B} sequences, as table has, got shape {tuple(q.shape)}")
    if window is not None:
        _whole(window, who, "window", 1, _MOST)
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"mxq.nn.cache_attend: scale must be positive and finite, got {scale}")
    T = q.shape[0] if starts is not None else q.shape[0] * q.shape[1]
    if T * H > _MOST // 2:
        raise ValueError(f"mxq.nn.cache_attend: {T} queries of {H} heads are too many")
    dev = _lib.compute_device(parts[0], q)
    if parts[0].device != dev:
        parts = tuple(t.to(dev).contiguous() for t in parts)
        spec = _checked(cache, parts, who)
    qd = _columns(q if q.ndim == 3 else q.reshape(T, H, D), dev)
    td, ld = _lib.to_device(table, dev), _lib.to_device(lengths, dev).contiguous()
    if td.stride(1) != 1 and td.shape[1] > 1:
        td = td.contiguous()
    sd = None if starts is None else _lib.to_device(starts, dev).contiguous()
    out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    att = _lib.AttendSpec(_lib.DTYPE_CODE[q.dtype], int(bool(causal)), scale, T, B, H, qd.stride(0), qd.stride(1),
                          td.shape[1], td.stride(0), 0 if window is None else window)
    with _lib.on(dev):
        size = _lib.call("mxq_cache_attend_workspace", spec, att, int(sd is not None))
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _lib.run("mxq_cache_attend", qd.data_ptr(), *(t.data_ptr() for t in parts), spec, td.data_ptr(), ld.data_ptr(),
                 _lib.ptr(sd), out.data_ptr(), _lib.ptr(lse), att, _lib.ptr(work), _lib.stream(dev))
    if q.ndim == 4:
        out = out.reshape(q.shape)
        lse = None if lse is None else lse.reshape(q.shape[:-1])
    out = _lib.back(out, q)
    return (out, _lib.back(lse, q)) if return_lse else out
