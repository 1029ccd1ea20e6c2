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
import functools
from typing import NamedTuple, Optional, Tuple, Union

import torch

from .. import _lib
from ..element_quant.formats import Format, get
from ._moe import _no_tangent, _whole
from ._packed_linear import BLOCK

__all__ = ["PackedCache", "packed_cache", "cache_write", "cache_read", "cache_attend"]

_FORMATS = {"MXFP8_E4M3": (0, 32), "MXFP8_E5M2": (1, 32), "MXFP4": (5, 16)}      # MXQ_FMT_* and a block's bytes
MAX_HEAD_DIM = 256
_MOST = 2 ** 31 - 1
_MOST_KEYS = 2 ** 31 - 2 ** 16


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


def _remembered(make):
    """make, remembered per its arguments: shapes, strides, types and numbers, all plain values.  What a call's checks and
    its spec depend on costs it one lookup; errors are raised as make raises them."""
    return functools.lru_cache(maxsize=512, typed=True)(make)


def _spec(key, who):
    """The spec of a cache with these (fmt, head_dim, shapes, strides, types), checked."""
    fmt, head_dim, shapes, strides, dtypes = key
    for t in dtypes:
        if t != torch.uint8:
            raise TypeError(f"mxq.nn.{who}: a cache's codes and scales must be uint8, got {t}")
    code, each = _format(fmt, who)
    _whole(head_dim, who, "the cache's head_dim", 1, MAX_HEAD_DIM)
    blocks = -(-head_dim // BLOCK)
    shapes = tuple(map(tuple, shapes))
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


def _key(cache, who):
    """What _spec takes of a cache."""
    if not isinstance(cache, PackedCache):
        raise TypeError(f"mxq.nn.{who}: cache must be a PackedCache, got {type(cache).__name__}")
    a, b, c, d, fmt, head_dim = cache
    return (fmt, head_dim, (a.shape, b.shape, c.shape, d.shape), (a.stride(), b.stride(), c.stride(), d.stride()),
            (a.dtype, b.dtype, c.dtype, d.dtype))


def _device(cache, who, *others):
    """The GPU that a call on this cache runs on."""
    dev = cache.k_codes.device
    if cache.k_scales.device != dev or cache.v_codes.device != dev or cache.v_scales.device != dev:
        raise ValueError(f"mxq.nn.{who}: a cache's tensors must be on one device, got {[t.device for t in cache[:4]]}")
    return dev if dev.type == "cuda" else _lib.compute_device(*others)


def _there(cache, dev):
    """A copy of a cache in host memory on dev, its rows next to each other."""
    return PackedCache(*(t.to(dev).contiguous() for t in cache[:4]), cache.fmt, cache.head_dim)


def _no_grad(who: str, *tensors) -> None:
    _no_tangent(who, *tensors)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"mxq.nn.{who}: a cache's bytes have no gradient; call it under torch.no_grad()")


def _check_slots(shape, dtype, who):
    if dtype not in (torch.int32, torch.int64):
        raise TypeError(f"mxq.nn.{who}: slots must be int32 or int64, got {dtype}")
    if len(shape) != 1 or shape[0] > _MOST:
        raise ValueError(f"mxq.nn.{who}: slots must have one axis, got shape {tuple(shape)}")


def _columns(t, dev):
    """t on dev, its last axis's elements next to each other."""
    t = _lib.to_device(t, dev)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


@_remembered
def _write_spec(key, k_shape, k_dtype, v_shape, v_dtype, slots_shape, slots_dtype):
    who = "cache_write"
    spec = _spec(key, who)
    _check_slots(slots_shape, slots_dtype, who)
    shape = (slots_shape[0], spec.kv_heads, spec.head_dim)
    for what, s, dtype in (("k", k_shape, k_dtype), ("v", v_shape, v_dtype)):
        if dtype not in _lib.DTYPE_CODE:
            raise TypeError(f"mxq.nn.cache_write: {what} must be float32, bfloat16 or float16, got {dtype}")
        if tuple(s) != shape:
            raise ValueError(f"mxq.nn.cache_write: {what} must have shape {shape}, got {tuple(s)}")
    if k_dtype != v_dtype:
        raise TypeError(f"mxq.nn.cache_write: k and v must have one dtype, got {k_dtype} and {v_dtype}")
    return spec, _lib.DTYPE_CODE[k_dtype]


def cache_write(k: torch.Tensor, v: torch.Tensor, cache: PackedCache, slots: torch.Tensor) -> None:
    """Quantizes k and v (T x kv_heads x head_dim; float32, bfloat16 or float16) into the rows of `slots` (T whole numbers).

    A token whose slot is not in the cache (-1, say) is left out; where several have one slot the last one's row stays.  A
    block with an infinity or a NaN reads back as NaN."""
    who = "cache_write"
    spec, code = _write_spec(_key(cache, who), k.shape, k.dtype, v.shape, v.dtype, slots.shape, slots.dtype)
    _no_grad(who, k, v)
    dev = _device(cache, who, k)
    if cache.k_codes.device != dev:                             # a cache in host memory: written on the GPU, copied back
        there = _there(cache, dev)
        cache_write(k, v, there, slots)
        for t, new in zip(cache[:4], there):
            t.copy_(new)
        return
    kd, vd = _columns(k, dev), _columns(v, dev)
    sd = _lib.to_device(slots, dev).contiguous()
    kt, kh, _ = kd.stride()
    vt, vh, _ = vd.stride()
    with _lib.on(dev):
        _lib.run("mxq_cache_write", kd.data_ptr(), vd.data_ptr(), code, sd.shape[0], kt, kh, vt, vh, sd.data_ptr(),
                 sd.dtype == torch.int64, cache.k_codes.data_ptr(), cache.k_scales.data_ptr(), cache.v_codes.data_ptr(),
                 cache.v_scales.data_ptr(), spec, _lib.stream(dev))


@_remembered
def _read_spec(key, slots_shape, slots_dtype, dtype):
    spec = _spec(key, "cache_read")
    _check_slots(slots_shape, slots_dtype, "cache_read")
    if dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"mxq.nn.cache_read: dtype must be float32, bfloat16 or float16, got {dtype}")
    return spec, (slots_shape[0], spec.kv_heads, spec.head_dim), _lib.DTYPE_CODE[dtype]


def cache_read(cache: PackedCache, slots: torch.Tensor,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v), T x kv_heads x head_dim each, of the rows of `slots`: code times scale, rounded once to dtype (float32,
    bfloat16 or float16); zeros for a slot that is not in the cache."""
    who = "cache_read"
    spec, shape, code = _read_spec(_key(cache, who), slots.shape, slots.dtype, dtype)
    dev = _device(cache, who, slots)
    if cache.k_codes.device != dev:
        k, v = cache_read(_there(cache, dev), slots, dtype)
        return _lib.back(k, cache.k_codes), _lib.back(v, cache.k_codes)
    sd = _lib.to_device(slots, dev).contiguous()
    k, v = torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)
    with _lib.on(dev):
        _lib.run("mxq_cache_read", cache.k_codes.data_ptr(), cache.k_scales.data_ptr(), cache.v_codes.data_ptr(),
                 cache.v_scales.data_ptr(), spec, sd.data_ptr(), sd.dtype == torch.int64, shape[0], k.data_ptr(),
                 v.data_ptr(), code, _lib.stream(dev))
    return k, v


def _check_indices(t, who, what, shape):
    if t[1] != torch.int32:
        raise TypeError(f"mxq.nn.{who}: {what} must be int32, got {t[1]}")
    if len(t[0]) != len(shape) or any(n is not None and m != n for m, n in zip(t[0], shape)):
        raise ValueError(f"mxq.nn.{who}: {what} must have shape {shape}, got {tuple(t[0])}")


@_remembered
def _attend_spec(key, q_shape, q_dtype, q_strides, table, table_row, lengths, starts, scale, causal, window):
    """(cache spec, attention spec, bytes of workspace); table, lengths and starts as (shape, dtype)."""
    who = "cache_attend"
    spec = _spec(key, who)
    code = _lib.DTYPE_CODE.get(q_dtype)
    if code is None:
        raise TypeError(f"mxq.nn.cache_attend: q must be float32, bfloat16 or float16, got {q_dtype}")
    G, D = spec.kv_heads, spec.head_dim
    if len(q_shape) != (4 if starts is None else 3):
        raise ValueError(f"mxq.nn.cache_attend: q must be B x n x heads x head_dim, or T x heads x head_dim with starts, got "
                         f"shape {tuple(q_shape)}")
    H = q_shape[-2]
    if q_shape[-1] != D or H % G or not H:
        raise ValueError(f"mxq.nn.cache_attend: q must have a multiple of {G} heads of {D} columns, got shape {tuple(q_shape)}")
    _check_indices(table, who, "table", (None, None))
    B, pages = table[0]
    _check_indices(lengths, who, "lengths", (B,))
    if starts is not None:
        _check_indices(starts, who, "starts", (B + 1,))
    elif q_shape[0] != B:
        raise ValueError(f"mxq.nn.cache_attend: q must have {B} sequences, as table has, got shape {tuple(q_shape)}")
    if window is not None:
        _whole(window, who, "window", 1, _MOST)
    scale = D ** -0.5 if scale is None else scale
    if not 0.0 < _lib.c_f32(scale).value <= 2.0 ** 127:                        # as the kernels take it
        raise ValueError(f"mxq.nn.cache_attend: scale must be positive, and 2^127 at most, got {scale}")
    if pages * spec.page_size > _MOST_KEYS:
        raise ValueError(f"mxq.nn.cache_attend: {pages} pages of {spec.page_size} keys a sequence are more than {_MOST_KEYS}")
    T = q_shape[0] if starts is not None else q_shape[0] * q_shape[1]
    if T * H > _MOST // 2:
        raise ValueError(f"mxq.nn.cache_attend: {T} queries of {H} heads are too many")
    att = _lib.AttendSpec(code, causal, scale, T, B, H, *q_strides, pages, table_row, 0 if window is None else window)
    return spec, att, _lib.call("mxq_cache_attend_workspace", spec, att, int(starts is not None))


def cache_attend(q: torch.Tensor, cache: PackedCache, table: torch.Tensor, lengths: torch.Tensor,
                 starts: Optional[torch.Tensor] = None, *, scale: Optional[float] = None, causal: bool = True,
                 window: Optional[int] = None, return_lse: bool = False):
    """softmax(scale q k^T) v over the cache: a tensor like q, and with return_lse the float32 logarithm of each query's sum
    of exp(scale q k^T), q's shape without its last axis.

    q: B x n x heads x head_dim, or with starts (B + 1 ascending int32) T x heads x head_dim, sequence b's queries being
    [starts[b], starts[b + 1]); float32, bfloat16 or float16.  heads is a multiple of the cache's; neighbouring heads share
    one.  table (B x pages, at most 2^31 - 2^16 keys; int32) names each sequence's pages and lengths (B, int32) says how many
    keys it has, its newest tokens', written before, among them.  The last query is at the last key; query j of n is at position
    p = lengths[b] - n + j.  causal: it sees keys up to p; window: from p - window + 1 on.  scale (head_dim ** -0.5 by default)
    must be positive as a float32, and 2^127 at most.

    Lengths are held to the table's pages and starts to T.  A key on a page that the cache does not have (-1, say) is not
    there.  A query that sees no key, or that belongs to no sequence, gets zeros and an lse of -inf; so does one whose every
    score is -inf.  A query that sees a value that is no finite number gets no finite number in its column.  Keys and values
    below 2^-126 are rounded to bfloat16's subnormals, those of 2^128 and more are infinite.  Sums are float32; the weights
    exp(scale q k^T - max) are held to 2^-16, float32 queries' whole, but those of bfloat16 queries are rounded to bfloat16 in a
    sequence of more than 64 rows (its queries times the heads that share one of keys)."""
    who = "cache_attend"
    strides = q.stride()
    dense = q.ndim < 3 or strides[-1] == 1 or q.shape[-1] < 2
    if q.ndim == 4 and q.shape[0] > 1 and q.shape[1] > 1:                      # a token's stride is one number
        dense = dense and strides[0] == strides[1] * q.shape[1]
    if dense:
        strides = (strides[0], strides[2]) if q.ndim == 4 and q.shape[1] == 1 else strides[-3:-1]
    else:
        strides = (q.shape[-2] * q.shape[-1], q.shape[-1])
    rows = table.ndim != 2 or table.shape[1] < 2 or table.stride(1) == 1       # a row's pages lie next to each other
    spec, att, size = _attend_spec(
        _key(cache, who), q.shape, q.dtype, strides, (table.shape, table.dtype),
        0 if table.ndim != 2 else table.stride(0) if rows else table.shape[1], (lengths.shape, lengths.dtype),
        None if starts is None else (starts.shape, starts.dtype), None if scale is None else float(scale), bool(causal), window)
    _no_grad(who, q)
    dev = _device(cache, who, q)
    if cache.k_codes.device != dev:                             # a cache in host memory
        return cache_attend(q, _there(cache, dev), table, lengths, starts, scale=scale, causal=causal, window=window,
                            return_lse=return_lse)
    if q.device != dev or table.device != dev:                  # a view's copy has strides of its own: the spec is of the copy
        got = cache_attend(_lib.to_device(q, dev), cache, _lib.to_device(table, dev), lengths, starts, scale=scale,
                           causal=causal, window=window, return_lse=return_lse)
        return tuple(_lib.back(t, q) for t in got) if return_lse else _lib.back(got, q)
    qd, td = q if dense else q.contiguous(), table if rows else table.contiguous()
    ld = _lib.to_device(lengths, dev).contiguous()
    sd = None if starts is None else _lib.to_device(starts, dev).contiguous()
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev) if return_lse else None
    with _lib.on(dev):
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _lib.run("mxq_cache_attend", qd.data_ptr(), cache.k_codes.data_ptr(), cache.k_scales.data_ptr(),
                 cache.v_codes.data_ptr(), cache.v_scales.data_ptr(), spec, td.data_ptr(), ld.data_ptr(), _lib.ptr(sd),
                 out.data_ptr(), _lib.ptr(lse), att, _lib.ptr(work), _lib.stream(dev))
    return (out, lse) if return_lse else out
