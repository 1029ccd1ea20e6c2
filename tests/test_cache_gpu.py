"""A key and value cache in MX formats: rows written (against packed.quantize's bytes), read back (against 64 bits, exactly)
and attended over (against 64 bits, within oracle.cache's bound), at the sizes and masks where each can go wrong."""
import math

import numpy as np
import pytest
import torch

from mxq import _lib, nn, packed
from oracle import cache as oc

pytestmark = pytest.mark.gpu
FORMATS = ("MXFP8_E4M3", "MXFP8_E5M2", "MXFP4")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _filled(gen, pages, page, heads, dim, fmt, low=118, high=130):
    """A cache of random finite codes and scales, its last blocks filled up with zeros."""
    cache = nn.packed_cache(pages, page, heads, dim, fmt)
    top = {"MXFP8_E4M3": 0x7F, "MXFP8_E5M2": 0x7C, "MXFP4": 0x8}[fmt]
    sign = {"MXFP8_E4M3": 0x80, "MXFP8_E5M2": 0x80, "MXFP4": 0x8}[fmt]
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        width = scales.shape[-1] * 32
        c = torch.randint(0, top, (*codes.shape[:3], width), generator=gen, device="cuda")
        c |= sign * torch.randint(0, 2, c.shape, generator=gen, device="cuda")
        if fmt == "MXFP8_E5M2":
            c -= (c & 0x60 == 0x60) * 0x40                        # exponents of 2^-7 to 2^8
            scales.copy_(torch.randint(low - 6, high - 6, scales.shape, generator=gen, device="cuda"))
        else:
            scales.copy_(torch.randint(low, high, scales.shape, generator=gen, device="cuda") - (6 if fmt == "MXFP8_E4M3" else 0))
        c[..., dim:] = 0
        c = c.to(torch.uint8)
        codes.copy_(c if fmt != "MXFP4" else c[..., 0::2] | c[..., 1::2] << 4)
    return cache


def _table(gen, lengths, page, pages, width=None):
    """Pages of each sequence, drawn without order; -1 past its length."""
    need = [-(-max(l, 0) // page) for l in lengths]
    table = torch.full((len(lengths), max(max(need), width or 1)), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    assert sum(need) <= pages
    first = 0
    for b, k in enumerate(need):
        table[b, :k] = order[first:first + k]
        first += k
    return table


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _check(got, want, bound, what=""):
    assert got.shape == want.shape, what
    none = torch.isinf(want) & (got == want)
    off = torch.where(none, 0.0, (got.double() - want).abs()) - bound
    assert not torch.isnan(off).any(), what
    assert not (off > 0).any(), (what, float(off.max()), float((off / bound.clamp_min(1e-300)).max()))


def _attend(q, cache, table, lengths, starts=None, **more):
    out, lse = nn.cache_attend(q, cache, table, lengths, starts, return_lse=True, **more)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    want, want_lse, bound, lse_bound = oc.attend(q, cache, table, lengths, starts, **more)
    _check(out, want, bound, "out")
    _check(lse, want_lse, lse_bound, "lse")
    return out, lse


def _case(seed, lengths, n, heads, kv_heads, dim, page, fmt, dtype, ragged=False, size=1.0, **more):
    gen = _gen(seed)
    pages = sum(-(-max(l, 0) // page) for l in lengths) + 2
    cache = _filled(gen, pages, page, kv_heads, dim, fmt)
    table = _table(gen, lengths, page, pages)
    if ragged:
        q = torch.randn(sum(n), heads, dim, generator=gen, device="cuda")
        starts = _i32([0] + list(np.cumsum(n)))
    else:
        q, starts = torch.randn(len(lengths), n, heads, dim, generator=gen, device="cuda"), None
    return _attend((q * size).to(dtype), cache, table, _i32(lengths), starts, **more)


# ------------------------------------------------------------------------------------------ rows written and read

def _pairs(codes, fmt):
    return codes if fmt != "MXFP4" else codes[..., 0::2] | codes[..., 1::2] << 4


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim, page, heads", [(128, 16, 8), (64, 1, 1), (80, 7, 3), (1, 5, 2), (33, 64, 5), (256, 3, 2), (100, 48, 1)])
def test_write_is_packed_quantize(cuda, dim, page, heads, dtype, fmt):
    """The bytes of mxq.packed.quantize(x, fmt, "ocp", axis=-1), with the last block filled up with zeros; rows of no slot
    as they were; and the values read back in every type."""
    gen, pages, T = _gen(dim), 11, 37
    cache = nn.packed_cache(pages, page, heads, dim, fmt)
    for t in cache[:4]:
        t.fill_(0xA5)
    x = [(torch.randn(T, heads, dim, generator=gen, device="cuda") * torch.exp(3 * torch.randn(T, heads, 1, generator=gen, device="cuda")))
         .to(DTYPES[dtype]) for _ in range(2)]
    x[0][3], x[1][5] = 0, -0.0
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:T]
    T = len(slots)
    x = [t[:T] for t in x]
    slots[::9] = -1
    slots = slots.int()
    nn.cache_write(*x, cache, slots)
    written = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    written[slots[slots >= 0].long()] = True
    written = written.view(pages, page)
    filled = torch.nn.functional.pad
    for t, codes, scales in ((x[0], cache.k_codes, cache.k_scales), (x[1], cache.v_codes, cache.v_scales)):
        width = scales.shape[-1] * 32
        want_codes, want_scales = packed.quantize(filled(t, (0, width - dim)), fmt, "ocp", axis=-1)
        kept = slots >= 0
        page_of, at = slots[kept].long() // page, slots[kept].long() % page
        assert torch.equal(codes[page_of, :, at], _pairs(want_codes, fmt)[kept])
        assert torch.equal(scales[page_of, :, at], want_scales[kept])
        assert (codes.transpose(1, 2)[~written] == 0xA5).all() and (scales.transpose(1, 2)[~written] == 0xA5).all()
    for out in DTYPES.values():
        k, v = nn.cache_read(cache, slots, out)
        for got, want in zip((k, v), oc.rows(cache, slots)):
            assert got.dtype == out and torch.equal(got, want.to(out))


def test_write_borders(cuda):
    """Maxima next to powers of two, subnormal blocks, the largest float32, ties and saturation, against packed.quantize."""
    for fmt in FORMATS:
        base = torch.tensor([2.0 ** e * f for e in (-126, -20, 0, 1, 100, 127) for f in
                             (1.0, 1 - 2.0 ** -24, 1 - 2.0 ** -23, 1 - 2.0 ** -20, 1 + 2.0 ** -23, 1.75, 1.8125, 1.84375, 1.875, 1.9999)] +
                            [2.0 ** -149, 2.0 ** -140, 2.0 ** -127, 3 * 2.0 ** -128, 3.4028234663852886e38, 0.0], device="cuda")
        ratios = torch.tensor([(-1) ** i * r for i, r in enumerate(
            (1, .5, .75, .625, .5625, .53125, .25, .1875, .15625, 2.0 ** -7, 2.0 ** -9, 3 * 2.0 ** -11, 2.0 ** -14, 2.0 ** -17, 0, 2.0 ** -30))], device="cuda")
        x = (base[:, None] * torch.cat([ratios, ratios.flip(0) * 0.999])[None])[:, None]
        cache = nn.packed_cache(len(x), 1, 1, 32, fmt)
        nn.cache_write(x, -x, cache, torch.arange(len(x), device="cuda"))
        for t, codes, scales in ((x, cache.k_codes, cache.k_scales), (-x, cache.v_codes, cache.v_scales)):
            want_codes, want_scales = packed.quantize(t, fmt, "ocp", axis=-1)
            assert torch.equal(scales[:, 0, 0], want_scales[:, 0]), fmt
            assert torch.equal(codes[:, 0, 0], _pairs(want_codes, fmt)[:, 0]), fmt


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_specials(cuda, fmt):
    """A block with an infinity or a NaN is NaN, its neighbours are not."""
    for dtype in DTYPES.values():
        x = torch.ones(4, 1, 96, dtype=dtype, device="cuda")
        x[0, 0, 40], x[1, 0, 0], x[2, 0, 95] = math.inf, math.nan, -math.inf
        cache = nn.packed_cache(1, 4, 1, 96, fmt)
        nn.cache_write(x, x, cache, torch.arange(4, device="cuda"))
        for got in nn.cache_read(cache, torch.arange(4, device="cuda"), dtype):
            none = torch.isnan(got[:, 0].view(4, 3, 32))
            want = torch.zeros(4, 3, 1, dtype=torch.bool, device="cuda")
            want[0, 1] = want[1, 0] = want[2, 2] = True
            assert torch.equal(none, want.expand(4, 3, 32)) and (got[~torch.isnan(got)] == 1).all()


@pytest.mark.parametrize("T", [2, 40, 1000, 3000, 20000, 33000, 70000])
def test_write_same_slot_again(cuda, T):
    """The last token's row stays, of keys and of values, wherever the others are."""
    gen = _gen(T)
    pages, page = 40, 16
    cache = nn.packed_cache(pages, page, 2, 32, "MXFP8_E4M3")
    slots = torch.randint(-1, pages * page + 2, (T,), generator=gen, device="cuda")
    x = torch.randint(1, 9, (T, 2, 32), generator=gen, device="cuda").float()
    nn.cache_write(x, -x, cache, slots)
    last = torch.full((pages * page,), -1, dtype=torch.int64)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            last[s] = t
    written = (last >= 0).nonzero()[:, 0].cuda()
    k, v = nn.cache_read(cache, written, torch.float32)
    want = x[last.cuda()[written]]
    assert torch.equal(k, want) and torch.equal(v, -want)


@pytest.mark.parametrize("T", [1, 1023, 1024, 1025, 1500])
@pytest.mark.parametrize("fmt, dtype, dim, heads, page", [("MXFP8_E4M3", "bf16", 256, 40, 3), ("MXFP4", "f16", 40, 3, 16), ("MXFP8_E5M2", "f32", 100, 33, 7)])
def test_write_and_read_few_and_many_tokens(cuda, fmt, dtype, dim, heads, page, T):
    """One token a workgroup and several, rows of more items than a workgroup has threads, tokens and heads apart."""
    gen = _gen(T + dim)
    pages = -(-T // page) + 2
    cache = nn.packed_cache(pages, page, heads, dim, fmt)
    for t in cache[:4]:
        t.fill_(0x5A)
    wide = torch.randn(T, 2 * heads, dim + 3, generator=gen, device="cuda").to(DTYPES[dtype])
    x = (wide[:, 1::2, 3:], wide[:, ::2, :dim])
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:T]
    slots[1::11] = pages * page
    nn.cache_write(*x, cache, slots)
    kept = slots < pages * page
    page_of, at = slots[kept] // page, slots[kept] % page
    free = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    free[page_of, at] = False
    for t, codes, scales in ((x[0], cache.k_codes, cache.k_scales), (x[1], cache.v_codes, cache.v_scales)):
        want_codes, want_scales = packed.quantize(torch.nn.functional.pad(t, (0, scales.shape[-1] * 32 - dim)), fmt, "ocp", axis=-1)
        assert torch.equal(codes[page_of, :, at], _pairs(want_codes, fmt)[kept])
        assert torch.equal(scales[page_of, :, at], want_scales[kept])
        assert (codes.transpose(1, 2)[free] == 0x5A).all() and (scales.transpose(1, 2)[free] == 0x5A).all()
    for out in DTYPES.values():
        for got, want in zip(nn.cache_read(cache, slots.int(), out), oc.rows(cache, slots)):
            assert torch.equal(got, want.to(out))


@pytest.mark.parametrize("fmt", FORMATS)
def test_read_every_code_and_scale(cuda, fmt):
    """Each code under each scale byte, rounded once: subnormal, overflowing and NaN ones too."""
    codes = torch.arange(16 if fmt == "MXFP4" else 256, device="cuda").repeat_interleave(2 if fmt == "MXFP4" else 1)
    dim = 32 if fmt == "MXFP4" else 256
    cache = nn.packed_cache(256, 1, 1, dim, fmt)
    bytes_ = codes.to(torch.uint8)
    cache.k_codes.copy_(bytes_[0::2] | bytes_[1::2] << 4 if fmt == "MXFP4" else bytes_)
    cache.v_codes.copy_(cache.k_codes.flip(-1))
    for scales in (cache.k_scales, cache.v_scales):
        scales.copy_(torch.arange(256, device="cuda").to(torch.uint8)[:, None, None, None])
    slots = torch.arange(256, device="cuda")
    for T in (256, 2560):
        for out in DTYPES.values():
            for got, want in zip(nn.cache_read(cache, slots.repeat(T // 256), out), oc.rows(cache, slots)):
                want = want.to(out).repeat(T // 256, 1, 1)
                assert torch.equal(got.nan_to_num(nan=12345.0, posinf=math.inf, neginf=-math.inf),
                                   want.nan_to_num(nan=12345.0, posinf=math.inf, neginf=-math.inf)), out


def test_read_more_rows_than_a_launch(cuda):
    """2^27 rows of one column and some more: several launches of as many threads as one may have."""
    gen = _gen(5)
    cache = _filled(gen, 8, 16, 1, 1, "MXFP8_E4M3")
    T = 2 ** 27 + 5
    slots = torch.randint(0, 128, (T,), dtype=torch.int32, device="cuda", generator=gen)
    slots[-1] = 128
    for got, want in zip(nn.cache_read(cache, slots, torch.bfloat16), oc.rows(cache, torch.arange(128, device="cuda"))):
        want = torch.cat([want.bfloat16().flatten(), torch.zeros(1, dtype=torch.bfloat16, device="cuda")])
        assert torch.equal(got.flatten(), want[slots])


def test_slots_of_64_bits_and_none(cuda):
    cache = _filled(_gen(1), 4, 8, 2, 64, "MXFP4")
    before = [t.clone() for t in cache[:4]]
    far = torch.tensor([-1, 32, 2 ** 32, 2 ** 32 + 5, -2 ** 40, 2 ** 62, 31], device="cuda")
    x = torch.ones(7, 2, 64, device="cuda")
    nn.cache_write(x, x, cache, far)
    for t, old in zip(cache[:4], before):
        old[3, :, 7] = t[3, :, 7]
        assert torch.equal(t, old)
    k, v = nn.cache_read(cache, far, torch.float32)
    assert (k[:6] == 0).all() and (v[:6] == 0).all() and (k[6] == 1).all() and (v[6] == 1).all()
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    nn.cache_write(x[:0], x[:0], cache, none)
    assert nn.cache_read(cache, none)[0].shape == (0, 2, 64)


def test_write_strides(cuda):
    """Rows inside a projection's output, columns apart, and a cache whose rows lie token by token inside a larger one."""
    gen = _gen(3)
    T, G, D = 19, 3, 72
    wide = torch.randn(T, G * 3, D + 9, generator=gen, device="cuda").bfloat16()
    k, v = wide[:, :G, 5:5 + D], wide[:, 2 * G:, 1:1 + D]
    whole = nn.packed_cache(6, 8, G, D, "MXFP8_E5M2")
    parts = [torch.full((8, 8, G + 2, t.shape[-1] + 3), 0x11, dtype=torch.uint8, device="cuda") for t in whole[:4]]
    views = [p[1:7, :, 1:1 + G, 2:2 + t.shape[-1]].transpose(1, 2) for p, t in zip(parts, whole)]
    other = nn.PackedCache(*views, "MXFP8_E5M2", D)
    slots = torch.randperm(48, generator=gen, device="cuda")[:T].int()
    nn.cache_write(k, v, whole, slots)
    nn.cache_write(k, v, other, slots)
    nn.cache_write(k.double().transpose(1, 2).contiguous().transpose(1, 2).bfloat16(), v, other, slots)
    for a, b in zip(nn.cache_read(whole, slots), nn.cache_read(other, slots)):
        assert torch.equal(a, b)
    for p, t in zip(parts, whole):
        assert (p[0] == 0x11).all() and (p[7] == 0x11).all() and (p[:, :, 0] == 0x11).all() and (p[:, :, -1] == 0x11).all()
        assert (p[..., :2] == 0x11).all() and (p[..., -1] == 0x11).all()
    q = torch.randn(2, 1, 6, D, generator=gen, device="cuda").bfloat16()
    table, lengths = _i32([[0, 3, 5], [1, 2, 4]]), _i32([17, 24])
    assert torch.equal(nn.cache_attend(q, whole, table, lengths), nn.cache_attend(q, nn.PackedCache(
        *(t.transpose(1, 2).contiguous().transpose(1, 2) for t in whole[:4]), "MXFP8_E5M2", D), table, lengths))


def test_host_tensors(cuda):
    """A cache in host memory is written in place and attended over, as other operands there are taken."""
    gen = _gen(4)
    here = _filled(gen, 5, 4, 2, 40, "MXFP4")
    host = nn.PackedCache(*(t.cpu() for t in here[:4]), "MXFP4", 40)
    x, slots = torch.randn(3, 2, 40, generator=gen, device="cuda"), torch.tensor([2, 19, 7])
    nn.cache_write(x, x, here, slots)
    nn.cache_write(x.cpu(), x, host, slots)
    for a, b in zip(here, host[:4]):
        assert torch.equal(a.cpu(), b)
    assert nn.cache_read(host, slots)[0].device.type == "cpu"
    q = torch.randn(1, 1, 4, 40, generator=gen, device="cuda")
    args = (_i32([[1, 4, 0]]), _i32([11]))
    out = nn.cache_attend(q.cpu(), host, args[0].cpu(), args[1].cpu())
    assert out.device.type == "cpu" and torch.equal(out, nn.cache_attend(q, here, *args).cpu())


@pytest.mark.parametrize("here", [True, False])
def test_host_views(cuda, here):
    """Queries and tables that are views of larger tensors in host memory, with a cache on the GPU and one beside them."""
    gen = _gen(21)
    cache = _filled(gen, 30, 16, 2, 40, "MXFP8_E4M3")
    wide = torch.randn(3, 5, 12, 45, generator=gen, device="cuda").bfloat16()
    tables = torch.randint(0, 30, (6, 40), generator=gen, device="cuda").int()
    lengths = torch.tensor([160, 9, 77, 3, 50, 33], device="cuda").int()[::2]
    starts = torch.tensor([0, 9, 1, 9, 4, 9, 5], device="cuda").int()[::2]
    taken = cache if here else nn.PackedCache(*(t.cpu() for t in cache[:4]), *cache[4:])
    queries = (lambda w: (w[..., 3:7, 5:], None), lambda w: (w[:, 2:3, :4, :40], None), lambda w: (w[..., :1, :40].expand(3, 5, 4, 40), None),
               lambda w: (w[0, :, 4:8, :40], True), lambda w: (w[1, :, ::3, 5:], True), lambda w: (w[:, 0, :1, :40].expand(3, 4, 40), True))
    for cut in queries:
        for part in (lambda t: t[:3, 4:14], lambda t: t[::2, 20:], lambda t: t[:10, :3].t(), lambda t: t[:1, 7:17].expand(3, 10)):
            (q, ragged), table, of = cut(wide), part(tables), None
            host, args = cut(wide.cpu())[0], [taken, part(tables.cpu()), lengths.cpu()]
            if ragged:
                of, args = starts, [*args, starts.cpu()]
            assert table.shape[0] == 3
            want, want_lse = nn.cache_attend(q.contiguous(), cache, table.contiguous(), lengths, of, return_lse=True)
            out, lse = nn.cache_attend(host, *args, return_lse=True)
            assert out.device.type == lse.device.type == "cpu" and torch.equal(out.cuda(), want) and torch.equal(lse.cuda(), want_lse)
            assert torch.equal(nn.cache_attend(q, *args), want)
            assert torch.equal(nn.cache_attend(host, cache, table, lengths, of).cuda(), want)


# ---------------------------------------------------------------------------------------------------- attention

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim", [1, 7, 32, 33, 64, 65, 80, 96, 100, 128, 129, 160, 192, 225, 256])
def test_attend_formats_types_and_columns(cuda, dim, dtype, fmt):
    _case(dim, [45, 0, 1, 300], 1, 8, 2, dim, 16, fmt, DTYPES[dtype])
    _case(dim + 1, [45, 70], 9, 8, 2, dim, 16, fmt, DTYPES[dtype])


@pytest.mark.parametrize("page", [1, 2, 7, 15, 16, 17, 24, 32, 48, 64, 100, 256, 1000])
def test_attend_pages_and_lengths(cuda, page):
    lengths = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500]
    _case(page, lengths, 1, 4, 2, 64, page, "MXFP4", torch.bfloat16)
    _case(page, lengths, 2, 4, 2, 96, page, "MXFP8_E4M3", torch.float16)
    _case(page, lengths[5:12], 37, 4, 2, 96, page, "MXFP4", torch.bfloat16)


@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (5, 5), (6, 3), (28, 4), (16, 1), (17, 1), (40, 1), (128, 1), (48, 3)])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 16, 17, 33, 70])
def test_attend_heads_and_queries(cuda, n, heads, kv_heads):
    for causal in (True, False):
        _case(n, [n, 100, n + 31], n, heads, kv_heads, 64, 16, "MXFP8_E4M3", torch.bfloat16, causal=causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [None, 1, 2, 31, 32, 33, 100, 5000])
def test_attend_windows(cuda, window, causal):
    for n in (1, 7, 50, 200):
        _case(n, [257, 40, n], n, 4, 2, 80, 16, "MXFP4", torch.bfloat16, window=window, causal=causal)
        _case(n, [257, 40, n], n, 2, 2, 128, 24, "MXFP8_E5M2", torch.float32, window=window, causal=causal)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_attend_ragged(cuda, dtype):
    """Sequences of no query, of one and of many, lengths below their queries."""
    n = [1, 0, 17, 130, 0, 3, 64, 1, 40]
    lengths = [5, 9, 17, 200, 0, 1, 30, 0, 300]
    for fmt, dim, page, window in (("MXFP4", 128, 16, None), ("MXFP8_E4M3", 80, 10, 50), ("MXFP8_E5M2", 256, 64, None)):
        _case(dim, lengths, n, 6, 3, dim, page, fmt, DTYPES[dtype], ragged=True, window=window)
    _case(9, lengths, n, 6, 3, 64, 16, "MXFP4", DTYPES[dtype], ragged=True, causal=False)


@pytest.mark.parametrize("lengths", [[20000], [9000, 100, 0, 20001, 3], [4097] * 5, [100] * 70 + [30000]])
def test_attend_long(cuda, lengths):
    """Contexts cut into runs that are joined, short ones beside them."""
    for n, fmt, dim, dtype in ((1, "MXFP4", 128, torch.bfloat16), (2, "MXFP8_E4M3", 64, torch.float32), (1, "MXFP8_E5M2", 256, torch.float16)):
        _case(len(lengths), lengths, n, 4, 1, dim, 64, fmt, dtype)
    if len(lengths) < 10:
        _case(1, lengths, [40, 1, 3, 0, 90][:len(lengths)], 4, 1, 96, 16, "MXFP4", torch.bfloat16, ragged=True)
        _case(1, lengths, [40, 1, 3, 0, 90][:len(lengths)], 4, 1, 96, 16, "MXFP4", torch.bfloat16, ragged=True, window=6000)


def test_attend_many_sequences(cuda):
    lengths = [(37 * i) % 91 for i in range(300)]
    _case(0, lengths, 1, 2, 1, 64, 16, "MXFP4", torch.bfloat16)
    _case(0, lengths, [i % 3 for i in range(300)], 2, 1, 64, 16, "MXFP4", torch.bfloat16, ragged=True)


@pytest.mark.parametrize("fmt, dtype, dim, n, heads", [("MXFP4", "bf16", 130, 260, 128), ("MXFP8_E4M3", "f32", 256, 260, 64)])
@pytest.mark.parametrize("ragged", [False, True])
def test_attend_tiles_enough_to_stay_whole(cuda, fmt, dtype, dim, n, heads, ragged):
    """So many rows that no tile is cut, the last one of a sequence not full."""
    for page in (16, 24):
        _case(n, [n + 40, n - 10, 300], [n, n, n] if ragged else n, heads, 1, dim, page, fmt, DTYPES[dtype], ragged=ragged)


@pytest.mark.parametrize("lengths, n, heads, kv_heads", [
    ([(61 * i) % 997 for i in range(100)], 1, 2, 1),              # more sequences than a wave has lanes
    ([(61 * i) % 997 for i in range(100)], 3, 8, 4),
    ([(61 * i) % 997 for i in range(330)], 1, 2, 2),
    ([(331 * i) % 3700 + 300 for i in range(40)], 1, 16, 8), ([(331 * i) % 3900 for i in range(100)], 2, 8, 4),    # longer, the same
    ([2500], 700, 1, 1), ([1100, 700], 350, 6, 3)])               # prompts: tiles that weigh more and more
def test_attend_pieces(cuda, lengths, n, heads, kv_heads):
    for fmt, dim, page, dtype in (("MXFP4", 64, 16, torch.bfloat16), ("MXFP8_E4M3", 128, 20, torch.float16)):
        _case(len(lengths), lengths, n, heads, kv_heads, dim, page, fmt, dtype)


@pytest.mark.parametrize("lengths", [[300, 900, 40], [31, 2000, 500]])
@pytest.mark.parametrize("fmt, dtype, dim, window", [("MXFP4", "f32", 256, None), ("MXFP8_E4M3", "bf16", 200, 333)])
def test_attend_many_tiles_of_unlike_sequences(cuda, fmt, dtype, dim, window, lengths):
    """Tiles between one and three times the workgroups that take equal pieces of them."""
    for page in (16, 12):
        _case(lengths[1], lengths, [70, 160, 30], 256, 2, dim, page, fmt, DTYPES[dtype], ragged=True, window=window)


def test_attend_tiny_and_large_scale_bytes(cuda):
    """Values of about 2^-100 and 2^110: no sum passes float32, and products below its smallest normal number, taken as
    zeros, would be less than half a step of bfloat16."""
    for n in (1, 60):
        for fmt, low in (("MXFP4", 26), ("MXFP4", 200), ("MXFP8_E4M3", 32), ("MXFP8_E5M2", 32), ("MXFP8_E4M3", 240)):
            gen = _gen(low)
            cache = _filled(gen, 9, 16, 2, 96, fmt, low, low + 3)
            cache.k_scales.copy_(torch.randint(118, 126, cache.k_scales.shape, generator=gen, device="cuda"))
            q = torch.randn(1, n, 4, 96, generator=gen, device="cuda").bfloat16()
            _attend(q, cache, torch.arange(9, dtype=torch.int32, device="cuda")[None], _i32([140]))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt", FORMATS)
def test_attend_values_below_the_smallest_normal(cuda, fmt, dtype):
    """Each value is off by half a step of bfloat16's subnormals at most, 2^-134, and so is their mean by weights; no value is
    taken for zero that is more than that."""
    for n in (1, 100):
        for low in (0, 1, 2, 4, 8):
            gen = _gen(low)
            cache = _filled(gen, 5, 16, 1, 64, fmt)
            cache.v_scales.fill_(low)
            q = torch.randn(1, n, 4, 64, generator=gen, device="cuda").to(DTYPES[dtype])
            args = q, cache, torch.arange(5, device="cuda").int()[None], _i32([77])
            want, _, bound, _ = oc.attend(*args)
            assert dtype == "f16" or (want != 0).any()
            _check(nn.cache_attend(*args), want, bound + 2.0 ** -134, (fmt, low, n))


@pytest.mark.parametrize("B, n", [(64, 3), (65, 3), (70, 20), (256, 1), (257, 1), (600, 2)])
def test_attend_sequences_of_short_contexts(cuda, B, n):
    """Contexts too short to be cut, of as many sequences as are looked through for a tile and of more; ragged ones of one
    query and of many in turn."""
    lengths = [(29 * i) % 100 for i in range(B)]
    _case(B, lengths, n, 8, 2, 64, 16, "MXFP4", torch.bfloat16)
    _case(B, lengths, [1 if i % 5 else 17 * (i % 3) for i in range(B)], 8, 2, 96, 24, "MXFP8_E4M3", torch.float16, ragged=True)


@pytest.mark.parametrize("size", [1e-3, 30.0, 3000.0])
def test_attend_score_sizes(cuda, size):
    """Nearly even weights, and scores so far apart that one key has all the weight."""
    for n in (1, 70):
        _case(n, [400, 33], n, 4, 2, 128, 16, "MXFP8_E4M3", torch.bfloat16, size=size)
        _case(n, [400, 33], n, 4, 2, 64, 16, "MXFP4", torch.float32, size=size, scale=0.3)


@pytest.mark.parametrize("lengths, n, heads, kv_heads", [([40] * 30, 1, 8, 8), ([33, 60, 7], 1, 40, 4), ([50, 45], 5, 24, 2), ([45, 64], 2, 32, 2),
                                                         ([100, 5000], 1, 8, 2)])
@pytest.mark.parametrize("fmt, dim", [("MXFP4", 64), ("MXFP8_E4M3", 128), ("MXFP8_E5M2", 200)])
def test_attend_weights_of_few_bfloat16_rows(cuda, fmt, dim, lengths, n, heads, kv_heads):
    """Tiles of few rows take bfloat16 queries' weights as two bfloat16, too: within the oracle's bound for 2^-16, beside which
    a weight rounded to bfloat16 alone would show, keys being few."""
    gen = _gen(25)
    pages = sum(-(-l // 16) for l in lengths)
    cache, table = _filled(gen, pages, 16, kv_heads, dim, fmt), _table(gen, lengths, 16, pages)
    q = torch.randn(len(lengths), n, heads, dim, generator=gen, device="cuda").bfloat16()
    out, lse = nn.cache_attend(q, cache, table, _i32(lengths), return_lse=True)
    want, want_lse, bound, lse_bound = oc.attend(q, cache, table, _i32(lengths), rounded=2.0 ** -16)
    _check(out, want, bound, "out")
    _check(lse, want_lse, lse_bound, "lse")


@pytest.mark.parametrize("B, n, heads", [(1024, 1, 16), (1, 128, 128)])
def test_attend_float16_weights_are_rounded_to_the_nearest(cuda, B, n, heads):
    """Values of 1 and -1 under weights of 1 and exp(-t), t to 2^-6, are tanh(t / 2), small enough for float16 to show the
    weight's own error: that of a weight's two bfloat16 is 2^-17 at most here (a weight in [1/2, 1) is eight bits and a
    remainder below 2^-8, whose half step is 2^-17 at most), as often up as down, and half of it the output's, beside the output's
    rounding, 2^-19 at most.  The mean of 16384 errors is then within 6 / 128 of 2^-18 + 2^-19, and 4 units of float32 for
    exp2, its argument and the quotient, which may lean one way: below 2^-20 together.  Weights cut off instead lean by
    2/3 2^-17, half of it the output's: 2^-18.6."""
    t = (torch.rand(B, n, heads, generator=_gen(24), device="cuda") * 2.0 ** -6).half()
    q = torch.zeros(B, n, heads, 32, dtype=torch.float16, device="cuda")
    q[..., 0] = t
    cache = nn.packed_cache(1, 2, 1, 32, "MXFP8_E4M3")
    k, v = torch.zeros(2, 1, 32, device="cuda"), torch.ones(2, 1, 32, device="cuda")
    k[1, 0, 0], v[1] = -1, -1
    nn.cache_write(k, v, cache, torch.arange(2, device="cuda"))
    out = nn.cache_attend(q, cache, _i32([[0]]).expand(B, 1), _i32([2]).expand(B), scale=1.0, causal=False)
    assert t.numel() == 16384 and abs(float((out[..., 0].double() - torch.tanh(t.double() / 2)).mean())) <= 2.0 ** -20


def test_attend_rising_scores(cuda):
    """Each key larger than the one before: the maximum moves in every step."""
    gen = _gen(7)
    for n, dtype in ((1, torch.bfloat16), (40, torch.float32)):
        cache = nn.packed_cache(20, 16, 1, 64, "MXFP8_E4M3")
        k = (torch.arange(320, device="cuda")[:, None, None] * torch.ones(64, device="cuda")) / 8
        v = torch.randn(320, 1, 64, generator=gen, device="cuda")
        nn.cache_write(k, v, cache, torch.arange(320, device="cuda"))
        q = torch.rand(1, n, 2, 64, generator=gen, device="cuda").to(dtype)
        table = torch.arange(20, dtype=torch.int32, device="cuda")[None]
        _attend(q, cache, table, _i32([320]))
        _attend(-q, cache, table, _i32([320]))


def test_attend_pages_that_do_not_exist(cuda):
    """-1, the number of pages and far numbers inside a sequence: their keys are not there; all of them: zeros."""
    gen = _gen(8)
    cache = _filled(gen, 12, 16, 2, 64, "MXFP4")
    table = _i32([[3, -1, 5, 12, 7], [-1, -1, -2 ** 31, 2 ** 31 - 1, 13], [1, 2, 4, 6, 8]])
    for n in (1, 3, 66):
        q = torch.randn(3, n, 4, 64, generator=gen, device="cuda").bfloat16()
        out, lse = _attend(q, cache, table, _i32([70, 75, 80]))
        assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
        _attend(q, cache, table, _i32([70, 75, 10 ** 9]))                # held to the table
        _attend(q, cache, table, _i32([-5, -2 ** 31, 20]))
    cache7 = _filled(gen, 12, 7, 2, 64, "MXFP4")
    for n in (1, 66):
        _attend(torch.randn(3, n, 4, 64, generator=gen, device="cuda").bfloat16(), cache7, table, _i32([35, 30, 29]))


def test_attend_rows_of_no_sequence(cuda):
    """Queries before the first sequence, behind the last one: zeros; starts past the queries are held to them."""
    gen = _gen(9)
    cache = _filled(gen, 12, 16, 2, 128, "MXFP4")
    table, lengths = _i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]]), _i32([40, 33, 48])
    q = torch.randn(150, 4, 128, generator=gen, device="cuda").bfloat16()
    for starts in ([2, 3, 3, 20], [0, 1, 2, 3], [5, 5, 5, 5], [10, 110, 111, 150], [0, 20, 10 ** 6, 2 ** 31 - 1], [-7, 4, 150, 200]):
        out, lse = nn.cache_attend(q, cache, table, lengths, _i32(starts), return_lse=True)
        low, high = max(starts[0], 0), min(starts[3], 150)
        assert (out[:low] == 0).all() and (out[high:] == 0).all() and (lse[:low] == -math.inf).all() and (lse[high:] == -math.inf).all()
        _attend(q, cache, table, lengths, _i32([min(max(s, 0), 150) for s in starts]))
        assert not torch.isnan(out).any()
    none = nn.cache_attend(q, cache, table[:0], lengths[:0], _i32([0]))
    assert (none == 0).all()
    assert nn.cache_attend(q[:0], cache, table, lengths, _i32([0, 0, 0, 0])).shape == (0, 4, 128)
    # starts that do not ascend give some answer of what there is
    nn.cache_attend(q, cache, table, lengths, _i32([50, 3, 140, 2]))
    # a table without pages: no keys
    out, lse = nn.cache_attend(q[:3, None], cache, table[:, :0], lengths, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_attend_rows_of_no_sequence_beside_cut_tiles(cuda):
    """The same where sequences are long enough to be cut and joined."""
    gen = _gen(18)
    cache = _filled(gen, 600, 16, 2, 64, "MXFP4")
    lengths = [8000, 30, 500]
    table = _table(gen, lengths, 16, 600)
    q = torch.randn(90, 8, 64, generator=gen, device="cuda").bfloat16()
    for starts in ([3, 20, 31, 32], [0, 70, 71, 85], [5, 5, 6, 89]):
        out, lse = _attend(q, cache, table, _i32(lengths), _i32(starts))
        assert (out[:starts[0]] == 0).all() and (out[starts[3]:] == 0).all()
        assert (lse[:starts[0]] == -math.inf).all() and (lse[starts[3]:] == -math.inf).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n, group", [(1, 1), (6, 2), (70, 2), (150, 4)])
def test_attend_nan_and_infinity_behind_the_mask(cuda, n, group, fmt):
    """What a query does not see does not reach it: keys ahead of it, before its window, past the length, on the rest of a
    page; a NaN that it sees makes it NaN."""
    gen = _gen(10)
    for dtype in DTYPES.values():
        for dim, page in ((64, 16), (128, 24), (200, 32)):
            length = 170
            pages = -(-length // page) + 3
            cache = _filled(gen, pages, page, 1, dim, fmt)
            table = _table(gen, [length], page, pages)
            slots = table[0].long()[torch.arange(length, device="cuda") // page] * page + torch.arange(length, device="cuda") % page
            used = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
            used[slots] = True
            for scales in (cache.k_scales, cache.v_scales):
                free = (~used).nonzero()[:, 0]
                scales[free // page, :, free % page] = 255
            q = torch.randn(1, n, group, dim, generator=gen, device="cuda").to(dtype)
            bad = length - max(n // 2, 1)                      # seen by the second half of the queries alone
            where = (slots[bad] // page, 0, slots[bad] % page)
            for part in (cache.k_scales, cache.v_scales):
                old = part[where].clone()
                part[where] = 255
                args = (q, cache, table, _i32([length]))
                out, lse = nn.cache_attend(*args, return_lse=True)
                sees = torch.arange(length - n, length, device="cuda") >= bad
                part[where] = old
                want, want_lse, bound, lse_bound = oc.attend(*args)
                assert torch.isnan(out[0, sees]).all() if part is cache.k_scales else torch.isnan(out[0, sees]).any(-1).all()
                if n > 1:
                    _check(out[0, ~sees], want[0, ~sees], bound[0, ~sees])
                    _check(lse[0, ~sees], want_lse[0, ~sees], lse_bound[0, ~sees])
                # and before a window
                part[where] = 255
                out = nn.cache_attend(*args, window=2)
                part[where] = old
                want, _, bound, _ = oc.attend(*args, window=2)
                at = torch.arange(length - n, length, device="cuda")
                free = (at < bad) | (at - 2 >= bad)
                _check(out[0, free], want[0, free], bound[0, free])


def test_attend_infinite_values_behind_the_mask(cuda):
    """E5M2's infinities among the values, and scales that make finite codes infinite."""
    gen = _gen(11)
    for n in (5, 100):
        cache = _filled(gen, 10, 16, 1, 64, "MXFP8_E5M2")
        table = torch.arange(10, dtype=torch.int32, device="cuda")[None]
        q = torch.randn(1, n, 4, 64, generator=gen, device="cuda").bfloat16()
        want, _, bound, _ = oc.attend(q, cache, table, _i32([160]))
        cache.v_codes[9, 0, 15, ::3] = 0x7C
        cache.v_scales[9, 0, 14, 1] = 254
        out = nn.cache_attend(q, cache, table, _i32([160]))
        _check(out[0, :n - 2], want[0, :n - 2], bound[0, :n - 2])
        assert (~torch.isfinite(out[0, n - 1])).any(-1).all()


@pytest.mark.parametrize("keys, n, heads, joined", [
    (300, 1, 4, False), (300, 1, 40, False), (300, 70, 4, False),        # tiles that stay whole, of few and of many rows
    (20000, 1, 4, True), (20000, 4, 12, True), (9000, 100, 4, True)])    # cut ones, joined row by row and all at once
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_attend_nan_and_infinity_of_no_weight(cuda, dtype, keys, n, heads, joined):
    """A value that is no finite number, under a score so low that its weight is zero: seen all the same, in whichever wave
    or part of a tile the largest score is.  Other columns are the best key's value exactly, all other weights being zero."""
    gen = _gen(22)
    for fmt, dim, page in (("MXFP8_E5M2", 128, 16), ("MXFP4", 64, 24), ("MXFP8_E4M3", 200, 32)):
        cache = _filled(gen, -(-keys // page), page, 1, dim, fmt)
        table, slots = torch.arange(cache.k_codes.shape[0], device="cuda").int()[None], torch.arange(keys, device="cuda")
        q = torch.zeros(1, n, heads, dim, dtype=DTYPES[dtype], device="cuda")
        q[..., 0] = 1
        for best, bad in ((0, keys - 1), (keys - 1, 0), (40, 41), (keys // 2, 100), (100, keys // 2), (70, 35), (keys // 3, 2 * keys // 3)):
            v = nn.cache_read(cache, slots, torch.float32)[1]
            k = torch.zeros_like(v)
            k[:, 0, 0] = -192
            k[best] = 0
            nn.cache_write(k, v, cache, slots)
            v = nn.cache_read(cache, slots, torch.float32)[1]
            where = (bad // page, 0, bad % page)
            scales, codes = cache.v_scales[where].clone(), cache.v_codes[where].clone()
            cache.v_scales[where + (1,)] = 255
            if fmt == "MXFP8_E5M2":
                cache.v_codes[where + (0,)] = 0x7C
            _lib.timer_enable(True)
            try:
                _lib.timer_read("k_attend_join")
                out, lse = nn.cache_attend(q, cache, table, _i32([keys]), scale=1.0, causal=False, return_lse=True)
                assert (_lib.timer_read("k_attend_join")[1] > 0) == joined
            finally:
                _lib.timer_enable(False)
            cache.v_scales[where], cache.v_codes[where] = scales, codes
            finite = torch.ones(dim, dtype=torch.bool, device="cuda")
            finite[32:64] = False
            finite[0] = fmt != "MXFP8_E5M2"
            assert (~torch.isfinite(out[..., ~finite])).all(), (fmt, best, bad)
            assert (out == v[best, 0].to(q.dtype))[..., finite].all() and (lse == 0).all(), (fmt, best, bad)


@pytest.mark.parametrize("fmt, code, scale", [("MXFP8_E5M2", 0x7C, 120), ("MXFP8_E5M2", 0x7B, 254), ("MXFP8_E4M3", 0x7E, 247), ("MXFP4", 7, 253)])
@pytest.mark.parametrize("n, heads", [(1, 4), (5, 12), (100, 4)])
def test_attend_infinite_keys(cuda, n, heads, fmt, code, scale):
    """Keys that are infinite, by their code or by their scale, under queries of few bits and of a type's most: scores of -inf
    have no weight, nothing but them gives zeros, and a score of +inf or of zero times infinity gives no number."""
    gen = _gen(23)
    sign = 8 if fmt == "MXFP4" else 0x80
    for dtype in DTYPES.values():
        for dim, page, pages in ((64, 16, 6), (128, 24, 4), (200, 16, 320)):
            cache = _filled(gen, pages, page, 1, dim, fmt)
            table, lengths = torch.arange(pages, device="cuda").int()[None], _i32([pages * page - 3])
            q = torch.randn(1, n, heads, dim, generator=gen, device="cuda")
            q[..., 33], q[..., 1] = q[..., 33].abs() + 1, 0
            q[:, :, ::2] = q[:, :, ::2].to(torch.float8_e4m3fn).float()
            q = q.to(dtype)

            def infinite(of, column, negative=False):
                """The keys of some pages infinite in this column, zero in the rest of its block."""
                c = torch.zeros(32, dtype=torch.int32, device="cuda")
                c[column % 32] = code | (sign if negative else 0)
                c = (c if fmt != "MXFP4" else c[0::2] | c[1::2] << 4).to(torch.uint8)
                block = column // 32
                cache.k_codes[of, :, :, block * len(c):(block + 1) * len(c)] = c
                cache.k_scales[of, :, :, block] = scale

            def call():
                return nn.cache_attend(q, cache, table, lengths, causal=False, return_lse=True)

            few = torch.tensor([1, pages - 1], device="cuda")
            others = table.clone()
            others[0, few] = -1
            want, want_lse, bound, lse_bound = oc.attend(q, cache, others, lengths, causal=False)
            infinite(few, 33, negative=True)
            out, lse = call()
            _check(out, want, bound, (dtype, dim))
            _check(lse, want_lse, lse_bound, (dtype, dim))
            infinite(few[:1], 33)
            assert torch.isnan(call()[0]).all()
            cache.k_codes[few[:1]] = 0
            infinite(few[:1], 1)
            assert torch.isnan(call()[0]).all()
            cache.k_codes.zero_()
            infinite(slice(None), 33, negative=True)
            out, lse = call()
            assert (out == 0).all() and (lse == -math.inf).all(), (dtype, dim)


@pytest.mark.parametrize("n, heads", [(3, 4), (7, 12), (100, 4)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_attend_queries_that_are_no_numbers(cuda, dtype, n, heads):
    """A NaN or an infinity in one query makes its own row NaN, and no other."""
    gen = _gen(26)
    for fmt, dim, page, keys in (("MXFP8_E4M3", 64, 16, 200), ("MXFP4", 128, 24, 200), ("MXFP8_E5M2", 200, 16, 6000)):
        cache = _filled(gen, -(-keys // page), page, 1, dim, fmt)
        cache.k_codes[..., 0] = {"MXFP8_E4M3": 0x38, "MXFP8_E5M2": 0x3C, "MXFP4": 0x22}[fmt]      # no key is zero where they are
        table, lengths = torch.arange(cache.k_codes.shape[0], device="cuda").int()[None], _i32([keys])
        q = torch.randn(1, n, heads, dim, generator=gen, device="cuda").to(DTYPES[dtype])
        want, want_lse, bound, lse_bound = oc.attend(q, cache, table, lengths)
        bad = torch.zeros(n, heads, dtype=torch.bool, device="cuda")
        bad[0, 1] = bad[n // 2, 0] = bad[n - 1, heads - 1] = True
        q[0, 0, 1, 0], q[0, n // 2, 0, 0], q[0, n - 1, heads - 1, 0] = math.nan, math.inf, math.nan
        out, lse = nn.cache_attend(q, cache, table, lengths, return_lse=True)
        assert torch.isnan(out[0, bad]).all() and torch.isnan(lse[0, bad]).all()
        _check(out[0, ~bad], want[0, ~bad], bound[0, ~bad], (fmt, dim))
        _check(lse[0, ~bad], want_lse[0, ~bad], lse_bound[0, ~bad], (fmt, dim))


def test_attend_strides(cuda):
    gen = _gen(12)
    cache = _filled(gen, 9, 16, 2, 72, "MXFP8_E4M3")
    table, lengths = _i32([[0, 1, 2, 3], [4, 5, 6, 7]]), _i32([50, 61])
    wide = torch.randn(2, 12, 5, 4 * 3, 72 + 5, generator=gen, device="cuda").bfloat16()
    q = wide[:, 4, :, 4:8, 3:75]
    assert torch.equal(nn.cache_attend(q, cache, table, lengths), nn.cache_attend(q.contiguous(), cache, table, lengths))
    swapped = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(nn.cache_attend(swapped, cache, table, lengths), nn.cache_attend(q.contiguous(), cache, table, lengths))
    apart = wide[:, 4, :, 4:8, ::2][..., :36]
    cache36 = _filled(gen, 9, 16, 2, 36, "MXFP8_E4M3")
    assert torch.equal(nn.cache_attend(apart, cache36, table, lengths), nn.cache_attend(apart.contiguous(), cache36, table, lengths))
    big = torch.full((2, 9), 10 ** 9, dtype=torch.int32, device="cuda")
    big[:, 2:6] = table
    assert torch.equal(nn.cache_attend(q, cache, big[:, 2:6], lengths), nn.cache_attend(q, cache, table, lengths))
    assert torch.equal(nn.cache_attend(q, cache, table.t().contiguous().t(), lengths), nn.cache_attend(q, cache, table, lengths))


def test_attend_same_bits_again(cuda):
    gen = _gen(13)
    lengths = [3000, 70, 9000, 1]
    cache = _filled(gen, 800, 16, 2, 128, "MXFP4")
    table = _table(gen, lengths, 16, 800)
    q = torch.randn(4, 3, 8, 128, generator=gen, device="cuda").bfloat16()
    first = nn.cache_attend(q, cache, table, _i32(lengths), return_lse=True)
    for _ in range(5):
        again = nn.cache_attend(q, cache, table, _i32(lengths), return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("fmt, page", [("MXFP4", 16), ("MXFP8_E4M3", 20)])
def test_attention_layer(cuda, fmt, page):
    """Projections on packed weights around the cache and its attention: prompts in pieces, then token by token, several
    sequences at once, their queries, keys and values views of one product.  Each step's attention is held to the oracle on
    the cache as it is, whose rows are the step's keys and values quantized; the layer's output is close to the same layer
    on float64."""
    gen = _gen(20)
    width, H, G, D, B, pages = 256, 8, 2, 64, 3, 40
    pack = lambda w: packed.quantize(w, "MXFP8_E4M3", axis=-1)                                # noqa: E731
    w_in = torch.randn((H + 2 * G) * D, width, generator=gen, device="cuda") / 16
    w_out = torch.randn(width, H * D, generator=gen, device="cuda") / 23
    w_in, w_out = pack(w_in), pack(w_out)
    plain = [packed.dequantize(*w, "MXFP8_E4M3", axis=-1).double() for w in (w_in, w_out)]
    cache = nn.packed_cache(pages, page, G, D, fmt)
    lengths = [0] * B
    table = torch.randperm(pages, generator=gen, device="cuda")[:B * 12].view(B, 12).int()
    for tokens in ([50, 7, 1], [64, 1, 0], [1, 1, 1], [1, 1, 1], [3, 0, 40]):
        starts = [0] + list(np.cumsum(tokens))
        x = torch.randn(starts[-1], width, generator=gen, device="cuda").bfloat16()
        at = torch.tensor([l + j for l, n in zip(lengths, tokens) for j in range(n)], device="cuda")
        which = torch.tensor([b for b, n in enumerate(tokens) for _ in range(n)], device="cuda")
        lengths = [l + n for l, n in zip(lengths, tokens)]
        slots = table[which, at // page].long() * page + at % page
        y = nn.packed_linear(x, *w_in, "MXFP8_E4M3").view(-1, H + 2 * G, D)
        q, k, v = y[:, :H], y[:, H:H + G], y[:, H + G:]
        nn.cache_write(k, v, cache, slots)
        for got, t in zip(nn.cache_read(cache, slots, torch.float32), (k, v)):
            codes, scales = packed.quantize(t, fmt, "ocp", axis=-1)
            assert torch.equal(got, packed.dequantize(codes, scales, fmt, axis=-1).float())
        if tokens == [1] * B:
            _attend(q[:, None], cache, table, _i32(lengths))
        out, _ = _attend(q, cache, table, _i32(lengths), _i32(starts))
        got = nn.packed_linear(out.reshape(-1, H * D), *w_out, "MXFP8_E4M3", residual=x)
        full = (x.double() @ plain[0].t()).view(-1, H + 2 * G, D)
        assert ((y.double() - full).abs() <= 2.0 ** -8 * full.abs() + 256 * 2.0 ** -23 * (x.double().abs() @ plain[0].abs().t()).view_as(full)).all()
        full = out.reshape(-1, H * D).double() @ plain[1].t()
        size = out.reshape(-1, H * D).double().abs() @ plain[1].abs().t() + x.double().abs()
        full = full + x.double()
        assert ((got.double() - full).abs() <= 2.0 ** -8 * full.abs() + 512 * 2.0 ** -23 * size).all()


def test_generation_captured_in_a_graph(cuda):
    """Write, then attend: a step captured once and replayed with new rows, slots, pages and lengths, the program's own
    steps between; two such graphs alive at once."""
    gen = _gen(14)
    pages, page, G, D, B = 600, 16, 2, 128, 3
    new = lambda: _filled(_gen(15), pages, page, G, D, "MXFP4")                       # noqa: E731
    graphs = []
    for prompt in (0, 40):
        n = prompt or 1
        cache = new()
        k, v = (torch.zeros(B * n, G, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        q = torch.zeros(B, n, 8, D, device="cuda", dtype=torch.bfloat16)
        slots = torch.zeros(B * n, dtype=torch.int64, device="cuda")
        table, lengths = torch.zeros(B, 190, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")

        def step():
            nn.cache_write(k, v, cache, slots)
            return nn.cache_attend(q, cache, table, lengths, return_lse=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, (k, v, q, slots, table, lengths), cache, n))
    other = new()
    for replay in range(4):
        for graph, out, (k, v, q, slots, table, lengths), cache, n in graphs:
            for t in (k, v, q):
                t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
            long = [(50 + 900 * replay), 40 + replay, 2900 - 800 * replay]
            lengths.copy_(_i32(long))
            table.copy_(_table(gen, long, page, pages, 190))
            at = torch.tensor([[l - n + j for j in range(n)] for l in long], device="cuda").clamp_min(0)
            slots.copy_((table.long().gather(1, at // page) * page + at % page).flatten())
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(other, cache[:4]):
                a.copy_(b)
            nn.cache_write(k, v, other, slots)
            want = nn.cache_attend(q, other, table, lengths, return_lse=True)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            for a, b in zip(other, cache[:4]):
                assert torch.equal(a, b)


def test_launches_are_timed(cuda):
    """The library's timers see a launch for each of a call's kernels: whole tiles in one, cut ones joined."""
    gen = _gen(19)
    cache = _filled(gen, 600, 16, 2, 64, "MXFP4")
    names = ("k_cache_write", "k_cache_read", "k_attend", "k_attend_join", "k_attend_none")
    q = torch.randn(2, 4, 64, generator=gen, device="cuda").bfloat16()
    slots = torch.arange(3, device="cuda")
    _lib.timer_enable(True)
    try:
        for name in names:
            _lib.timer_read(name)
        nn.cache_write(*nn.cache_read(cache, slots), cache, slots)
        for length, starts in ((100, None), (9000, None), (100, [0, 1, 1])):
            nn.cache_attend(q[:, None] if starts is None else q, cache, _table(gen, [length, 1], 16, 600), _i32([length, 1]),
                            None if starts is None else _i32(starts))
        nn.cache_attend(q, cache, _i32([]).view(0, 3), _i32([]), _i32([0]))
        got = {name: _lib.timer_read(name)[1] for name in names}
    finally:
        _lib.timer_enable(False)
    assert got == {"k_cache_write": 1, "k_cache_read": 1, "k_attend": 3, "k_attend_join": 1, "k_attend_none": 1}


def test_other_stream(cuda):
    gen = _gen(16)
    cache = _filled(gen, 300, 16, 2, 64, "MXFP4")
    lengths = [4000, 300]
    table = _table(gen, lengths, 16, 300)
    q = torch.randn(2, 2, 4, 64, generator=gen, device="cuda").bfloat16()
    want = nn.cache_attend(q, cache, table, _i32(lengths))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            got = nn.cache_attend(q, cache, table, _i32(lengths))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_cache_past_32_bit_offsets(cuda):
    """Pages more than 2^32 bytes from the cache's first: written, read and attended over as in a small cache."""
    gen = _gen(17)
    for fmt, pages in (("MXFP8_E4M3", 70000), ("MXFP4", 140000)):
        big = nn.packed_cache(pages, 64, 8, 128, fmt)
        assert big.k_codes.numel() > 1 << 32
        small = nn.packed_cache(12, 64, 8, 128, fmt)
        T, far = 600, pages - 12
        k, v = (torch.randn(T, 8, 128, generator=gen, device="cuda").bfloat16() for _ in range(2))
        slots = torch.arange(T, device="cuda") + 64
        nn.cache_write(k, v, small, slots)
        nn.cache_write(k, v, big, slots + far * 64)
        for a, b in zip(nn.cache_read(small, slots), nn.cache_read(big, slots + far * 64)):
            assert torch.equal(a, b) and (a != 0).any()
        assert (big.k_codes[0] == 0).all() and (big.k_codes[(1 << 32) // big.k_codes.stride(0)] == 0).all()
        table = torch.arange(1, 11, dtype=torch.int32, device="cuda")[None]
        for n in (1, 60, 300):
            q = torch.randn(1, n, 16, 128, generator=gen, device="cuda").bfloat16()
            want = nn.cache_attend(q, small, table, _i32([600]))
            assert torch.equal(nn.cache_attend(q, big, table + far, _i32([600])), want)
        del big
        torch.cuda.empty_cache()
