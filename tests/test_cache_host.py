"""Refusals of the cache's operators, on the CPU: every check runs before any device work.  And without a GPU a valid call
fails loudly."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from mxq import _lib, nn


def _cache(pages=4, page=16, heads=2, dim=40, fmt="MXFP4", **more):
    return nn.packed_cache(pages, page, heads, dim, fmt, device="cpu", **more)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("change, error, text", [
    (dict(pages=0), ValueError, "pages must be an integer from 1"),
    (dict(page_size=True), ValueError, "page_size must be an integer"),
    (dict(kv_heads=65536), ValueError, "kv_heads must be an integer from 1 to 65535"),
    (dict(head_dim=257), ValueError, "head_dim must be an integer from 1 to 256"),
    (dict(pages=2 ** 20, page_size=2 ** 12), ValueError, "slots"),
    (dict(fmt="MXFP6_E3M2"), ValueError, "fmt must name one of"),
    (dict(fmt="FP32"), ValueError, "fmt must name one of"),
    (dict(fmt="MXFP9"), ValueError, "Unknown format"),
])
def test_packed_cache_refuses(change, error, text):
    with pytest.raises(error, match=text):
        nn.packed_cache(**{**dict(pages=4, page_size=16, kv_heads=2, head_dim=40, fmt="MXFP4", device="cpu"), **change})


def test_packed_cache_shapes():
    for fmt, each in (("MXFP4", 16), ("MXFP8_E4M3", 32), ("e5m2", 32)):
        for dim, blocks in ((1, 1), (32, 1), (33, 2), (128, 4), (256, 8)):
            c = _cache(3, 5, 7, dim, fmt)
            assert c.k_codes.shape == c.v_codes.shape == (3, 7, 5, blocks * each) and c.page_size == 5
            assert c.k_scales.shape == c.v_scales.shape == (3, 7, 5, blocks)
            assert all(t.dtype == torch.uint8 for t in c[:4])


@pytest.mark.parametrize("change, error, text", [
    (dict(cache=(1, 2)), TypeError, "cache must be a PackedCache"),
    (dict(cache=_cache()._replace(k_codes=torch.zeros(4, 2, 16, 32))), TypeError, "must be uint8"),
    (dict(cache=_cache()._replace(k_scales=_cache(pages=5).k_scales)), ValueError, "must have codes"),
    (dict(cache=_cache()._replace(v_codes=_cache().v_codes[0])), ValueError, "pages x kv_heads"),
    (dict(cache=_cache()._replace(head_dim=65)), ValueError, "must have codes"),
    (dict(cache=_cache()._replace(head_dim=0)), ValueError, "head_dim must be"),
    (dict(cache=_cache()._replace(fmt="MXFP8_E4M3")), ValueError, "must have codes"),
    (dict(cache=_cache()._replace(fmt="MXFP6_E2M3")), ValueError, "fmt must name one of"),
    (dict(cache=_cache()._replace(k_codes=_cache().k_codes.transpose(2, 3).contiguous().transpose(2, 3))), ValueError,
     "next to each other"),
    (dict(cache=_cache()._replace(k_codes=_cache().k_codes[:1].expand(4, -1, -1, -1))), ValueError, "expanded"),
    (dict(slots=torch.zeros(3)), TypeError, "slots must be int32 or int64"),
    (dict(slots=_i32(3, 1)), ValueError, "slots must have one axis"),
    (dict(k=torch.zeros(3, 2, 41)), ValueError, "k must have shape"),
    (dict(v=torch.zeros(2, 2, 40)), ValueError, "v must have shape"),
    (dict(k=torch.zeros(3, 2, 40, dtype=torch.float64)), TypeError, "k must be float32"),
    (dict(v=torch.zeros(3, 2, 40, dtype=torch.float16)), TypeError, "one dtype"),
    (dict(k=torch.zeros(3, 2, 40, requires_grad=True)), RuntimeError, "no_grad"),
])
def test_cache_write_refuses(change, error, text):
    args = {**dict(k=torch.zeros(3, 2, 40), v=torch.zeros(3, 2, 40), cache=_cache(), slots=_i32(3)), **change}
    with pytest.raises(error, match=text):
        nn.cache_write(**args)


@pytest.mark.parametrize("change, error, text", [
    (dict(cache=None), TypeError, "cache must be a PackedCache"),
    (dict(slots=torch.zeros(3)), TypeError, "slots must be int32 or int64"),
    (dict(dtype=torch.float64), TypeError, "dtype must be"),
])
def test_cache_read_refuses(change, error, text):
    with pytest.raises(error, match=text):
        nn.cache_read(**{**dict(cache=_cache(), slots=_i32(3)), **change})


@pytest.mark.parametrize("change, error, text", [
    (dict(cache=None), TypeError, "cache must be a PackedCache"),
    (dict(q=torch.zeros(3, 6, 40)), ValueError, "q must be B x n"),
    (dict(q=torch.zeros(3, 1, 6, 40), starts=_i32(4)), ValueError, "q must be B x n"),
    (dict(q=torch.zeros(3, 1, 5, 40)), ValueError, "multiple of 2 heads"),
    (dict(q=torch.zeros(3, 1, 0, 40)), ValueError, "multiple of 2 heads"),
    (dict(q=torch.zeros(3, 1, 6, 41)), ValueError, "multiple of 2 heads"),
    (dict(q=torch.zeros(3, 1, 6, 40, dtype=torch.float64)), TypeError, "q must be float32"),
    (dict(q=torch.zeros(3, 1, 6, 40, requires_grad=True)), RuntimeError, "no_grad"),
    (dict(q=torch.zeros(2, 1, 6, 40)), ValueError, "q must have 3 sequences"),
    (dict(table=torch.zeros(3, 2)), TypeError, "table must be int32"),
    (dict(table=_i32(3)), ValueError, "table must have shape"),
    (dict(lengths=_i32(2)), ValueError, "lengths must have shape"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), TypeError, "lengths must be int32"),
    (dict(q=torch.zeros(3, 6, 40), starts=_i32(3)), ValueError, "starts must have shape"),
    (dict(q=torch.zeros(3, 6, 40), starts=torch.zeros(4)), TypeError, "starts must be int32"),
    (dict(window=0), ValueError, "window must be an integer from 1"),
    (dict(scale=0.0), ValueError, "scale must be positive"),
    (dict(scale=float("nan")), ValueError, "scale must be positive"),
    (dict(scale=float("inf")), ValueError, "scale must be positive"),
    (dict(scale=1.8e38), ValueError, "scale must be positive"),
    (dict(table=_i32(1, 1).expand(3, 2 ** 27)), ValueError, "keys a sequence"),
    (dict(table=_i32(1, 1).expand(3, 2 ** 27 - 2 ** 12 + 1)), ValueError, "keys a sequence"),
])
def test_cache_attend_refuses(change, error, text):
    args = {**dict(q=torch.zeros(3, 1, 6, 40), cache=_cache(), table=_i32(3, 2), lengths=_i32(3)), **change}
    with pytest.raises(error, match=text):
        nn.cache_attend(**args)


@pytest.mark.parametrize("change, text", [
    (dict(cache=_cache()._replace(head_dim=0)), "head_dim must be"),            # before its default scale, 0 to a negative power
    (dict(cache=_cache()._replace(head_dim="40")), "head_dim must be"),
    (dict(scale=1e-50), "scale must be positive"),                              # zero as a float32
    (dict(scale=1e300), "scale must be positive"),
    (dict(scale=-1.0), "scale must be positive")])
def test_cache_attend_refuses_by_its_own_errors(change, text):
    with pytest.raises(ValueError, match=text):
        nn.cache_attend(**{**dict(q=torch.zeros(3, 1, 6, 40), cache=_cache(), table=_i32(3, 2), lengths=_i32(3)), **change})


def test_refused_views_are_not_copied(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "contiguous", lambda t, *args, **more: pytest.fail("copied"))
    with pytest.raises(ValueError, match="keys a sequence"):
        nn.cache_attend(torch.zeros(3, 1, 6, 40), _cache(), _i32(1, 1).expand(3, 2 ** 27), _i32(3))
    with pytest.raises(ValueError, match="too many"):
        nn.cache_attend(torch.zeros(3, 1, 1, 1).expand(3, 2 ** 27, 6, 40), _cache(), _i32(3, 2), _i32(3))


def test_forward_mode_tangents_are_refused():
    dual = lambda *shape: forward_ad.make_dual(torch.zeros(shape), torch.ones(shape))         # noqa: E731
    plain = torch.zeros
    with forward_ad.dual_level():
        for call in (lambda: nn.cache_write(dual(3, 2, 40), plain(3, 2, 40), _cache(), _i32(3)),
                     lambda: nn.cache_write(plain(3, 2, 40), dual(3, 2, 40), _cache(), _i32(3)),
                     lambda: nn.cache_attend(dual(3, 1, 6, 40), _cache(), _i32(3, 2), _i32(3))):
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is visible")
def test_no_gpu_fails_loudly():
    for call in (lambda: nn.packed_cache(4, 16, 2, 40),
                 lambda: nn.cache_write(torch.zeros(3, 2, 40), torch.zeros(3, 2, 40), _cache(), _i32(3)),
                 lambda: nn.cache_read(_cache(), _i32(3)),
                 lambda: nn.cache_attend(torch.zeros(3, 1, 6, 40), _cache(), _i32(3, 2), _i32(3))):
        with pytest.raises(RuntimeError, match="no GPU is visible"):
            call()


def test_c_entries_refuse():
    """Bad sizes, specs and NULL arguments come back as MXQ_EINVAL with a message, before any HIP call."""
    lib = _lib.load()
    buf = ctypes.cast((ctypes.c_uint8 * 4096)(), ctypes.c_void_p)

    def refused(text, name, *args):
        assert getattr(lib, name)(*args) == 1, (name, args)
        assert text in lib.mxq_last_error().decode(), lib.mxq_last_error()

    def cache(**change):
        good = dict(format=5, head_dim=64, pages=4, page_size=16, kv_heads=2)
        return _lib.CacheSpec(**{**good, **change})

    def attend(**change):
        good = dict(dtype=1, causal=1, scale=1.0, T=4, B=4, heads=4, q_token=256, q_head=64, table_pages=2, table_row=2)
        return _lib.AttendSpec(**{**good, **change})

    write = lambda spec, dtype=1, T=3, k=buf: (k, buf, dtype, T, 128, 64, 128, 64, buf, 0, buf, buf, buf, buf, spec, 0)  # noqa: E731
    read = lambda spec, dtype=1, T=3, k=buf: (buf, buf, buf, buf, spec, buf, 0, T, k, buf, dtype, 0)          # noqa: E731
    run = lambda spec, att, q=buf, starts=0: (q, buf, buf, buf, buf, spec, buf, buf, starts, buf, 0, att, 0, 0)  # noqa: E731
    bad = ((dict(format=2), "format"), (dict(format=4), "format"), (dict(head_dim=0), "head_dim"), (dict(head_dim=257), "head_dim"),
           (dict(pages=0), "out of range"), (dict(page_size=0), "out of range"), (dict(kv_heads=65536), "out of range"),
           (dict(pages=1 << 20, page_size=1 << 12), "out of range"))
    for change, text in bad:
        refused(text, "mxq_cache_write", *write(cache(**change)))
        refused(text, "mxq_cache_read", *read(cache(**change)))
        refused(text, "mxq_cache_attend", *run(cache(**change), attend()))
        assert lib.mxq_cache_attend_workspace(cache(**change), attend(), 0) == 0
    for name, make in (("mxq_cache_write", write), ("mxq_cache_read", read)):
        refused("dtype", name, *make(cache(), dtype=3))
        refused("out of range", name, *make(cache(), T=-1))
        refused("NULL", name, *make(cache(), k=0))
        refused("NULL", name, *make(None))
    for change, text in ((dict(dtype=3), "dtype"), (dict(heads=3), "multiple"), (dict(heads=0), "out of range"), (dict(T=-1), "out of range"),
                         (dict(T=1 << 29, heads=4), "out of range"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
                         (dict(scale=float("nan")), "scale"), (dict(window=-1), "window"), (dict(table_pages=-1), "table"),
                         (dict(scale=1.8e38), "scale"), (dict(table_pages=1 << 27), "table"), (dict(table_pages=(1 << 27) - (1 << 12) + 1), "table"),
                         (dict(T=5), "multiple of B"), (dict(B=0), "multiple of B")):
        refused(text, "mxq_cache_attend", *run(cache(), attend(**change)))
    refused("NULL", "mxq_cache_attend", *run(cache(), attend(), q=0))
    refused("NULL spec", "mxq_cache_attend", *run(None, attend()))
    refused("workspace", "mxq_cache_attend", *run(cache(pages=1 << 12), attend(table_pages=1 << 12)))


def test_workspace():
    """None where no sequence can have more keys than a workgroup takes; else one size for any number of sequences."""
    lib = _lib.load()
    cache = _lib.CacheSpec(5, 128, 4096, 16, 2)
    size = lambda ragged=0, **change: lib.mxq_cache_attend_workspace(cache, _lib.AttendSpec(**{**dict(      # noqa: E731
        dtype=1, causal=1, scale=1.0, T=4, B=4, heads=8, table_pages=1000, table_row=1000), **change}), ragged)
    assert size(table_pages=14) == 0 and size(T=0) == 0 and size(window=200) == 0
    assert 0 < size() == size(T=8) == size(T=40, B=40) <= 64 << 20


def test_most_workspace():
    """Of every type, width, head layout and batch: two parts of a tile for each workgroup, of 128 rows of 128 columns and of 32
    where there are prompts and tokens in one batch, two workgroups a CU."""
    lib, most = _lib.load(), {0: 0, 1: 0}
    for dtype in (0, 1, 2):
        for dim in (32, 64, 96, 128, 256):
            for kv_heads, group in ((1, 1), (2, 8), (1, 17), (4, 32), (1, 64), (2, 65), (1, 1024)):
                for T, B in ((4, 4), (64, 1), (8192, 1), (8192, 23), (512, 64), (600, 300), (100000, 100)):
                    for pages in (10, 200, 8192):
                        cache = _lib.CacheSpec(5, dim, 1 << 20, 16, kv_heads)
                        spec = _lib.AttendSpec(dtype=dtype, causal=1, scale=1.0, T=T, B=B, heads=kv_heads * group, table_pages=pages, table_row=pages)
                        for ragged in (0, 1):
                            if ragged or T % B == 0:
                                most[ragged] = max(most[ragged], lib.mxq_cache_attend_workspace(cache, spec, ragged))
    part = lambda rows, columns: 2 * 512 * rows * (columns + 2) * 4                                # noqa: E731
    assert most == {0: part(256, 64), 1: part(128, 128) + part(32, 128)} and most[1] < 86e6


@pytest.mark.parametrize("here", [False, True])
def test_strides_are_of_what_the_call_reads(monkeypatch, here):
    """A view is laid out anew by its copy to the call's device: the spec has the strides of the tensors whose memory the
    call is given.  The meta device stands for the GPU; nothing runs."""
    dev, read, called = torch.device("meta"), [], []
    monkeypatch.setattr(_lib, "compute_device", lambda *tensors: dev)
    monkeypatch.setattr(_lib, "stream", lambda dev: 0)
    monkeypatch.setattr(_lib, "back", lambda t, like: t)
    monkeypatch.setattr(_lib, "run", lambda name, *args: called.append(args))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: read.append(t) or len(read) - 1, raising=False)
    cache = nn.packed_cache(9, 16, 2, 40, "MXFP4", device="meta" if here else "cpu")
    wide = torch.zeros(3, 5, 12, 45)
    queries = ((wide[..., 3:7, 5:], None), (wide[:, 1:3, :4, :40], None), (wide[:, 2:3, :4, :40], None),
               (wide[:1, :, :2, :40].expand(3, 5, 2, 40), None), (wide[..., :1, :40].expand(3, 5, 4, 40), None),
               (wide[0, :, 4:8, :40], _i32(4)), (wide[0, ::2, ::3, 5:], _i32(4)), (wide[0, :, :1, :40].expand(5, 4, 40), _i32(4)))
    tables = (_i32(3, 9)[:, 2:6], _i32(3, 9)[:, ::2], _i32(4, 3).t(), _i32(1, 4).expand(3, 4), _i32(6, 4)[::2], _i32(3, 4))
    for q, starts in queries:
        for table in tables:
            for q_here, table_here in ((False, False), (True, False), (False, True)):
                read.clear(), called.clear()
                out = nn.cache_attend(q.to(dev) if q_here else q, cache, table.to(dev) if table_here else table, _i32(3), starts)
                (args,) = called
                assert out.shape == q.shape and all(t.device == dev for t in read)
                qd, td, spec = read[args[0]], read[args[6]], args[11]
                assert qd.shape == q.shape and td.shape == table.shape
                assert qd.stride(-1) == 1 and spec.q_head == qd.stride(-2) and td.stride(1) == 1 and spec.table_row == td.stride(0)
                if starts is not None or q.shape[1] > 1:
                    assert spec.q_token == qd.stride(-3) and (starts is not None or qd.stride(0) == q.shape[1] * qd.stride(1))
                else:
                    assert spec.q_token == qd.stride(0)
