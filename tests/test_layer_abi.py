"""The operators between a layer's products without a GPU: what they refuse on the host, and that calls without work need no
device."""
import ctypes

import pytest


@pytest.fixture
def L(pkg):
    lib = pkg.library()
    lib.hq_clear_error()
    yield lib
    lib.hq_clear_error()


def norm(L, xq=4096, xs=8192, y=0, r=4096, x=4096, d=4096, w=4096, n=256, eps=1e-5, ready=0, count=2, frame=320, x_stride=1024,
         d_stride=1024, y_stride=1024):
    return L.hq_norm_ready_ex(xq, xs, y, r, x, d, w, n, eps, ready, count, frame, x_stride, d_stride, y_stride, None)


@pytest.mark.parametrize("wrong, code, words", [
    (dict(n=48), 1, "multiple of 32"), (dict(n=0), 1, "multiple of 32"), (dict(n=-32), 1, "multiple of 32"),
    (dict(n=160, ready=2), 1, "multiple of 128"), (dict(n=384, ready=3), 1, "multiple of 256"), (dict(ready=4), 1, "ready = 4"),
    (dict(ready=-1), 1, "ready = -1"), (dict(eps=-1e-5), 1, "eps"), (dict(eps=float("nan")), 1, "eps"),
    (dict(eps=float("inf")), 1, "eps"), (dict(count=-1), 1, "count = -1"), (dict(x=None), 3, "x or w"), (dict(w=None), 3, "x or w"),
    (dict(xq=None), 3, "both NULL"), (dict(r=None), 3, "d without r"), (dict(xs=None), 3, "without xs"),
    (dict(x=4104), 2, "16-byte"), (dict(d=4100), 2, "16-byte"), (dict(w=4108), 2, "16-byte"), (dict(r=4104), 2, "16-byte"),
    (dict(y=4104), 2, "16-byte"), (dict(xq=4098), 2, "4-byte"), (dict(xs=8193), 2, "4-byte"), (dict(x_stride=1028), 2, "stride"),
    (dict(d_stride=-16), 2, "stride"), (dict(y=4096, y_stride=8), 2, "stride"), (dict(frame=328), 2, "frame"),
])
def test_norm_refusals(L, wrong, code, words):
    assert norm(L, **wrong) == code
    assert L.hq_last_error() == code and words in L.hq_last_error_message().decode()


@pytest.mark.parametrize("wrong, words", [
    (dict(x_stride=1008), "x_stride = 1008"), (dict(x_stride=0), "x_stride = 0"), (dict(x_stride=1008, d=None), "x_stride = 1008"),
    (dict(y=4096, y_stride=1008), "y_stride = 1008"), (dict(y=4096, y_stride=0), "y_stride = 0"), (dict(frame=240), "frame = 240"),
    (dict(frame=0), "frame = 0"),
])
def test_norm_rows_that_overlap(L, wrong, words):
    """rows of several tokens that are written may not reach into each other"""
    assert norm(L, **wrong) == 1
    assert L.hq_last_error() == 1 and words in L.hq_last_error_message().decode()


@pytest.mark.parametrize("wrong", [
    dict(xs=4096 + 256, frame=256), dict(xs=4096 + 256, frame=272), dict(xs=4096 + 256, frame=304, ready=2),
    dict(xs=4096 + 256, frame=368, ready=3), dict(xs=4096), dict(xs=4096 + 252), dict(xs=4096 - 16), dict(xs=4096 + 320, frame=320),
    dict(xs=4096 + 128, count=1), dict(xs=4096 - 16, count=1),
])
def test_norm_scales_that_overlap(L, wrong):
    """scales (n / 8 bytes; with planes n / 4, with sums n / 2) may lie in the activations' frames, beside them"""
    assert norm(L, **wrong) == 1
    assert L.hq_last_error() == 1 and "overlap" in L.hq_last_error_message().decode()


def test_norm_without_tokens(L):
    assert norm(L, x=None, count=0) == 0


def paged(pkg, **wrong):
    c = dict(k=4096, v=4096, ks=4096, vs=4096, form=0, pages=10, page=16, heads=2, dim=64)
    b = dict(starts=4096, lengths=4096, table=4096, sequences=2, tokens=3, longest=0, width=4)
    c.update({k: v for k, v in wrong.items() if k in c})
    b.update({k: v for k, v in wrong.items() if k in b})
    return pkg.cache.Cache(*c.values()), pkg.cache.Batch(*b.values())


COMMON = [
    (dict(form=2), 1, "form 2"), (dict(page=8), 1, "page = 8"), (dict(page=48), 1, "page = 48"), (dict(page=512), 1, "page = 512"),
    (dict(page=0), 1, "page = 0"), (dict(dim=24), 1, "dim = 24"), (dict(dim=0), 1, "dim = 0"), (dict(dim=272), 1, "dim = 272"),
    (dict(heads=0), 1, "heads = 0"), (dict(heads=1025), 1, "heads"), (dict(pages=-1), 1, "pages = -1"),
    (dict(sequences=-1), 1, "sequences = -1"), (dict(tokens=-1), 1, "tokens = -1"), (dict(tokens=1 << 25), 1, "tokens = "),
    (dict(longest=-1), 1, "longest = -1"), (dict(width=-1), 1, "width = -1"), (dict(width=1 << 27), 1, "a table of"),
    (dict(starts=None), 3, "starts"), (dict(lengths=None), 3, "lengths"), (dict(table=None), 3, "table"),
    (dict(table=4098), 2, "4-byte"), (dict(k=None), 3, "NULL"), (dict(vs=None), 3, "NULL"), (dict(v=4104), 2, "16-byte"),
    (dict(ks=4100), 2, "16-byte"),
]


@pytest.mark.parametrize("wrong, code, words", COMMON + [
    (dict(row=None), 3, "row"), (dict(row=4100), 2, "16-byte"), (dict(stride=520), 2, "stride"), (dict(stride=-512), 2, "stride"),
    (dict(stride=256), 1, "stride"),
])
@pytest.mark.parametrize("call", ["hq_cache_write_ex", "hq_cache_read_ex"])
def test_cache_refusals(pkg, L, call, wrong, code, words):
    c, b = paged(pkg, **wrong)
    row, stride = wrong.get("row", 4096) if "row" in wrong else 4096, wrong.get("stride", 512)
    assert getattr(L, call)(c, b, row, 4096, stride, 512, None) == code
    assert words in L.hq_last_error_message().decode()
    if "row" in wrong or "stride" in wrong:
        assert getattr(L, call)(c, b, 4096, row, 512, stride, None) == code


@pytest.mark.parametrize("wrong, code, words", COMMON + [
    (dict(q=None), 3, "row"), (dict(out=4100), 2, "16-byte"), (dict(q_stride=1032), 2, "stride"), (dict(out_stride=512), 1, "stride"),
    (dict(queries=3), 1, "3 query heads"), (dict(queries=0), 1, "query heads"), (dict(queries=1026), 1, "query heads"),
    (dict(scale=0.0), 1, "scale"), (dict(scale=-1.0), 1, "scale"), (dict(scale=float("nan")), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale"), (dict(window=-1), 1, "window"), (dict(cap=-1.0), 1, "cap"),
    (dict(cap=float("nan")), 1, "cap"), (dict(less=1), 1, "workspace"), (dict(work=4224), 2, "256-byte"), (dict(work=None), 3, "work"),
])
def test_attention_refusals(pkg, L, wrong, code, words):
    c, b = paged(pkg, **wrong)
    heads = wrong.get("queries", 4)
    need = L.hq_attention_work_bytes(*paged(pkg), 4)
    if "less" in wrong or "work" in wrong:
        if need == 0:
            pytest.skip("no workspace is needed")
    work = wrong["work"] if "work" in wrong else 4096
    status = L.hq_attention_ex(wrong.get("out", 4096), wrong["q"] if "q" in wrong else 4096, heads, wrong.get("out_stride", 1024),
                               wrong.get("q_stride", 1024), c, b, wrong.get("scale", 0.125), wrong.get("window", 0),
                               wrong.get("cap", 0.0), work, need - wrong.get("less", 0), None)
    assert status == code
    assert words in L.hq_last_error_message().decode()


def test_null_descriptions(pkg, L):
    c, b = paged(pkg)
    assert L.hq_cache_write_ex(None, b, 4096, 4096, 512, 512, None) == 3
    assert L.hq_cache_read_ex(c, None, 4096, 4096, 512, 512, None) == 3
    assert L.hq_attention_work_bytes(None, b, 4) == -1 and L.hq_last_error() == 3
    assert L.hq_attention_work_bytes(c, b, 5) == -1 and L.hq_last_error() == 1


def test_work_bytes_need_no_memory(pkg, L):
    """a workspace can be sized before anything is allocated"""
    c, b = paged(pkg, k=None, v=None, ks=None, vs=None, starts=None, lengths=None, table=None)
    assert L.hq_attention_work_bytes(c, b, 4) == L.hq_attention_work_bytes(*paged(pkg), 4) >= 0


def test_too_many(pkg, L):
    """what a launch's grid or 32-bit positions could not count is refused, a table that covers 2^30 positions is not"""
    for wrong, words in ((dict(sequences=(1 << 22) + 1), "sequences = "), (dict(sequences=2 ** 31 - 1), "sequences = "),
                         (dict(width=(1 << 26) + 1), "a table of")):
        assert L.hq_cache_write_ex(*paged(pkg, **wrong), 4096, 4096, 512, 512, None) == 1
        assert words in L.hq_last_error_message().decode()
    assert L.hq_cache_write_ex(*paged(pkg, width=1 << 26, tokens=0), 4096, 4096, 512, 512, None) == 0


@pytest.mark.parametrize("none", [dict(tokens=0), dict(sequences=0)])
def test_calls_without_tokens(pkg, L, none):
    c, b = paged(pkg, starts=None, lengths=None, table=None, **none)
    assert L.hq_cache_write_ex(c, b, None, None, 0, 0, None) == 0
    assert L.hq_cache_read_ex(c, b, None, None, 0, 0, None) == 0
    assert L.hq_attention_ex(None, None, 4, 0, 0, c, b, 0.125, 0, 0.0, None, 0, None) == 0


def test_structures_are_the_headers(pkg):
    """the ctypes structures lie as hq.h's on a 64-bit host"""
    C, B = pkg.cache.Cache, pkg.cache.Batch
    assert ctypes.sizeof(C) == 4 * 8 + 5 * 4 + 4 and C.form.offset == 32 and C.dim.offset == 48
    assert ctypes.sizeof(B) == 3 * 8 + 4 * 4 and B.sequences.offset == 24 and B.width.offset == 36


def test_shapes(pkg):
    k, v, s, nbytes = pkg.cache.shapes("f16", 3, 16, 2, 48)
    assert k == (3, 2, 16, 48) and v == (3, 2, 48, 16) and s == (3, 2, 16) and nbytes == 2 * 96 * (96 + 4)
