"""The operators around a step's layers without a GPU: what they refuse on the host, and that calls without work need no device."""
import ctypes

import pytest


@pytest.fixture
def L(pkg):
    lib = pkg.library()
    lib.hq_clear_error()
    yield lib
    lib.hq_clear_error()


def refused(L, status, code, words):
    assert status == code, L.hq_last_error_message()
    assert L.hq_last_error() == code and words in L.hq_last_error_message().decode()


def embed(L, out=4096, ids=4096, values=4096, scales=4096, packing=0, vocab=100, dim=256, scale=1.0, count=2, stride=1024):
    return L.hq_embed_ex(out, ids, values, scales, packing, vocab, dim, scale, count, stride, None)


@pytest.mark.parametrize("wrong, code, words", [
    (dict(packing=4), 1, "packing 4"), (dict(packing=-1), 1, "packing -1"), (dict(packing=256 + 11), 1, "packing 267"),
    (dict(packing=256), 1, "packing 256"), (dict(vocab=0), 1, "vocab = 0"), (dict(dim=0), 1, "dim = 0"),
    (dict(packing=1, dim=48), 1, "groups of 32"), (dict(packing=2, dim=192), 1, "groups of 128"),
    (dict(packing=3, dim=64), 1, "groups of 128"), (dict(packing=256 + 12, dim=384), 1, "groups of 256"),
    (dict(scale=float("nan")), 1, "scale"), (dict(scale=float("inf")), 1, "scale"), (dict(count=-1), 1, "count = -1"),
    (dict(out=None), 3, "NULL"), (dict(ids=None), 3, "NULL"), (dict(values=None), 3, "NULL"), (dict(scales=None), 3, "NULL"),
    (dict(out=4100), 2, "out"), (dict(ids=4098), 2, "ids"), (dict(values=4104), 2, "16-byte aligned"), (dict(scales=4098), 2, "scales"),
    (dict(values=4100, packing=1), 2, "8-byte aligned"), (dict(values=4097, packing=256 + 12), 2, "2-byte aligned"),
    (dict(scales=4104, packing=256 + 12), 2, "scales"), (dict(scales=4097, packing=2), 2, "scales"),
    (dict(stride=1032), 2, "out_stride"), (dict(stride=-1024), 2, "out_stride"), (dict(stride=1008), 1, "out_stride"),
])
def test_embed_refusals(L, wrong, code, words):
    refused(L, embed(L, **wrong), code, words)


def pool_and_batch(pkg, **wrong):
    q = dict(free=4096, count=4096, left=4096, missing=4096, pages=10, page=16)
    b = dict(starts=4096, lengths=4096, table=4096, sequences=2, tokens=3, longest=0, width=4)
    q.update({k: v for k, v in wrong.items() if k in q})
    b.update({k: v for k, v in wrong.items() if k in b})
    return pkg.cache.Batch(*b.values()), pkg.cache.Pool(*q.values())


POOL = [
    (dict(page=8), 1, "page = 8"), (dict(page=512), 1, "page = 512"), (dict(page=0), 1, "page = 0"), (dict(pages=-1), 1, "pages = -1"),
    (dict(free=None), 3, "free"), (dict(count=None), 3, "count"), (dict(left=None), 3, "left"), (dict(free=4098), 2, "free"),
    (dict(missing=4097), 2, "missing"), (dict(width=1 << 27), 1, "a table of"), (dict(sequences=-1), 1, "sequences = -1"),
    (dict(sequences=(1 << 22) + 1), 1, "sequences = "), (dict(width=-1), 1, "width = -1"), (dict(table=None), 3, "table"),
    (dict(table=4098), 2, "4-byte"),
]


@pytest.mark.parametrize("wrong, code, words", POOL + [
    (dict(tokens=-1), 1, "tokens = -1"), (dict(tokens=(1 << 24) + 1), 1, "tokens = "), (dict(starts=None), 3, "starts"),
    (dict(lengths=None), 3, "lengths"), (dict(held=None), 3, "held"), (dict(fresh=None), 3, "fresh"), (dict(fresh=4098), 2, "int32"),
    (dict(sequence=4098), 2, "int32"), (dict(position=4097), 2, "int32"), (dict(slot=4100), 2, "slot"), (dict(starts=4097), 2, "int32"),
])
def test_plan_refusals(pkg, L, wrong, code, words):
    b, q = pool_and_batch(pkg, **wrong)
    rest = dict(held=4096, fresh=4096, sequence=4096, position=4096, slot=4096)
    rest.update({k: v for k, v in wrong.items() if k in rest})
    refused(L, L.hq_batch_plan_ex(b, q, *rest.values(), None), code, words)


@pytest.mark.parametrize("wrong, code, words", POOL + [(dict(from_=4098), 2, "from"), (dict(to=4097), 2, "to")])
def test_give_refusals(pkg, L, wrong, code, words):
    b, q = pool_and_batch(pkg, **wrong)
    refused(L, L.hq_pages_give_ex(q, b.table, b.sequences, b.width, wrong.get("from_"), wrong.get("to"), None), code, words)


def test_null_descriptions(pkg, L):
    b, q = pool_and_batch(pkg)
    refused(L, L.hq_batch_plan_ex(None, q, 4096, 4096, None, None, None, None), 3, "batch")
    refused(L, L.hq_batch_plan_ex(b, None, 4096, 4096, None, None, None, None), 3, "pool")
    refused(L, L.hq_pages_give_ex(None, 4096, 2, 4, None, None, None), 3, "pool")


def adapters(pkg, L, less=0, **wrong):
    t = dict(a=4096, b=4096, from_=4096, y=4096, rows=64, from_stride=256, y_stride=256)
    c = dict(count=2, x=4096, x_stride=512, n=128, rank=16, adapters=3, form=1, scales=4096, which=4096)
    b = dict(starts=4096, lengths=None, table=None, sequences=2, tokens=3, longest=0, width=0)
    for d in (t, c, b):
        d.update({k: v for k, v in wrong.items() if k in d})
    targets = None if "targets" in wrong else (pkg.adapters.Target * 9)(*([pkg.adapters.Target(*t.values())] * 9))
    batch = None if "batch" in wrong else pkg.cache.Batch(*b.values())
    need = L.hq_adapters_work_bytes(2, 16, 3)
    assert need >= 0
    work = wrong["work"] if "work" in wrong else 4096
    order = ("x", "x_stride", "n", "rank", "adapters", "form", "scales", "which")
    return L.hq_adapters_ex(targets, c["count"], *(c[k] for k in order), batch, work, need - less, None)


@pytest.mark.parametrize("wrong, code, words", [
    (dict(count=-1), 1, "count = -1"), (dict(count=9), 1, "count = 9"), (dict(rank=0), 1, "rank = 0"), (dict(rank=12), 1, "rank = 12"),
    (dict(rank=264), 1, "rank = 264"), (dict(n=0), 1, "n = 0"), (dict(n=48), 1, "n = 48"), (dict(adapters=-1), 1, "adapters = -1"),
    (dict(form=0), 1, "form 0"), (dict(form=3), 1, "form 3"), (dict(rows=-1), 1, "-1 rows"), (dict(rows=(1 << 23) + 1), 1, "rows"), (dict(tokens=-1), 1, "tokens = -1"),
    (dict(sequences=-1), 1, "sequences = -1"), (dict(tokens=(1 << 24) + 1), 1, "tokens = "), (dict(targets=None), 3, "targets"),
    (dict(batch=None), 3, "batch"), (dict(starts=None), 3, "starts"), (dict(which=None), 3, "which"), (dict(x=None), 3, "x NULL"),
    (dict(a=None), 3, "a, b or y"), (dict(b=None), 3, "a, b or y"), (dict(y=None), 3, "a, b or y"), (dict(x=4104), 2, "16-byte"),
    (dict(a=4104), 2, "16-byte"), (dict(b=4098), 2, "16-byte"), (dict(from_=4098), 2, "4-byte"), (dict(y=4098), 2, "4-byte"),
    (dict(starts=4098), 2, "4-byte"), (dict(which=4098), 2, "4-byte"), (dict(scales=4097), 2, "4-byte"), (dict(x_stride=520), 2, "x_stride"),
    (dict(x_stride=-512), 2, "x_stride"), (dict(x_stride=496), 1, "x_stride"), (dict(y_stride=258), 2, "stride"),
    (dict(from_stride=-256), 2, "stride"), (dict(y_stride=240), 1, "strides"), (dict(from_stride=240), 1, "strides"),
    (dict(less=1), 1, "workspace"), (dict(work=None), 3, "work"), (dict(work=4224), 2, "256-byte"),
])
def test_adapters_refusals(pkg, L, wrong, code, words):
    refused(L, adapters(pkg, L, **wrong), code, words)


@pytest.mark.parametrize("none", [dict(count=0), dict(tokens=0), dict(sequences=0)])
def test_adapters_without_work(pkg, L, none):
    assert adapters(pkg, L, which=None, x=None, work=None, **none) == 0


def test_adapters_work_bytes(L):
    for wrong in ((-1, 16, 3), (9, 16, 3), (2, 12, 3), (2, 0, 3), (2, 16, -1), (2, 16, (1 << 24) + 1)):
        assert L.hq_adapters_work_bytes(*wrong) == -1 and L.hq_last_error() == 1


def test_adapters_of_many_sequences(pkg, L):
    """more than 2^21 sequences of several tokens are refused before a launch that has no room for their blocks"""
    for longest in (0, 2):
        refused(L, adapters(pkg, L, sequences=(1 << 21) + 1, longest=longest), 1, "sequences = 2097153")
    for more in (dict(sequences=1 << 21), dict(sequences=1 << 22, longest=1)):
        refused(L, adapters(pkg, L, x=4104, **more), 2, "16-byte")  # (the sequences pass)


def test_adapters_work_covers_what_is_written(L):
    """a launch writes splits x tokens x projections x rank numbers (up to 4 splits where its blocks, of 16 tokens and 64 numbers, are
    so many times within 256), of the projections that have rows: fewer than the call states, which may be split more often; so the
    bytes grow with projections, ranks and tokens"""
    def written(count, rank, tokens):
        blocks = max(1, -(-tokens // 16) * -(-(-(-count * rank // 16)) // 4))
        return 4 * max(1, min(4, 256 // blocks)) * tokens * count * rank
    tokens = [0, 1, 7, 16, 17, 100, 250, 256, 335, 336, 337, 447, 448, 449, 671, 672, 673, 1000, 1024, 1040, 1365, 2048, 4095, 4097, 1 << 24]
    for rank in (8, 16, 24, 64, 72, 128, 136, 256):
        for count in range(1, 9):
            need = [L.hq_adapters_work_bytes(count, rank, t) for t in tokens]
            assert need == sorted(need)
            for t, n in zip(tokens, need):
                assert n >= max(written(c, rank, t) for c in range(1, count + 1)), (count, rank, t)
                assert n >= L.hq_adapters_work_bytes(count, rank - 8, t) or rank == 8
                assert n >= L.hq_adapters_work_bytes(count - 1, rank, t)


def sample(L, tokens=4096, chance=4096, logits=4096, u=4096, temperature=4096, top_k=4096, top_p=4096, min_p=4096, rows=2, vocab=100,
           stride=400, less=0, **more):
    need = L.hq_sample_work_bytes(2, 100)
    work = more["work"] if "work" in more else 4096
    return L.hq_sample_ex(tokens, chance, logits, u, temperature, top_k, top_p, min_p, rows, vocab, stride, work, need - less, None)


@pytest.mark.parametrize("wrong, code, words", [
    (dict(rows=-1), 1, "rows = -1"), (dict(rows=(1 << 20) + 1), 1, "rows = "), (dict(vocab=0), 1, "vocab = 0"), (dict(vocab=-5), 1, "vocab = -5"),
    (dict(vocab=(1 << 20) + 1), 1, "vocab = "), (dict(tokens=None), 3, "tokens"), (dict(logits=None), 3, "logits"), (dict(u=None), 3, "u NULL"),
    (dict(tokens=4098), 2, "4-byte"), (dict(chance=4097), 2, "4-byte"), (dict(logits=4098), 2, "4-byte"), (dict(u=4098), 2, "4-byte"),
    (dict(temperature=4098), 2, "4-byte"), (dict(top_k=4097), 2, "4-byte"), (dict(top_p=4098), 2, "4-byte"), (dict(min_p=4099), 2, "4-byte"),
    (dict(stride=402), 2, "stride"), (dict(stride=-400), 2, "stride"), (dict(stride=396), 1, "stride"), (dict(less=1), 1, "workspace"),
    (dict(work=None), 3, "work"), (dict(work=4224), 2, "256-byte"),
])
def test_sample_refusals(L, wrong, code, words):
    if ("less" in wrong or "work" in wrong) and L.hq_sample_work_bytes(2, 100) == 0:
        pytest.skip("no workspace is needed")
    refused(L, sample(L, **wrong), code, words)


def test_sample_work_bytes(L):
    for wrong in ((-1, 100), (2, 0), (2, (1 << 20) + 1), ((1 << 20) + 1, 5)):
        assert L.hq_sample_work_bytes(*wrong) == -1 and L.hq_last_error() == 1
    assert L.hq_sample_work_bytes(0, 100) >= 0


def test_calls_without_work(L):
    assert embed(L, out=None, count=0) == 0
    assert sample(L, tokens=None, rows=0) == 0


def test_structures_are_the_headers(pkg):
    """the ctypes structures lie as hq.h's on a 64-bit host"""
    P, T = pkg.cache.Pool, pkg.adapters.Target
    assert ctypes.sizeof(P) == 4 * 8 + 2 * 4 and P.pages.offset == 32 and P.page.offset == 36
    assert ctypes.sizeof(T) == 4 * 8 + 3 * 4 + 4 and T.y.offset == 24 and T.rows.offset == 32 and T.y_stride.offset == 40
