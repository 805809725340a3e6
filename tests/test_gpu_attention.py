"""hq_attention_ex against the formula in 64 bits (layer_model.Paged.attention, which also says how far a float32 kernel may
be from it), over forms, head layouts, lengths, windows, caps, ragged batches and places that nobody may look at."""
import ctypes

import numpy as np
import pytest

from gpu_util import Arena
from layer_model import F, Paged

pytestmark = pytest.mark.gpu
FORMS = ["int8", "f16"]


@pytest.fixture(scope="module")
def arena():
    import torch
    assert torch.cuda.is_available(), "the GPU tests need a GPU"
    return Arena(1 << 29)


def check(p, q, window=0, cap=0.0, pad=0, scale=None):
    scale = scale or 1 / np.sqrt(p.dim)
    got = p.run_attention(q, scale, window, cap, pad)
    want, far = p.attention(q, scale, window, cap)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    off = np.where(nan, 0, np.abs(got - np.where(nan, 0, want)))
    worst = np.unravel_index(np.argmax(off - np.where(nan, 0, far)), off.shape)
    assert (off <= np.where(nan, 0, far)).all(), f"at {worst}: {got[worst]!r}, {want[worst]!r} +- {far[worst]!r}"
    return got


def queries(rng, p, heads, size=2.0):
    return (rng.standard_normal((p.tokens, heads, p.dim)) * size).astype(F)


# head layouts: one head, several alone, shared by 2, 4, 5, 6, 16 and 20 query heads
LAYOUTS = [(1, 1, 16), (6, 6, 48), (16, 4, 64), (4, 2, 80), (6, 2, 96), (8, 2, 128), (10, 2, 128), (16, 1, 112), (12, 2, 256),
           (20, 1, 32)]
# one token after 0, 1, 2, 63 .. positions; a few; prompts from the start and on top of others; a ragged batch
BATCHES = [([1], [1]), ([2, 1, 64, 65], [1, 1, 1, 1]), ([257, 16, 600], [1, 1, 1]), ([40, 300], [5, 3]), ([70], [70]),
           ([333, 9, 130, 64, 200], [60, 1, 0, 130, 17])]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads, kv, dim", LAYOUTS)
@pytest.mark.parametrize("lengths, new", BATCHES)
def test_attention(pkg, arena, form, heads, kv, dim, lengths, new):
    rng = np.random.default_rng(dim * heads + sum(lengths))
    arena.reset()
    page = [16, 32, 64, 128, 256][(dim + len(new)) % 5]
    p = Paged(pkg, arena, rng, form, kv, dim, page, lengths, new)
    p.fill(rng)
    check(p, queries(rng, p, heads), pad=16 * (dim % 3))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 5000])
def test_window(pkg, arena, form, page, window):
    rng = np.random.default_rng(window)
    arena.reset()
    p = Paged(pkg, arena, rng, form, 2, 64, page, [700, 130, 90], [1, 100, 3])
    p.fill(rng)
    check(p, queries(rng, p, 4), window=window)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("cap", [0.5, 30.0])
@pytest.mark.parametrize("window", [0, 40])
def test_cap(pkg, arena, form, cap, window):
    rng = np.random.default_rng(2)
    arena.reset()
    p = Paged(pkg, arena, rng, form, 1, 128, 32, [300, 90], [1, 50])
    p.fill(rng)
    check(p, queries(rng, p, 6, size=6.0), window=window, cap=cap)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("gone_as", [-1, -2 ** 31, 10 ** 6])
def test_rows_that_see_nothing(pkg, arena, form, gone_as):
    """pages given back, new tokens before position 0, a sequence without positions: zeros where nothing is seen, and what is
    not seen (NaN here) shows nowhere"""
    rng = np.random.default_rng(3)
    arena.reset()
    gone = [(0, i) for i in range(12)] + [(1, 2), (1, 3), (1, 4)] + [(3, i) for i in range(4)]
    p = Paged(pkg, arena, rng, form, 2, 64, 16, [200, 120, 4, 60, 0, 30], [1, 70, 9, 40, 3, 1], gone=gone, gone_as=gone_as)
    p.fill(rng)
    q = queries(rng, p, 6)
    got = check(p, q)
    assert (got[0] != 0).any()  # (8 positions on its last page)
    assert (got[71:76] == 0).all() and (got[80:120] == 0).all() and (got[120:123] == 0).all()
    got = check(p, q, window=8)
    assert (got[80:120] == 0).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new", [1, 6, 90])
def test_nan_is_seen_by_who_sees_it(pkg, arena, form, new):
    """a key or value of infinities or NaN makes NaN of every token that sees it and of no other"""
    rng = np.random.default_rng(4)
    for which, bad in (("k", np.nan), ("v", np.inf), ("v", np.nan)):
        arena.reset()
        p = Paged(pkg, arena, rng, form, 2, 64, 16, [150, 150], [new, new])
        p.fill(rng)
        at = 150 - new + new // 2
        page, slot = p.place(0, at)
        vector = np.zeros((2, 64), F)
        vector[1, 5] = bad
        good = np.ones((2, 64), F)
        p.put(0, at, vector if which == "k" else good, vector if which == "v" else good)
        p.send()
        got = check(p, queries(rng, p, 4))
        assert np.isnan(got[new // 2:new, 2:]).all() and not np.isnan(got[:new // 2]).any()
        assert not np.isnan(got[:, :2]).any() and not np.isnan(got[new:]).any()


@pytest.mark.parametrize("form", FORMS)
def test_hard_values(pkg, arena, form):
    """scores far apart (one position takes all, early or late), equal scores, values of very different sizes, zeros, keys and
    queries near the ends of float32"""
    rng = np.random.default_rng(5)
    for sharp, at in ((200.0, 3), (200.0, 290), (0.0, 0)):
        arena.reset()
        p = Paged(pkg, arena, rng, form, 1, 64, 32, [300, 300], [1, 40])
        p.fill(rng)
        q = queries(rng, p, 4)
        for s in range(2):
            k, v, _ = p.vectors(s, [at])
            p.put(s, at, (np.sign(k[0]) * 3).astype(F), (v[0] * 1e-6).astype(F))  # (its values tiny, as a sink's)
        p.send()
        check(p, q * F(sharp / 20) if sharp else q * F(0))
    arena.reset()
    p = Paged(pkg, arena, rng, form, 1, 64, 32, [300, 300], [1, 40])
    p.fill(rng)
    for s in range(2):
        for j in range(300):
            k, v, _ = p.vectors(s, [j])
            size = 10.0 ** rng.integers(-25, 25)
            p.put(s, j, k[0].astype(F) * F(1e15), (v[0] * (0 if j % 7 == 0 else size)).astype(F))
    p.send()
    check(p, queries(rng, p, 2) * F(1e-15))
    p.v[:], p.k[:] = 0, 0
    p.vs[:], p.ks[:] = 0, 0
    p.send()
    assert (check(p, queries(rng, p, 2)) == 0).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lengths, new, heads, kv, dim", [([5000, 1], [1, 1], 8, 2, 128), ([3001] * 9, [1] * 9, 8, 2, 64),
                                                          ([2600, 700], [300, 1], 4, 1, 64), ([4097], [4], 4, 1, 256),
                                                          ([700] * 70, [1] * 70, 2, 1, 32)])
def test_long(pkg, arena, form, lengths, new, heads, kv, dim):
    """positions that several workgroups share, and more sequences than a wave has lanes"""
    rng = np.random.default_rng(6)
    arena.reset()
    p = Paged(pkg, arena, rng, form, kv, dim, 64, lengths, new)
    p.fill(rng)
    q = queries(rng, p, heads)
    got = check(p, q)
    assert np.array_equal(got.view(np.uint32), p.run_attention(q, 1 / np.sqrt(dim)).view(np.uint32)), "runs differ"


@pytest.mark.parametrize("form", FORMS)
def test_longest_is_a_hint(pkg, arena, form):
    """whatever `longest` says, the numbers hold, also where it is wrong"""
    for longest in (1, 2, 33, 60, 1000):
        rng = np.random.default_rng(7)
        arena.reset()
        p = Paged(pkg, arena, rng, form, 2, 64, 32, [333, 9, 130, 64], [60, 1, 0, 33], longest=longest)
        p.fill(rng)
        check(p, queries(rng, p, 8))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim, new", [(64, [12, 3]), (64, [13, 3]), (128, [24, 1]), (128, [25, 1]), (256, [4, 24]), (256, [4, 25])])
@pytest.mark.parametrize("lengths, width", [([140, 90], 0), ([140, 90], 60), ([1500, 700], 0)])
def test_few_rows_or_many(pkg, arena, form, dim, new, lengths, width):
    """on either side of what decides how rows are tiled, and whether a block has a tile's positions whole"""
    rng = np.random.default_rng(dim + sum(new))
    arena.reset()
    p = Paged(pkg, arena, rng, form, 2, dim, 64, lengths, new, extra_width=width, longest=max(new))
    p.fill(rng)
    check(p, queries(rng, p, 8))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("sequences, longest, dim", [(20, 900, 64), (32, 1900, 128), (33, 1000, 64)])
def test_many_sequences(pkg, arena, form, sequences, longest, dim):
    """a token each of many sequences of all lengths, with 8 heads of keys: a block a tile from as many on as the GPU has
    compute units"""
    rng = np.random.default_rng(sequences)
    arena.reset()
    lengths = [1 + i * (longest - 1) // (sequences - 1) for i in range(sequences)]
    p = Paged(pkg, arena, rng, form, 8, dim, 64, lengths, [1] * sequences, extra_width=0, longest=1)
    p.fill(rng)
    check(p, queries(rng, p, 8 if dim == 128 else 16))


@pytest.mark.parametrize("starts", [[0, 5, 3, 9], [-4, 2, 100, 9], [3, 3, 8, 9], [0, 9, 0, 9]])
@pytest.mark.parametrize("longest", [0, 1])
def test_contradicting_starts(pkg, arena, starts, longest):
    """starts that fall, start below 0 or pass the tokens' end write nothing outside the rows and the workspace (numbers undefined)"""
    rng = np.random.default_rng(1)
    arena.reset()
    p = Paged(pkg, arena, rng, "int8", 1, 32, 16, [300, 20, 300], [3, 3, 3], longest=longest)
    p.fill(rng)
    arena.write(p.batch.starts, np.asarray(starts, np.int32))
    lib, heads = pkg.library(), 30
    q = arena.put(queries(rng, p, heads))
    guards = [arena.put(np.full(4096, 77, np.uint8))]
    out = arena.alloc(9 * heads * 128)
    guards.append(arena.put(np.full(4096, 77, np.uint8)))
    need = lib.hq_attention_work_bytes(p.cache, p.batch, heads)
    work = arena.alloc(need)
    guards.append(arena.put(np.full(4096, 77, np.uint8)))
    assert lib.hq_attention_ex(out, q, heads, heads * 128, heads * 128, p.cache, p.batch, 0.1, 0, 0.0, work, need, None) == 0
    for at in guards:
        assert (arena.get(at, np.uint8, 4096) == 77).all()


@pytest.mark.parametrize("new", [1, 40])
def test_no_pages(pkg, arena, new):
    """a cache without pages (its pointers NULL): zeros, and nothing is read"""
    rng = np.random.default_rng(1)
    arena.reset()
    p = Paged(pkg, arena, rng, "f16", 2, 64, 16, [50, 60], [new, new])
    p.cache.pages, p.cache.k, p.cache.v, p.cache.ks, p.cache.vs = 0, None, None, None, None
    assert (p.run_attention(queries(rng, p, 8), 0.1) == 0).all()


def test_stream_and_graph(pkg, arena):
    """another stream than torch's, and a captured step (write, attention) replayed with other lengths and inputs, each replay
    against the eager call"""
    import torch
    rng = np.random.default_rng(8)
    arena.reset()
    lib = pkg.library()
    assert lib.hq_init() == 0
    p = Paged(pkg, arena, rng, "int8", 2, 64, 16, [400, 90, 33], [1, 1, 1], extra_width=4)
    p.fill(rng)
    heads = 8
    aq, ao = arena.put(np.zeros((3, heads, 64), F)), arena.put(np.zeros((3, heads, 64), F))
    ak = arena.put(np.zeros((3, 2, 64), F))
    need = lib.hq_attention_work_bytes(ctypes.byref(p.cache), ctypes.byref(p.batch), heads)
    work = arena.alloc(max(need, 256), fill=np.full(max(need, 256), 0xff, np.uint8))
    stream = torch.cuda.Stream()

    def step():
        h = stream.cuda_stream
        assert lib.hq_cache_write_ex(ctypes.byref(p.cache), ctypes.byref(p.batch), ak, ak, 512, 512, h) == 0
        assert lib.hq_attention_ex(ao, aq, heads, 2048, 2048, ctypes.byref(p.cache), ctypes.byref(p.batch), 0.125, 0, 0.0,
                                   work, need, h) == 0

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step()
    for replay in range(4):
        p.lengths = [400 - 90 * replay, 90 + replay, 33 + replay]  # (on pages that the sequences have)
        arena.write(p.batch.lengths, np.asarray(p.lengths, np.int32))
        k = rng.standard_normal((3, 2, 64)).astype(F)
        q = (rng.standard_normal((3, heads, 64)) * 2).astype(F)
        arena.write(ak, k)
        arena.write(aq, q)
        for t, s, position in p.positions():
            p.put(s, position, k[t], k[t])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = arena.get(ao, F, 3 * heads * 64).reshape(3, heads, 64)
        want, far = p.attention(q, 0.125)
        nan = np.isnan(want)
        assert np.array_equal(nan, np.isnan(got)) and (np.abs(got - want)[~nan] <= far[~nan]).all(), f"replay {replay}"
        eager = p.run_attention(q, 0.125)
        assert np.array_equal(eager.view(np.uint32), got.view(np.uint32)), f"replay {replay} and the eager call"


def test_offsets_past_32_bits(pkg, arena):
    """a pool whose last pages lie past 4 GiB: written, attended to and read back there"""
    import torch
    rng = np.random.default_rng(9)
    arena.reset()
    heads, dim, page = 8, 128, 64
    pages = (1 << 32) // (heads * page * dim) + 40
    k = torch.empty(pages * heads * page * dim, dtype=torch.int8, device="cuda:0")
    v = torch.empty_like(k)
    ks = torch.empty(pages * heads * page, dtype=torch.float32, device="cuda:0")
    vs = torch.empty_like(ks)
    small = Paged(pkg, arena, rng, "int8", heads, dim, page, [150], [150])
    far = np.full_like(small.table, -1)
    far[0, :3] = pages - 1 - np.arange(3) * 7
    at = arena.put(far)
    lib = pkg.library()
    cache = pkg.cache.Cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), 0, pages, page, heads, dim)
    batch = pkg.cache.Batch(small.batch.starts, small.batch.lengths, at, 1, 150, 0, small.width)
    x = rng.standard_normal((2, 150, heads, dim)).astype(F)
    row = 4 * heads * dim
    ak, av = arena.put(x[0]), arena.put(x[1])
    assert lib.hq_cache_write_ex(ctypes.byref(cache), ctypes.byref(batch), ak, av, row, row, None) == 0
    for t, s, position in small.positions():
        small.put(s, position, x[0, t], x[1, t])
    q = queries(rng, small, 16)
    aq, ao = arena.put(q), arena.put(np.zeros_like(q))
    need = lib.hq_attention_work_bytes(ctypes.byref(cache), ctypes.byref(batch), 16)
    work = arena.alloc(max(need, 256))
    assert lib.hq_attention_ex(ao, aq, 16, 2 * row, 2 * row, ctypes.byref(cache), ctypes.byref(batch), 0.1, 0, 0.0, work, need,
                               None) == 0
    got = arena.get(ao, F, q.size).reshape(q.shape)
    want, bound = small.attention(q, 0.1)
    assert (np.abs(got - want) <= bound).all()
    back = [arena.put(np.zeros((150, heads, dim), F)) for _ in range(2)]
    assert lib.hq_cache_read_ex(ctypes.byref(cache), ctypes.byref(batch), *back, row, row, None) == 0
    kk, vv, _ = small.vectors(0, range(150))
    for a, w in zip(back, (kk, vv)):
        assert np.array_equal(arena.get(a, F, w.size).reshape(w.shape), w.astype(F))
