"""hq_attention_ex at the ends of its arguments' ranges and of what its plans are sized for."""
import numpy as np
import pytest

from gpu_util import Arena
from layer_model import F, Paged
from test_gpu_attention import check, queries

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arena():
    import torch
    assert torch.cuda.is_available(), "the GPU tests need a GPU"
    return Arena(1 << 29)


@pytest.mark.parametrize("form", ["int8", "f16"])
@pytest.mark.parametrize("new", [[9, 3], [9, 30], [200, 30]])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30 + 2 ** 25, 2 ** 30])
def test_large_windows(pkg, arena, form, new, window):
    """a window past all positions is none, also where some of a sequence's new tokens are before position 0"""
    rng = np.random.default_rng(window % 1000)
    arena.reset()
    p = Paged(pkg, arena, rng, form, 1, 64, 16, [4, 40], new)
    p.fill(rng)
    q = queries(rng, p, 4)
    got = check(p, q, window=window)
    assert np.array_equal(got.view(np.uint32), p.run_attention(q, 1 / np.sqrt(64)).view(np.uint32))
    assert (got[new[0] - 4:new[0]] != 0).any(axis=(1, 2)).all()


def attended(p, q, window=0):
    """hq_attention_ex of q with exactly the workspace it asks for, of any content, and bytes behind it that nobody may touch"""
    lib, heads, arena = p.pkg.library(), q.shape[1], p.arena
    stride = 4 * heads * p.dim
    aq, ao = arena.put(q), arena.put(np.full_like(q, -5))
    need = lib.hq_attention_work_bytes(p.cache, p.batch, heads)
    assert need > 0
    work = arena.alloc(need + 4096, fill=np.full(need + 4096, 0x7f, np.uint8))
    assert lib.hq_attention_ex(ao, aq, heads, stride, stride, p.cache, p.batch, 1 / np.sqrt(p.dim), window, 0.0, work, need,
                               None) == 0, lib.hq_last_error_message()
    got = arena.get(ao, F, q.size).reshape(q.shape)
    assert (arena.get(work + need, np.uint8, 4096) == 0x7f).all(), "wrote behind the workspace"
    return got


def empty_places(sequences):
    """some sequences without new tokens, among them the last and first of a plan's 1024"""
    return [0 if i in (0, 5, 1022, 1023, 1024, 1025, sequences - 1) or i % 17 == 3 else 1 for i in range(sequences)]


@pytest.mark.parametrize("form, sequences, heads, kv, empty", [("int8", 1100, 8, 2, True), ("f16", 4200, 4, 1, False),
                                                               ("int8", 2049, 4, 1, True)])
def test_more_sequences_than_a_plan_holds_at_once(pkg, arena, form, sequences, heads, kv, empty):
    """a token each of more than 1024 sequences, `longest` not known: planned in the workspace, 1024 at a time"""
    rng = np.random.default_rng(sequences)
    arena.reset()
    new = empty_places(sequences) if empty else [1] * sequences
    p = Paged(pkg, arena, rng, form, kv, 16, 16, [int(rng.integers(1, 70)) for _ in range(sequences)], new)
    p.fill(rng)
    q = queries(rng, p, heads)
    got = attended(p, q)
    want, far = p.attention(q, 1 / np.sqrt(16))
    assert (np.abs(got - want) <= far).all()


def test_more_tiles_than_a_plan_holds_at_once(pkg, arena):
    """2100 tokens of 256 query heads over one of keys: 4200 tiles of 128 rows, more than the plan keeps beside it"""
    rng = np.random.default_rng(3)
    arena.reset()
    p = Paged(pkg, arena, rng, "int8", 1, 16, 16, [900, 77, 1300], [900, 1, 1199])
    p.fill(rng)
    q = queries(rng, p, 256)
    got = attended(p, q, window=8)
    held = {s: p.vectors(s, range(n)) for s, n in enumerate(p.lengths)}
    for t, s, position in p.positions():  # (the formula and the bound of layer_model.Paged.attention, all heads at once)
        seen = slice(max(0, position - 7), position + 1)
        k, v = held[s][0][seen, 0], held[s][1][seen, 0]
        a = q[t].astype(np.float64) @ k.T * float(F(0.25))
        size = (np.abs(q[t].astype(np.float64)) @ np.abs(k).T).max(1) * 0.25
        e = np.exp(a - a.max(1, keepdims=True))
        want = e @ v / e.sum(1, keepdims=True)
        ds = size * (2.0 ** -21 + 4 * 2.0 ** -23) + np.abs(a).max(1) * 2.0 ** -22
        far = np.abs(v).max() * (2 * ds + 2.0 ** -20 + np.sqrt(len(v)) * 2.0 ** -22)
        assert (np.abs(got[t] - want) <= far[:, None]).all(), f"token {t}"


@pytest.mark.parametrize("form", ["int8", "f16"])
@pytest.mark.parametrize("new", [1, 3])
def test_few_rows_past_32_bits(pkg, arena, form, new):
    """single tokens and a few over pages that lie past 4 GiB, and past 2^32 elements"""
    import torch
    rng = np.random.default_rng(9)
    arena.reset()
    heads, dim, page = 8, 128, 64
    pages = (1 << 32) // (heads * page * dim) + 40
    kind = torch.int8 if form == "int8" else torch.float16
    k = torch.empty(pages * heads * page * dim, dtype=kind, device="cuda:0")
    v = torch.empty_like(k)
    ks = torch.empty(pages * heads * page, dtype=torch.float32, device="cuda:0")
    vs = torch.empty_like(ks)
    small = Paged(pkg, arena, rng, form, heads, dim, page, [150], [150])
    far_table = np.full_like(small.table, -1)
    far_table[0, :3] = pages - 1 - np.arange(3) * 7
    table, lengths = arena.put(far_table), small.batch.lengths
    lib = pkg.library()
    cache = pkg.cache.Cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), small.cache.form, pages, page, heads, dim)
    x = rng.standard_normal((2, 150, heads, dim)).astype(F)
    row = 4 * heads * dim
    batch = pkg.cache.Batch(small.batch.starts, lengths, table, 1, 150, 0, small.width)
    assert lib.hq_cache_write_ex(cache, batch, arena.put(x[0]), arena.put(x[1]), row, row, None) == 0
    for t, s, position in small.positions():
        small.put(s, position, x[0, t], x[1, t])
    small.new, small.starts, small.tokens = [new], np.array([0, new], np.int32), new
    q = queries(rng, small, 16)
    batch = pkg.cache.Batch(arena.put(small.starts), lengths, table, 1, new, new, small.width)
    aq, ao = arena.put(q), arena.put(np.zeros_like(q))
    need = lib.hq_attention_work_bytes(cache, batch, 16)
    work = arena.alloc(max(need, 256))
    assert lib.hq_attention_ex(ao, aq, 16, 2 * row, 2 * row, cache, batch, 0.1, 0, 0.0, work, need, None) == 0
    got = arena.get(ao, F, q.size).reshape(q.shape)
    want, bound = small.attention(q, 0.1)
    assert (np.abs(got - want) <= bound).all()
