"""hq_embed_ex against the packings' readers (tests' own packers, the oracle's block reader), to the bit."""
import numpy as np
import pytest

import blocks_model as bm
from gpu_util import Arena, first_difference, same_bits
from streams import pack6, pack_binary, pack_ternary

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.fixture(scope="module")
def arena():
    import torch
    assert torch.cuda.is_available(), "the GPU tests need a GPU"
    return Arena(1 << 27)


def table(rng, packing, vocab, dim):
    """(the values' bytes, the scales, the float32 weights before the caller's scale)"""
    count = vocab * dim
    if packing == "int8":
        group = min(32, dim & -dim)
        v = rng.integers(-128, 128, count).astype(np.int8)
        scales, values = (rng.random(count // group) * 0.01).astype(F), v
    elif packing == "int6":
        v = (4 * rng.integers(-32, 32, count)).astype(np.int8)
        group, scales, values = 32, (rng.random(count // 32) * 0.01).astype(F), pack6(v)
    else:
        group = 128
        scales = (rng.random(count // 128) * 0.01 + 1e-3).astype(np.float16)
        if packing == "ternary":
            codes = rng.integers(0, 4, count).astype(np.uint8)
            v, values = codes.astype(np.int8) - 1, pack_ternary(codes)
        else:
            bits = rng.integers(0, 2, count).astype(np.uint8)
            v, values = 2 * bits.astype(np.int8) - 1, pack_binary(bits, dim)
    wide = scales.astype(F)
    return values, scales, (v.reshape(-1, group).astype(F) * wide[:, None]).reshape(vocab, dim)


def run(pkg, arena, ids, values, scales, packing, vocab, dim, scale=1.0, pad=0, stream=None):
    lib = pkg.library()
    out = arena.put(np.full((max(1, len(ids)), dim + pad), -7, F))
    status = lib.hq_embed_ex(out, arena.put(np.asarray(ids, np.int32)), values, scales, packing, vocab, dim, scale, len(ids),
                             4 * (dim + pad), stream)
    assert status == 0, lib.hq_last_error_message()
    got = arena.get(out, F, max(1, len(ids)) * (dim + pad)).reshape(-1, dim + pad)
    assert (got[:, dim:] == -7).all(), "wrote between the rows"
    return got[:len(ids), :dim]


def wanted(rows, ids, scale):
    want = (rows * F(scale)).astype(F)
    return np.stack([want[i] if 0 <= i < len(want) else np.zeros_like(want[0]) for i in ids])


@pytest.mark.parametrize("packing, dim", [
    ("int8", 32), ("int8", 288), ("int8", 4096), ("int8", 1056), ("int8", 48), ("int8", 36), ("int6", 32), ("int6", 288),
    ("int6", 2080), ("ternary", 128), ("ternary", 2176), ("binary", 128), ("binary", 640), ("binary", 4096)])
@pytest.mark.parametrize("count, scale, pad", [(1, 1.0, 0), (5, 16.97, 4), (67, 0.125, 0)])
def test_rows(pkg, arena, packing, dim, count, scale, pad):
    rng = np.random.default_rng(dim + count)
    arena.reset()
    vocab = 37
    values, scales, rows = table(rng, packing, vocab, dim)
    av, asc = arena.put(values), arena.put(scales)
    ids = rng.integers(0, vocab, count)
    ids[0] = vocab - 1
    if count > 4:
        ids[1:5] = (0, -1, vocab, -2 ** 31)
    got = run(pkg, arena, ids, av, asc, pkg.HQ_PACK[packing], vocab, dim, scale, pad)
    want = wanted(rows, ids, scale)
    assert same_bits(got, want), first_difference(got, want)


@pytest.mark.parametrize("dim", [1, 3, 27, 30, 33])
def test_int8_rows_of_odd_lengths(pkg, arena, dim):
    """groups of 1 and 2 (the row's largest power of two): rows that begin anywhere"""
    rng = np.random.default_rng(dim)
    arena.reset()
    values, scales, rows = table(rng, "int8", 50, dim)
    ids = rng.integers(0, 50, 20)
    pad = -dim % 4
    got = run(pkg, arena, ids, arena.put(values), arena.put(scales), 0, 50, dim, 3.0, pad)
    assert same_bits(got, wanted(rows, ids, 3.0))


@pytest.mark.parametrize("name", sorted(bm.TYPES))
@pytest.mark.parametrize("dim, count, off", [(256, 1, 0), (1280, 9, 2), (4096, 3, 0)])
def test_block_types(pkg, oracle, arena, name, dim, count, off):
    rng = np.random.default_rng(dim)
    arena.reset()
    kind, vocab = bm.TYPES[name], 11
    raw = bm.random_blocks(rng, kind, vocab * dim // 256)
    books = bm.codebooks(rng)
    tables = arena.alloc(34992)
    assert pkg.load_kernels().sb_tables(tables, arena.put(books)) == 34992
    at = arena.alloc(raw.size + off) + off
    arena.write(at, raw)
    ids = rng.integers(0, vocab, count)
    ids[-1] = vocab - 1
    if count > 3:
        ids[0], ids[1] = vocab, -1
    got = run(pkg, arena, ids, at, tables, pkg.HQ_PACK_BLOCKS + kind, vocab, dim, 2.5)
    area = oracle.sb_tables(books)
    flat = np.ascontiguousarray(raw).reshape(vocab, -1)
    rows = np.stack([oracle.sb_row(flat[v], area, dim, kind) for v in range(vocab)])
    want = wanted(rows, ids, 2.5)
    assert same_bits(got, want), first_difference(got, want)


def test_infinite_and_subnormal_scales(pkg, arena):
    rng = np.random.default_rng(3)
    arena.reset()
    v = rng.integers(-128, 128, 4 * 64).astype(np.int8)
    scales = np.array([np.inf, 1e-42, 0.0, np.nan, -1.0, 3e38, 1e-38, 1.0], F)
    got = run(pkg, arena, [0, 1, 2, 3], arena.put(v), arena.put(scales), 0, 4, 64, 4.0)
    with np.errstate(all="ignore"):
        want = ((v.reshape(-1, 32).astype(F) * scales[:, None]) * F(4)).reshape(4, 64)
    assert np.array_equal(got, want, equal_nan=True)


def test_tables_past_4_gib(pkg):
    """the last rows of a table that 32 bits cannot address, by bytes of its values"""
    import torch
    lib, vocab, dim = pkg.library(), 1100000, 4096
    values = torch.zeros(vocab, dim, dtype=torch.int8, device="cuda")
    scales = torch.ones(vocab, dim // 32, device="cuda")
    values[-3:] = torch.arange(3 * dim, device="cuda").view(3, dim).remainder(251).sub(125).to(torch.int8)
    scales[-3:] = torch.rand(3, dim // 32, device="cuda")
    ids = torch.tensor([vocab - 1, vocab - 3, vocab, 0, vocab - 2], dtype=torch.int32, device="cuda")
    out = torch.empty(5, dim, device="cuda")
    torch.cuda.synchronize()
    assert lib.hq_embed_ex(out.data_ptr(), ids.data_ptr(), values.data_ptr(), scales.data_ptr(), 0, vocab, dim, 1.0, 5, 4 * dim,
                           torch.cuda.current_stream().cuda_stream) == 0
    for row, at in ((0, vocab - 1), (1, vocab - 3), (4, vocab - 2)):
        assert torch.equal(out[row], values[at].float() * scales[at].repeat_interleave(32))
    assert not out[2].any() and not out[3].any()


def test_many_rows(pkg, arena):
    """more rows than a grid's second dimension"""
    rng = np.random.default_rng(8)
    arena.reset()
    values, scales, rows = table(rng, "int8", 97, 32)
    ids = rng.integers(0, 97, 70001)
    got = run(pkg, arena, ids, arena.put(values), arena.put(scales), 0, 97, 32)
    assert same_bits(got, rows[ids])


def test_replayed(pkg, arena):
    """captured on a stream of its own, replayed with other ids"""
    import torch
    lib, rng = pkg.library(), np.random.default_rng(9)
    assert lib.hq_init() == 0
    arena.reset()
    values, scales, rows = table(rng, "ternary", 64, 256)
    av, asc, aid, out = arena.put(values), arena.put(scales), arena.put(np.zeros(7, np.int32)), arena.alloc(7 * 1024)
    torch.cuda.synchronize()
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        status = lib.hq_embed_ex(out, aid, av, asc, 2, 64, 256, 1.5, 7, 1024, stream.cuda_stream)
    assert status == 0
    for _ in range(3):
        ids = rng.integers(0, 64, 7)
        arena.write(aid, ids.astype(np.int32))
        torch.cuda.synchronize()
        g.replay()
        assert same_bits(arena.get(out, F, 7 * 256).reshape(7, 256), wanted(rows, ids, 1.5))


@pytest.mark.parametrize("dim", [2 ** 31 - 1, 2 ** 31 - 4])
def test_rows_as_long_as_can_be(pkg, dim):
    """a row that ends less than a block's values before 2^31, a weight and four a thread"""
    import torch
    group, guard = dim & -dim, 1024
    values = torch.randint(-128, 128, (dim + -dim % 16,), dtype=torch.int8, device="cuda")
    scales = torch.rand(dim // group, device="cuda")
    memory = torch.full((dim + 2 * guard,), -7.0, device="cuda")
    out, ids = memory[guard:], torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    lib = pkg.library()
    assert lib.hq_embed_ex(out.data_ptr(), ids.data_ptr(), values.data_ptr(), scales.data_ptr(), 0, 1, dim, 0.5, 1, 0, None) == 0, \
        lib.hq_last_error_message()
    torch.cuda.synchronize()
    assert (memory[:guard] == -7).all() and (memory[-guard:] == -7).all()
    for at in range(0, dim, 1 << 28):
        end = min(at + (1 << 28), dim)
        want = values[at:end].float().view(-1, group) * scales[at // group:end // group, None] * 0.5
        assert torch.equal(out[at:end], want.view(-1))
