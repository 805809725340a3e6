"""hq_cache_write_ex and hq_cache_read_ex: every byte of the cache against a plain quantizer, what is not new left as it was,
and the vectors read back exactly."""
import ctypes

import numpy as np
import pytest

from gpu_util import Arena, same_bits
from layer_model import F, Paged, quantized

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arena():
    import torch
    assert torch.cuda.is_available(), "the GPU tests need a GPU"
    return Arena(1 << 28)


def write(p, k, v, pad=0):
    lib = p.pkg.library()
    row = p.heads * p.dim
    wide = [np.full((max(1, p.tokens), row + extra), 9, F) for extra in (pad, 2 * pad)]
    for a, x in zip(wide, (k, v)):
        a[:p.tokens, :row] = x.reshape(p.tokens, row)
    ak, av = (p.arena.put(a) for a in wide)
    status = lib.hq_cache_write_ex(ctypes.byref(p.cache), ctypes.byref(p.batch), ak, av, *(4 * a.shape[1] for a in wide), None)
    assert status == 0, lib.hq_last_error_message()
    for t, s, position in p.positions():
        p.put(s, position, k[t], v[t])


def read(p):
    lib = p.pkg.library()
    row = p.heads * p.dim
    at = [p.arena.put(np.full((max(1, p.tokens), row), -4, F)) for _ in range(2)]
    status = lib.hq_cache_read_ex(ctypes.byref(p.cache), ctypes.byref(p.batch), *at, 4 * row, 4 * row, None)
    assert status == 0, lib.hq_last_error_message()
    return [p.arena.get(a, F, max(1, p.tokens) * row).reshape(-1, p.heads, p.dim)[:p.tokens] for a in at]


def check(p):
    for name in ("k", "v", "ks", "vs"):
        got, want = p.fetch(name), getattr(p, name)
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8)), \
            f"{name}: {np.argwhere(got.view(np.uint8) != want.view(np.uint8))[:3]}"


def check_read(p):
    k, v = read(p)
    for t, s, position in p.positions():
        at = p.place(s, position)
        for got, want in ((k[t], None if at is None else (p.k[at[0], :, at[1]].astype(F) * p.ks[at[0], :, at[1], None])),
                          (v[t], None if at is None else (p.v[at[0], :, :, at[1]].astype(F) * p.vs[at[0], :, at[1], None]))):
            want = np.zeros_like(got) if want is None else want
            assert np.array_equal(np.isnan(got), np.isnan(want))
            assert same_bits(np.nan_to_num(got), np.nan_to_num(want)), f"token {t}"


BATCHES = [([1], [1]), ([200], [1]), ([65], [65]), ([300, 17, 64, 129], [300, 1, 0, 100]), ([5, 700, 128], [2, 650, 128]),
           ([33] * 70, [1] * 70)]


@pytest.mark.parametrize("form", ["int8", "f16"])
@pytest.mark.parametrize("heads, dim, page", [(1, 16, 16), (6, 48, 32), (2, 128, 64), (3, 80, 128), (2, 256, 256)])
@pytest.mark.parametrize("lengths, new", BATCHES)
def test_write_and_read(pkg, arena, form, heads, dim, page, lengths, new):
    rng = np.random.default_rng(dim + sum(new))
    arena.reset()
    p = Paged(pkg, arena, rng, form, heads, dim, page, lengths, new)
    k, v = (rng.standard_normal((p.tokens, heads, dim)).astype(F) * s for s in (3, 0.1))
    write(p, k, v, pad=4)
    check(p)
    check_read(p)


@pytest.mark.parametrize("form", ["int8", "f16"])
def test_places_without_a_page(pkg, arena, form):
    """new tokens before position 0, on entries that are no page and past the table: nothing is written, zeros are read"""
    rng = np.random.default_rng(5)
    for gone_as in (-1, -2 ** 31, 2 ** 31 - 1, 1000):
        arena.reset()
        p = Paged(pkg, arena, rng, form, 2, 32, 16, [40, 3, 90], [40, 8, 60], gone=[(0, 1), (2, 2), (2, 5)], gone_as=gone_as)
        k, v = (rng.standard_normal((p.tokens, 2, 32)).astype(F) for _ in range(2))
        write(p, k, v)
        check(p)
        check_read(p)
    arena.reset()
    p = Paged(pkg, arena, rng, form, 2, 32, 16, [64, 64], [64, 64], extra_width=-1)  # positions 48.. are past the table
    write(p, *(rng.standard_normal((p.tokens, 2, 32)).astype(F) for _ in range(2)))
    check(p)
    check_read(p)


@pytest.mark.parametrize("form", ["int8", "f16"])
def test_hard_vectors(pkg, arena, form):
    """zeros, subnormals, scales at the smallest, the largest numbers, infinities and NaN; a vector's neighbours are not touched"""
    rng = np.random.default_rng(6)
    arena.reset()
    p = Paged(pkg, arena, rng, form, 1, 64, 16, [24], [24])
    k = rng.standard_normal((24, 1, 64)).astype(F)
    sizes = [0, 1e-45, 1e-38, 2.0 ** -100, 127 * 2.0 ** -100, 2.0 ** -93, 2.0 ** -86, 1e-20, 65504, 1e10, 3e38]
    for i, size in enumerate(sizes):
        with np.errstate(all="ignore"):
            k[i] = np.clip(k[i] / np.abs(k[i]).max(), -1, 1) * F(size)
    k[11, 0, 3], k[12, 0, 0], k[13, 0, 63] = np.inf, -np.inf, np.nan
    k[14], k[15] = np.inf, np.nan
    k[16] = np.arange(64, dtype=F) - 31.5  # halves: ties to even
    k[17, 0] = 0
    k[17, 0, 5] = 1.5
    write(p, k, k[::-1].copy())
    check(p)
    check_read(p)


def test_int8_is_quantize_x(pkg, arena, oracle):
    """a head of 32 values is a group of quantize_x's: the same bytes and scales"""
    rng = np.random.default_rng(7)
    arena.reset()
    p = Paged(pkg, arena, rng, "int8", 4, 32, 16, [50], [50])
    k = rng.standard_normal((50, 4, 32)).astype(F)
    write(p, k, k)
    for t, s, position in p.positions():
        page, slot = p.place(s, position)
        q, scales = oracle.quantize_x(k[t].reshape(-1), 0)
        assert np.array_equal(p.fetch("k")[page, :, slot].reshape(-1), np.asarray(q).view(np.int8))
        assert same_bits(p.fetch("ks")[page, :, slot], scales)


def test_quantized_is_near():
    """(the model itself) an int8's value is within half a step of the vector's, a float16's within 2^-11 of itself"""
    x = np.random.default_rng(8).standard_normal((100, 64)).astype(F)
    e, s = quantized(x, "int8")
    assert (np.abs(e * s[:, None] - x) <= 0.5001 * s[:, None]).all()
    e, s = quantized(x, "f16")
    assert (np.abs(e.astype(F) * s[:, None] - x) <= np.abs(x) * 2.0 ** -11 + s[:, None] * 2.0 ** -25).all()


@pytest.mark.parametrize("starts", [[0, 5, 3, 9], [-4, 2, 100, 9], [3, 3, 8, 9]])
def test_contradicting_starts(pkg, arena, starts):
    """starts that fall, start below 0 or pass the tokens' end touch nothing outside the rows and pages (numbers undefined)"""
    import torch
    rng = np.random.default_rng(1)
    arena.reset()
    p = Paged(pkg, arena, rng, "int8", 1, 32, 16, [20, 20, 20], [3, 3, 3])
    arena.write(p.batch.starts, np.asarray(starts, np.int32))
    lib = pkg.library()
    a = arena.put(np.ones((9, 32), F))
    guard = arena.put(np.full(4096, 77, np.uint8))
    assert lib.hq_cache_write_ex(ctypes.byref(p.cache), ctypes.byref(p.batch), a, a, 128, 128, None) == 0
    out = [arena.put(np.zeros((9, 32), F)) for _ in range(2)]
    after = arena.put(np.full(4096, 77, np.uint8))
    assert lib.hq_cache_read_ex(ctypes.byref(p.cache), ctypes.byref(p.batch), *out, 128, 128, None) == 0
    torch.cuda.synchronize()
    for at in (guard, after):
        assert (arena.get(at, np.uint8, 4096) == 77).all()
