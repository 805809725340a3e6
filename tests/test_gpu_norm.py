"""hq_norm_ready_ex against the formula in 64 bits and against quantize_x, interleave and sums_x of its own y, to the bit."""
import numpy as np
import pytest

import layer_model
from gpu_util import Arena, same_bits

pytestmark = pytest.mark.gpu
F = np.float32
READY = ("biased", "plain", "planes", "sums")
UNIT = {"biased": 32, "plain": 32, "planes": 128, "sums": 256}


@pytest.fixture(scope="module")
def arena():
    import torch
    assert torch.cuda.is_available(), "the GPU tests need a GPU"
    return Arena(1 << 27)


def run(pkg, arena, x, d, w, ready, eps=1e-5, pad=0, in_place=False, with_y=True, with_xq=True, with_r=True):
    """(r, y, xq, xs's bytes) of a call whose rows are `pad` floats further apart than they are long"""
    lib = pkg.library()
    t, n = x.shape
    arena.reset()

    def rows(a, fill):
        wide = np.full((t, n + pad), fill, F)
        if a is not None:
            wide[:, :n] = a
        return arena.put(wide)

    ax, aw = rows(x, 3), arena.put(w)
    ad = rows(d, 3) if d is not None else 0
    ar = (ax if in_place else rows(None, -2)) if with_r else 0
    ay = rows(None, -3) if with_y else 0
    tail = pkg.cache.READY_BYTES[ready](n)
    frame = (n + tail + 15) // 16 * 16 + 16
    acts = arena.put(np.full(t * frame, 0xA5, np.uint8)) if with_xq else 0
    stride = 4 * (n + pad)
    status = lib.hq_norm_ready_ex(acts, acts + n if with_xq else 0, ay, ar, ax, ad, aw, n, eps, pkg.cache.READY[ready], t, frame,
                                  stride, stride, stride, None)
    assert status == 0, lib.hq_last_error_message()

    def back(at):
        got = arena.get(at, F, t * (n + pad)).reshape(t, n + pad)
        assert not pad or (got[:, n:] == got[0, n]).all()
        return got[:, :n]

    r = back(ar) if with_r else None
    y = back(ay) if with_y else None
    if not with_xq:
        return r, y, None, None
    got = arena.get(acts, np.uint8, t * frame).reshape(t, frame)
    assert (got[:, n + tail:] == 0xA5).all(), "wrote past the scales"
    return r, y, got[:, :n], got[:, n:n + tail]


def check_ready(oracle, y, xq, xs, ready):
    for t in range(y.shape[0]):
        n = y.shape[1]
        q, s = oracle.quantize_x(y[t], 64 if ready == "biased" else 0)
        scales = xs[t, :n // 8].copy().view(F)
        assert same_bits(scales, s), f"token {t}: scales"
        q = np.asarray(q).view(np.int8)
        if ready == "planes":
            want = q.reshape(-1, 16, 4).transpose(0, 2, 1).reshape(-1)  # byte 16 p + c of 64 is value 4 c + p
            assert np.array_equal(xq[t].view(np.int8), want), f"token {t}: planes"
            sums = xs[t, n // 8:].copy().view(np.int32)
            assert np.array_equal(sums, -q.reshape(-1, 32).astype(np.int32).sum(1)), f"token {t}: sums"
            continue
        assert np.array_equal(xq[t].view(np.int8), q), f"token {t}: bytes"
        if ready == "sums":
            sums = xs[t, n // 8:].copy().view(np.int16)
            q = q.astype(np.int16)
            assert np.array_equal(sums, np.concatenate([q.reshape(-1, 16).sum(1), q.reshape(-1, 8).sum(1)]))


def check_norm(x, d, w, r, y, eps=1e-5):
    want_r, want_y = layer_model.norm(x, d, w, eps)
    assert r is None or same_bits(r, want_r)
    # y is the 64-bit number rounded once: another order of the sum moves it by some 2^-50 of itself, so that at most one value
    # in 2^20 or so falls on the other side of a rounding, by one step
    want = want_y.astype(F)
    off = y.view(np.int32).astype(np.int64) - want.view(np.int32)
    assert np.abs(off).max() <= 1 and np.count_nonzero(off) <= 1 + y.size // (1 << 20)


@pytest.mark.parametrize("ready", READY)
@pytest.mark.parametrize("n, tokens, pad", [(256, 1, 0), (768, 5, 4), (1280, 33, 0), (5120, 3, 16), (16640, 2, 0),
                                            (33024, 2, 4)])
def test_norm(pkg, arena, oracle, ready, n, tokens, pad):
    rng = np.random.default_rng(n + tokens)
    x = (rng.standard_normal((tokens, n)) * np.exp(rng.standard_normal(n))).astype(F)
    d = (rng.standard_normal((tokens, n)) * 0.3).astype(F)
    w = (1 + 0.3 * rng.standard_normal(n)).astype(F)
    r, y, xq, xs = run(pkg, arena, x, d, w, ready, pad=pad)
    check_norm(x, d, w, r, y)
    check_ready(oracle, y, xq, xs, ready)


@pytest.mark.parametrize("n", [32, 96, 288, 1056, 4128])
@pytest.mark.parametrize("ready", ["biased", "plain"])
def test_norm_odd_rows(pkg, arena, oracle, ready, n):
    rng = np.random.default_rng(n)
    x, d = (rng.standard_normal((7, n)).astype(F) for _ in range(2))
    w = rng.standard_normal(n).astype(F)
    r, y, xq, xs = run(pkg, arena, x, d, w, ready, in_place=True)
    check_norm(x, d, w, r, y)
    check_ready(oracle, y, xq, xs, ready)


@pytest.mark.parametrize("n", [288, 20480])
def test_norm_without(pkg, arena, oracle, n):
    """without the residual, without r, without y, without the activations: what is left is the same"""
    rng = np.random.default_rng(9)
    x, w = rng.standard_normal((4, n)).astype(F), rng.standard_normal(n).astype(F)
    _, y, xq, xs = run(pkg, arena, x, None, w, "biased", with_r=False)
    check_norm(x, None, w, None, y)
    check_ready(oracle, y, xq, xs, "biased")
    r, none, xq2, xs2 = run(pkg, arena, x, None, w, "biased", with_y=False)
    assert same_bits(r, x) and none is None and np.array_equal(xq2, xq) and np.array_equal(xs2, xs)
    _, y3, _, _ = run(pkg, arena, x, None, w, "biased", with_xq=False, with_r=False)
    assert same_bits(y3, y)


def test_norm_rows_alone_and_together(pkg, arena):
    """a token's numbers do not depend on the tokens beside it, nor on a row of infinities or NaN there"""
    rng = np.random.default_rng(3)
    x, d = (rng.standard_normal((9, 1120)).astype(F) for _ in range(2))
    w = rng.standard_normal(1120).astype(F)
    x[2, 5], x[4, 7], x[6] = np.inf, np.nan, 0
    d[6] = 0
    together = run(pkg, arena, x, d, w, "plain")
    for t in range(9):
        alone = run(pkg, arena, x[t:t + 1], d[t:t + 1], w, "plain")
        for a, b in zip(alone, together):
            assert np.array_equal(a[0].view(np.uint8), b[t].view(np.uint8))
    assert np.isnan(together[1][2, 5]) and (together[1][2, :5] == 0).all()  # inf / sqrt(inf); finite / sqrt(inf)
    assert np.isnan(together[1][4]).all()
    assert (together[1][6] == 0).all() and (together[3][6].view(F) == 0).all()


@pytest.mark.parametrize("size", [1e-30, 1e18, 1e25])
def test_norm_sizes(pkg, arena, size):
    """squares far below and above float32's range: the sum is held in 64 bits"""
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((2, 512)) * size).astype(F)
    w = np.ones(512, F)
    _, y, _, _ = run(pkg, arena, x, None, w, "plain", eps=0.0)
    check_norm(x, None, w, None, y, eps=0.0)
