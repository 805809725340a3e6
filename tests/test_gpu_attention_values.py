"""hq_attention_ex where values, keys and queries are of very different sizes: every output against the formula in 64 bits, held to
what the row itself sees and weighs, whatever else its tile, its sequence or its pages hold.

How far (`bound`): with p_j the row's weights (their sum 1), s_j and e_jd the scales and elements of the values, per output d
  (2 ds + 2^-20 + sqrt(n) 2^-22) sum_j p_j |s_j e_jd|    a score's error ds (its operands' 22 bits and its sums, twice: numerator and
      sum), a weight's 22 bits with the roundings of its factors, and the roundings of n additions as a random walk, margin 4
  + sum_j min(2^-25 W, p_j s_j) |e_jd|                   W the row's largest p_j s_j: a weight times its scale is held to 2^-25 of it
  + sum over p_j < 2^-120 of p_j |s_j e_jd|              weights that a float32 exponential does not hold
None of it knows a position that the row does not see."""
import numpy as np
import pytest

from gpu_util import Arena
from layer_model import F, Paged

pytestmark = pytest.mark.gpu
FORMS = ["int8", "f16"]
# new tokens of a sequence of 300 positions: 2 query heads a key head; a few rows, and a prompt's tiles from position 0
NEW = [1, 8, 300]


@pytest.fixture(scope="module")
def arena():
    import torch
    assert torch.cuda.is_available(), "the GPU tests need a GPU"
    return Arena(1 << 29)


def bound(p, q, scale, window=0, cap=0.0):
    """(out, how far) in 64 bits of q (tokens, query heads, dim)"""
    heads, group, scale = q.shape[1], q.shape[1] // p.heads, float(F(scale))
    out, far = np.zeros(q.shape), np.zeros(q.shape)
    held = {}
    for t, s, position in p.positions():
        if s not in held:
            k, v, there = p.vectors(s, range(p.lengths[s]))
            at = [p.place(s, i) or (0, 0) for i in range(p.lengths[s])]
            steps = np.array([p.vs[page, :, slot] for page, slot in at]).astype(np.float64)
            held[s] = k, v, there, steps
        k, v, there, steps = held[s]
        lo = max(0, position + 1 - window) if window else 0
        seen = np.arange(lo, position + 1)
        seen = seen[there[lo:position + 1]] if position >= 0 else seen[:0]
        if not seen.size:
            continue
        for h in range(heads):
            kk, vv, ss = k[seen, h // group], np.abs(v[seen, h // group]), steps[seen, h // group]
            qq = q[t, h].astype(np.float64)
            a = kk @ qq * scale
            ds = np.max(np.abs(kk) @ np.abs(qq)) * scale * (2.0 ** -21 + np.sqrt(p.dim) * 2.0 ** -23)
            if cap:
                a = float(F(cap)) * np.tanh(a / float(F(cap)))
            ds += np.max(np.abs(a)) * 2.0 ** -22
            w = np.exp(a - a.max())
            w /= w.sum()
            out[t, h] = w @ v[seen, h // group]
            elements = vv / np.where(ss > 0, ss, 1)[:, None]
            far[t, h] = ((2 * ds + 2.0 ** -20 + np.sqrt(seen.size) * 2.0 ** -22) * (w @ vv)
                         + np.minimum(2.0 ** -25 * (w * ss).max(), w * ss) @ elements + np.where(w < 2.0 ** -120, w, 0) @ vv)
    return out, far


def check(p, q, window=0, cap=0.0, scale=None):
    scale = scale or 1 / np.sqrt(p.dim)
    want, far = bound(p, q, scale, window, cap)
    got = p.run_attention(q, scale, window, cap)
    assert np.isfinite(got).all(), f"{np.argwhere(~np.isfinite(got))[:3]}"
    off = np.abs(got - want)
    worst = np.unravel_index(np.argmax(off / np.maximum(far, 1e-300)), off.shape)
    assert (off <= far).all(), f"at {worst}: {got[worst]!r}, {want[worst]!r} +- {far[worst]!r}"
    return got


def queries(rng, p, heads, size=2.0):
    return (rng.standard_normal((p.tokens, heads, p.dim)) * size).astype(F)


def made(pkg, arena, rng, form, lengths, new, dim=64, kv=1, page=32, sizes=None, longest=0):
    """a cache whose values at position j of a sequence are of sizes[j]"""
    arena.reset()
    p = Paged(pkg, arena, rng, form, kv, dim, page, lengths, new, longest=longest)
    p.fill(rng)
    if sizes is not None:
        for s, length in enumerate(lengths):
            k, v, _ = p.vectors(s, range(length))
            for j in range(length):
                p.put(s, j, k[j].astype(F), (v[j] * sizes[j]).astype(F))
        p.send()
    return p


# a value's size by its position of 300
SIZES = {
    "in turn": lambda rng: np.array([1.0, 1e12, 1.0, 1e-12])[np.arange(300) % 4],
    "growing": lambda rng: 10.0 ** np.linspace(-25, 25, 300),
    "shrinking": lambda rng: 10.0 ** np.linspace(25, -25, 300),
    "by 2^12 a token": lambda rng: 2.0 ** (12 * (np.arange(300) % 13) - 72),
    "any": lambda rng: 10.0 ** rng.uniform(-25, 25, 300),
    "one later": lambda rng: np.where(np.arange(300) == 297, 2.0 ** 30, 1.0),
    "some zero": lambda rng: np.where(np.arange(300) % 3 == 0, 0.0, 1.0),
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("window", [0, 1, 5, 70])
@pytest.mark.parametrize("sizes", SIZES)
def test_values_of_different_size(pkg, arena, form, new, window, sizes):
    rng = np.random.default_rng(11)
    p = made(pkg, arena, rng, form, [300], [new], sizes=SIZES[sizes](rng))
    check(p, queries(rng, p, 2), window=window)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim, kv, heads", [(16, 2, 6), (128, 1, 4), (256, 1, 2), (80, 1, 1)])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new", [3, 150])
def test_head_layouts(pkg, arena, form, dim, kv, heads, page, new):
    rng = np.random.default_rng(dim)
    p = made(pkg, arena, rng, form, [150, 90], [new, min(new, 90)], dim, kv, page, SIZES["in turn"](rng))
    check(p, queries(rng, p, heads))
    p = made(pkg, arena, rng, form, [150, 90], [new, min(new, 90)], dim, kv, page, SIZES["any"](rng))
    check(p, queries(rng, p, heads), window=33, cap=20.0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new", [1, 120])
@pytest.mark.parametrize("apart", [3, 4, 5, 12, 20, 40, 80])
@pytest.mark.parametrize("at", [0, 130])
def test_one_position_takes_all(pkg, arena, form, new, apart, at):
    """a position that takes nearly all the weight (25 powers of 2 more) and whose values are 2^-apart of the others', or zero; then one
    whose weight is next to nothing and whose values are 2^apart of theirs"""
    for sign, size in ((1, 2.0 ** -apart), (1, 0.0), (-1, 2.0 ** apart)):
        rng = np.random.default_rng(apart + at)
        sizes = np.ones(300)
        sizes[at] = size
        p = made(pkg, arena, rng, form, [300], [new], sizes=sizes)
        k, v, _ = p.vectors(0, [at])
        q = queries(rng, p, 2, size=0.5)
        # its key along a direction that every query has: a score of 25 ln 2 more (less) than others' about 0
        q[..., 0] = 8.0
        key = np.zeros((1, 64), F)
        key[0, 0] = sign * 25 * np.log(2) * 8 / 8
        p.put(0, at, key, v[0].astype(F))
        for j in range(300):
            if j != at:
                k, v, _ = p.vectors(0, [j])
                k[0, :, 0] = 0
                p.put(0, j, k[0].astype(F), v[0].astype(F))
        p.send()
        check(p, q)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lengths, new, heads, dim", [([6000], [1], 4, 128), ([5000, 700], [2, 1], 4, 64), ([2600], [200], 4, 64),
                                                      ([1900] * 9, [1] * 9, 2, 128)])
def test_shared_positions(pkg, arena, form, lengths, new, heads, dim):
    """positions that several workgroups share: what they found is joined whatever their values' sizes"""
    rng = np.random.default_rng(12)
    most = max(lengths)
    for sizes in (10.0 ** np.linspace(-25, 25, most), 10.0 ** np.linspace(25, -25, most), 10.0 ** rng.uniform(-20, 20, most)):
        p = made(pkg, arena, rng, form, lengths, new, dim, page=64, sizes=sizes)
        q = queries(rng, p, heads)
        # scores that fall where the values' sizes rise, so that far apart positions weigh alike: by up to 2^100
        check(p, q)
        q[..., :] *= F(8)
        check(p, q)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new", NEW)
def test_weights_against_sizes(pkg, arena, form, new):
    """a score falls by the powers of 2 that its values' size rises by (and the other way round): all positions weigh alike, and the
    sums' maximum moves by up to 110 powers of 2 while they do"""
    for way in (1, -1):
        rng = np.random.default_rng(13)
        power = np.linspace(-55, 55, 300) * way
        p = made(pkg, arena, rng, form, [300], [new])
        q = queries(rng, p, 2, size=0.25)
        q[..., 0] = 8.0
        for j in range(300):
            k, v, _ = p.vectors(0, [j])
            k[0] = 0
            k[0, :, 0] = -power[j] * np.log(2)  # (times 8 / sqrt(64))
            p.put(0, j, k[0].astype(F), (v[0] * 2.0 ** power[j]).astype(F))
        p.send()
        check(p, q)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new", [2, 9, 120])
def test_not_a_number_among_sizes(pkg, arena, form, new):
    """NaN values whose tokens come later, and sizes far apart: earlier tokens are as without them"""
    rng = np.random.default_rng(14)
    sizes = SIZES["in turn"](rng)
    p = made(pkg, arena, rng, form, [150], [new], sizes=sizes)
    q = queries(rng, p, 2)
    want, far = bound(p, q, 0.125)
    p.put(0, 149, np.ones((1, 64), F), np.full((1, 64), np.nan, F))
    p.send()
    got = p.run_attention(q, 0.125)
    assert np.isnan(got[-1]).all() and (np.abs(got - want)[:-1] <= far[:-1]).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("keys, asks, cap", [(1e35, 1e-35, 0.0), (1e37, 1e-37, 0.0), (1e35, 1e-35, 5.0), (1e20, 1e-20, 0.0),
                                             (1e-28, 1e28, 0.0), (1e-25, 1e25, 3.0)])
def test_large_keys_small_queries(pkg, arena, form, new, keys, asks, cap):
    """scores of ordinary size whose factors are near the ends of float32"""
    rng = np.random.default_rng(15)
    p = made(pkg, arena, rng, form, [300], [new])
    for j in range(300):
        k, v, _ = p.vectors(0, [j])
        p.put(0, j, (k[0] * keys).astype(F), v[0].astype(F))
    p.send()
    check(p, queries(rng, p, 2) * F(asks), cap=cap)


def check_seen(p, q, at):
    """rows that do not see position `at`, or give it nothing, are the mean of the values they see, whose scores are all near 0 (below
    2^-40); rows that it takes are the caller's to check"""
    got = p.run_attention(q, 1 / np.sqrt(p.dim))
    assert np.isfinite(got).all()
    k, v, there = p.vectors(0, range(p.lengths[0]))
    for t, s, position in p.positions():
        for h in range(q.shape[1]):
            if position >= at and h == 0:
                continue
            seen = np.array([j for j in range(position + 1) if j != at])
            mean = v[seen, 0].mean(0)
            assert (np.abs(got[t, h] - mean) <= np.abs(v[seen, 0]).mean(0) * (2.0 ** -20 + np.sqrt(seen.size) * 2.0 ** -22)).all()
    return got


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new", [1, 8, 100])
@pytest.mark.parametrize("others", [1.0, 1e-20, 0.0])
def test_one_large_key(pkg, arena, form, new, others):
    """a key of 1e35 among small ones or zeros: 1e-30 times it takes all or nothing, by its sign, and what does not see it is as ever"""
    rng = np.random.default_rng(16)
    p = made(pkg, arena, rng, form, [300], [new])
    at = 299 - new // 2
    for j in range(300):
        k, v, _ = p.vectors(0, [j])
        k = k[0] * others
        if j == at:
            k[:] = 0
            k[0, 3] = 1e35
        p.put(0, j, k.astype(F), v[0].astype(F))
    p.send()
    q = queries(rng, p, 2) * F(1e-30)
    q[:, 0, 3], q[:, 1, 3] = 1e-30, -1e-30
    got = check_seen(p, q, at)
    value = p.vectors(0, [at])[1][0, 0]
    first = at - (300 - new)
    assert (np.abs(got[first:, 0] - value) <= 2.0 ** -20 * np.abs(value)).all()
