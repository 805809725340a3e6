"""hq_sample_ex against the definition in 64 bits (NumPy): the same token, and its chance to a float32's rounding.

A chance is a weight over a sum, both in 64 bits, rounded once: 2^-24 of it, and 2^-40 for the sums' orders; below 2^-126 float32's
steps are 2^-149, and a rounding is off by at most half of one.  A drawn number
that lies within 2^-40 of a border could go either way by rounding; with 24-bit numbers that does not happen by chance, and
where a test puts one on a border its weights are whole numbers that add exactly."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32


def near(chance, share):
    return abs(chance - share) <= (2.0 ** -24 + 2.0 ** -40) * share + 2.0 ** -150


def model(l, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.5):
    l = np.asarray(l, F)
    there = np.nonzero(l > -np.inf)[0]
    if not there.size:
        return -1, 0.0
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    x, most = l[there].astype(np.float64), l[there].max()
    with np.errstate(all="ignore"):
        w = np.where(l[there] == most, 1.0, np.exp((x - np.float64(most)) / np.float64(F(temperature))))
    order = np.argsort(-x, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])])
        keep = before[:-1] < np.float64(F(top_p)) * before[-1]
        keep[0] = True
        order = order[keep]
    if min_p > 0:
        order = order[w[order] >= min(np.float64(F(min_p)), 1.0)]
    kept = np.sort(order)
    sums = np.cumsum(w[kept])
    u = np.float64(F(u))
    over = np.nonzero(sums > (u if u >= 0 else 0.0) * sums[-1])[0]
    at = over[0] if over.size else np.nonzero(w[kept] > 0)[0][-1]
    return int(there[kept[at]]), w[kept[at]] / sums[-1]


class Rows:
    """logits of some rows on the device, `pad` floats further apart than they are long, `off` floats into their memory"""

    def __init__(self, pkg, logits, pad=0, off=0):
        import torch
        self.pkg, self.l = pkg, np.asarray(logits, F)
        rows, self.vocab = self.l.shape
        wide = np.full(rows * (self.vocab + pad) + off + 8, np.inf, F)  # (what lies between is larger than any)
        for r in range(rows):
            at = off + r * (self.vocab + pad)
            wide[at:at + self.vocab] = self.l[r]
        self.memory = torch.from_numpy(wide).cuda()
        self.logits, self.stride = self.memory.data_ptr() + 4 * off, 4 * (self.vocab + pad)
        lib = pkg.library()
        self.need = lib.hq_sample_work_bytes(rows, self.vocab)
        self.work = torch.full((self.need + 64,), 0xff, dtype=torch.uint8, device="cuda")
        self.tokens = torch.full((rows + 1,), -77, dtype=torch.int32, device="cuda")
        self.chance = torch.full((rows + 1,), -77.0, device="cuda")

    def call(self, u, temperature=None, top_k=None, top_p=None, min_p=None, chance=True, stream=None):
        """settings: a number a row, or None"""
        import torch
        rows = len(self.l)

        def put(v, kind):
            return None if v is None else torch.from_numpy(np.broadcast_to(np.asarray(v, kind), (rows,)).copy()).cuda()
        self.held = [put(u, F), put(temperature, F), put(top_k, np.int32), put(top_p, F), put(min_p, F)]
        torch.cuda.synchronize()
        at = [None if t is None else t.data_ptr() for t in self.held]
        lib = self.pkg.library()
        status = lib.hq_sample_ex(self.tokens.data_ptr(), self.chance.data_ptr() if chance else None, self.logits, *at, rows, self.vocab,
                                  self.stride, self.work.data_ptr(), self.need, stream)
        assert status == 0, lib.hq_last_error_message()

    def got(self):
        import torch
        torch.cuda.synchronize()
        assert int(self.tokens[-1]) == -77 and float(self.chance[-1]) == -77 and (self.work[self.need:] == 0xff).all()
        return self.tokens.cpu().numpy()[:-1], self.chance.cpu().numpy()[:-1]

    def check(self, u, stream=None, **settings):
        self.call(u, stream=stream, **settings)
        token, chance = self.got()
        one = lambda v, r: v if np.ndim(v) == 0 else np.asarray(v)[r]  # noqa: E731
        for r in range(len(self.l)):
            mine = {k: one(v, r) for k, v in settings.items() if v is not None}
            want, share = model(self.l[r], u=one(u, r), **mine)
            assert token[r] == want, (r, mine, one(u, r), token[r], want)
            assert near(chance[r], share), (r, chance[r], share)
        return token


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.3, top_p=0.5),
            dict(temperature=0.6, top_k=50, top_p=0.95, min_p=0.02), dict(top_k=1), dict(top_k=2, top_p=0.99), dict(top_k=1000, temperature=2.0),
            dict(temperature=0.02), dict(temperature=50.0, top_p=0.99), dict(temperature=0.05, top_k=300), dict(top_k=64), dict(top_k=65)]


def language(rng, rows, vocab, lift=8.0):
    """a few words stand out, the frequent first words more often"""
    l = 2 * rng.standard_normal((rows, vocab)) - 0.6 * np.log1p(np.arange(vocab) / 50)
    for r in range(rows):
        at = (vocab * rng.random(min(20, vocab)) ** 3).astype(int)
        l[r, at] += lift * rng.random(at.size)
    return l.astype(F)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 257, 1000, 1023, 1024, 1025, 2047, 2049, 4097, 8191, 16384, 32000, 50257, 128256, 300001])
def test_settings(pkg, vocab):
    rng = np.random.default_rng(vocab)
    rows = Rows(pkg, language(rng, len(SETTINGS), vocab))
    each = {k: [s.get(k, d) for s in SETTINGS] for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    for _ in range(4):
        rows.check(rng.random(len(SETTINGS)).astype(F), **each)
    rows.check(np.zeros(len(SETTINGS), F), **each)
    rows.check(np.full(len(SETTINGS), 1 - 2.0 ** -24, F), **each)


@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("shape", ["flat", "steep", "rising", "falling", "whole", "same", "two", "hidden", "huge", "around 0", "far apart", "one bin"])
def test_shapes(pkg, setting, shape):
    """logits of every kind of crowd: evenly spread, in order, with ties by the thousand, mostly hidden, of extreme sizes (to infinity)"""
    rng = np.random.default_rng(len(shape))
    for vocab in (3000, 40001):
        x = rng.standard_normal((2, vocab))
        l = {"flat": 0.1 * x, "steep": 30 * x, "rising": np.sort(3 * x, -1), "falling": -np.sort(-3 * x, -1), "whole": np.round(2 * x),
             "same": np.zeros_like(x) + 1.25, "two": np.where(x > 1, 2.0, -2.0),
             "hidden": np.where(rng.random(x.shape) < 0.999, -np.inf, x), "huge": 1e37 * x, "around 0": 1e-40 * x,
             "far apart": np.sign(x) * np.exp(20 * np.abs(x)), "one bin": np.where(x > 2, 1 + 1e-6 * np.round(x * 4), -20 + x)}[shape].astype(F)
        rows = Rows(pkg, l)
        for u in (rng.random(2), [0.0, 0.999], rng.random(2)):
            rows.check(np.asarray(u, F), **setting)


@pytest.mark.parametrize("pad, off", [(0, 1), (1, 0), (3, 2), (4, 0), (5, 4)])
@pytest.mark.parametrize("vocab", [777, 50257, 65536])
def test_rows_that_begin_anywhere(pkg, pad, off, vocab):
    rng = np.random.default_rng(pad + off)
    rows = Rows(pkg, language(rng, 5, vocab), pad, off)
    for setting in SETTINGS[:7]:
        rows.check(rng.random(5).astype(F), **setting)


def test_without_settings(pkg):
    rng = np.random.default_rng(1)
    l = language(rng, 4, 5000)
    rows = Rows(pkg, l)
    rows.check([0.1, 0.4, 0.7, 0.99])
    rows.call([0.1, 0.4, 0.7, 0.99], chance=False)
    assert (rows.got()[0] == [model(r, u=v)[0] for r, v in zip(l, (0.1, 0.4, 0.7, 0.99))]).all()


def test_words_that_are_never_drawn(pkg):
    """-infinity, NaN and rows of nothing else; the type's lowest value where all else is hidden; +infinity"""
    rng = np.random.default_rng(2)
    low = np.finfo(F).min
    l = rng.standard_normal((9, 4000)).astype(F)
    l[0, :] = -np.inf
    l[1, :] = np.nan
    l[2, ::2], l[2, 1::2] = -np.inf, np.nan
    l[3, 17:], l[3, :17] = -np.inf, np.nan
    l[3, 3999] = -5.0
    l[4, :] = low
    l[4, 5] = -np.inf
    l[5, 100:] = low
    l[6, 7], l[6, 70], l[6, 700] = np.inf, np.inf, np.nan
    l[7, 5:] = np.nan
    l[8, :], l[8, 3], l[8, 9] = -np.inf, -0.0, 0.0
    rows = Rows(pkg, l)
    for setting in SETTINGS:
        for u in (0.0, 0.3, 0.5, 0.99):
            token = rows.check(np.full(9, u, F), **setting)
            assert (token[:3] == -1).all() and token[3] == 3999 and token[6] in (7, 70) and token[8] in (3, 9)


def test_numbers_out_of_range(pkg):
    """u below 0 and NaN: the first kept token; 1 and more: the last.  Settings that mean off, or everything but one"""
    rng = np.random.default_rng(3)
    l = language(rng, 1, 3000)[0]
    rows = Rows(pkg, np.stack([l] * 6))
    u = np.array([-1.0, np.nan, 0.0, 1.0, 7.0, np.inf], F)
    for setting in (dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.01)):
        token = rows.check(u, **setting)
        assert token[0] == token[1] == token[2] < token[3] == token[4] == token[5]
    half = np.full(6, 0.5, F)
    rows.check(half, temperature=[np.nan, -1.0, -np.inf, np.inf, 1e-38, 3e38])
    rows.check(half, top_p=[0.0, -3.0, 1.0, 2.0, np.nan, 1e-30])
    rows.check(half, min_p=[0.0, -1.0, 1.0, 5.0, np.nan, np.inf])
    rows.check(half, top_k=[0, -1, -2 ** 31, 2 ** 31 - 1, 3000, 2999])


def test_borders_between_equal_weights(pkg):
    """equal logits: shares are whole numbers over a whole number, and a border belongs to the token behind it"""
    l = np.zeros((8, 64), F)
    rows = Rows(pkg, l)
    for k in (1, 2, 4, 8, 64):
        u = np.arange(8) / 8
        token = rows.check(u.astype(F), top_k=k)
        assert (token == (u * k).astype(int)).all()
    # the mass before the token reaches the share exactly: it is left out
    for p, most in ((0.25, 16), (0.5, 32), (0.75, 48), (0.015625, 1)):
        assert rows.check(np.full(8, 0.99999, F), top_p=p)[0] == most - 1


def test_rows_of_every_kind_at_once(pkg):
    """300 rows, each with its own settings"""
    rng = np.random.default_rng(5)
    rows, vocab = 300, 9999
    l = language(rng, rows, vocab)
    l[::11] = np.round(l[::11])
    l[5::13, 100:] = -np.inf
    l[7] = np.nan
    pick = lambda *v: rng.choice(v, rows)  # noqa: E731
    Rows(pkg, l).check(rng.random(rows).astype(F), temperature=pick(0.0, 0.5, 1.0, 1.5), top_k=pick(0, 0, 1, 20, 100, 3000),
                       top_p=pick(1.0, 0.3, 0.9, 0.999), min_p=pick(0.0, 0.0, 0.1, 0.001))


def test_frequencies(pkg):
    """drawn with evenly spaced numbers, tokens come as often as their chances say"""
    rng = np.random.default_rng(6)
    l = language(rng, 1, 500)[0]
    n = 4096
    rows = Rows(pkg, np.broadcast_to(l, (n, 500)))
    rows.call(((np.arange(n) + 0.5) / n).astype(F), top_k=20)
    token, _ = rows.got()
    x = np.sort(l)[::-1][:20].astype(np.float64)
    share = np.exp(x - x[0]) / np.exp(x - x[0]).sum()
    counts = np.array([(token == i).sum() for i in np.argsort(-l, kind="stable")[:20]])
    assert counts.sum() == n and (np.abs(counts - n * share) <= 1.001).all()


def test_logits_past_4_gib(pkg):
    """the last rows of logits that 32 bits cannot address"""
    import torch
    lib, rows, vocab = pkg.library(), 9000, 128256
    l = torch.full((rows, vocab), -5.0, device="cuda")
    at = torch.arange(rows, device="cuda") * 13 % vocab
    l[torch.arange(rows, device="cuda"), at] = 40.0
    u = torch.rand(rows, device="cuda")
    need = lib.hq_sample_work_bytes(rows, vocab)
    work, token = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert lib.hq_sample_ex(token.data_ptr(), None, l.data_ptr(), u.data_ptr(), None, None, None, None, rows, vocab, 4 * vocab,
                            work.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(token.long(), at)


def test_replayed(pkg):
    """captured on a stream of its own and replayed with other logits, numbers and settings, the workspace dirtied in between"""
    import torch
    rng = np.random.default_rng(7)
    rows = Rows(pkg, language(rng, 6, 20000))
    assert pkg.library().hq_init() == 0
    each = dict(temperature=[0.7, 1.0, 0.0, 1.0, 1.0, 0.9], top_k=[40, 0, 0, 0, 700, 3], top_p=[0.9, 0.95, 1.0, 1.0, 1.0, 0.5],
                min_p=[0.0, 0.0, 0.0, 0.1, 0.0, 0.0])
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    rows.check(rng.random(6).astype(F), stream=stream.cuda_stream, **each)
    held = rows.held
    lib, at = pkg.library(), [t.data_ptr() for t in held]
    with torch.cuda.graph(g, stream=stream):
        status = lib.hq_sample_ex(rows.tokens.data_ptr(), rows.chance.data_ptr(), rows.logits, *at, 6, rows.vocab, rows.stride,
                                  rows.work.data_ptr(), rows.need, stream.cuda_stream)
    assert status == 0
    for _ in range(4):
        l, u = language(rng, 6, 20000, 14 * rng.random()), rng.random(6).astype(F)
        rows.memory[:6 * 20000].copy_(torch.from_numpy(l).view(-1))
        held[0].copy_(torch.from_numpy(u))
        rows.work.fill_(0xff)
        rows.tokens[:6].fill_(-5)
        torch.cuda.synchronize()
        g.replay()
        token, chance = rows.got()
        for r in range(6):
            want, share = model(l[r], u=u[r], **{k: v[r] for k, v in each.items()})
            assert token[r] == want and near(chance[r], share)


@pytest.mark.parametrize("vocab", [8192, 8193, 10239, 10241, 40000])
@pytest.mark.parametrize("pad", [0, 3])
def test_many_flat_rows(pkg, vocab, pad):
    """rows whose top-p takes in most words, or words of one weight by the thousand, among ordinary ones"""
    rng = np.random.default_rng(vocab)
    kinds = [lambda: 0.05 * rng.standard_normal(vocab), lambda: language(rng, 1, vocab)[0], lambda: np.zeros(vocab),
             lambda: np.where(rng.random(vocab) < 0.5, -np.inf, 1.0), lambda: np.round(rng.standard_normal(vocab)),
             lambda: np.linspace(3, -3, vocab), lambda: np.full(vocab, -np.inf)]
    n = 5 * len(kinds)
    rows = Rows(pkg, np.stack([kinds[r % len(kinds)]() for r in range(n)]), pad)
    each = dict(temperature=rng.choice([0.9, 1.0, 3.0, 40.0], n), top_k=rng.choice([0, 0, 0, vocab // 2, vocab + 5], n),
                top_p=rng.choice([0.3, 0.9, 0.999, 1 - 2.0 ** -24], n), min_p=rng.choice([0.0, 0.0, 0.5], n))
    for u in (rng.random(n).astype(F), np.zeros(n, F), np.full(n, 1 - 2.0 ** -24, F)):
        rows.check(u, **each)


def test_flat_rows_replayed(pkg):
    """a captured call whose rows are flat in one replay and not in the next, two graphs on one workspace in turn"""
    import torch
    rng = np.random.default_rng(17)
    rows = Rows(pkg, 0.1 * rng.standard_normal((4, 20000)))
    stream, graphs = torch.cuda.Stream(), []
    rows.check(rng.random(4).astype(F), stream=stream.cuda_stream, top_p=0.95)
    held = rows.held
    lib = pkg.library()
    at = [None if t is None else t.data_ptr() for t in held]
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            assert lib.hq_sample_ex(rows.tokens.data_ptr(), rows.chance.data_ptr(), rows.logits, *at, 4, rows.vocab, rows.stride,
                                    rows.work.data_ptr(), rows.need, stream.cuda_stream) == 0
        graphs.append(g)
    for i in range(6):
        l = (0.1 * rng.standard_normal((4, 20000))).astype(F) if i % 3 else language(rng, 4, 20000)
        u = rng.random(4).astype(F)
        rows.memory[:4 * 20000].copy_(torch.from_numpy(l).view(-1))
        held[0].copy_(torch.from_numpy(u))
        rows.work[:rows.need].fill_(0xff)
        rows.tokens[:4].fill_(-5)
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        token, chance = rows.got()
        for r in range(4):
            want, share = model(l[r], u=u[r], top_p=0.95)
            assert token[r] == want and near(chance[r], share)


@pytest.mark.parametrize("vocab", [50, 700, 8192, 8193, 32000, 128256])
@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.9999), dict(min_p=1e-30), dict(top_k=40), dict(top_k=600, top_p=0.99999)], ids=str)
def test_the_last_kept_one_where_it_weighs_nothing(pkg, vocab, settings):
    """numbers of 1 and more draw the last kept token, also where what lies behind the heavy ones is less than a sum's rounding"""
    rng = np.random.default_rng(vocab + len(settings))
    l = language(rng, 24, vocab) * 2
    l[:, vocab // 3:] -= 60  # (10^-26 of the first third's)
    rows = Rows(pkg, l)
    for u in (1.0, 7.0, 3e38, np.inf):
        rows.check(u, **settings)
        rows.check(u, temperature=0.9, **settings)
    rows.check(np.where(np.arange(24) % 2, F(1.0), F(0.3)), **settings)


@pytest.mark.parametrize("u", [1.0, 7.0])
def test_the_last_kept_one_where_parts_keep_none(pkg, u):
    """flat rows whose top-p is spread over blocks, the last of which have words at the line that are not kept, and nothing else that is:
    the last kept one lies before them"""
    rng = np.random.default_rng(17)
    vocab, part = 128256, 8192
    for behind in (1, 3):
        l = rng.random((16, vocab)).astype(F)
        few = (16 - behind) * part
        l[:, few:] = -9
        for r in range(16):
            w = np.sort(np.exp(l[r].astype(np.float64)))[::-1]
            line = np.log(w[np.searchsorted(np.cumsum(w), 0.9 * w.sum())])
            for q in range(16 - behind, 16):
                l[r, q * part + rng.choice(5000, 3, replace=False)] = line - 2e-4 - 1e-4 * rng.random(3)
        rows = Rows(pkg, l)
        rows.check(u, top_p=0.9)
        assert (rows.got()[0] < few).all()
        rows.check(rng.random(16).astype(F), top_p=0.9)
