"""hq_adapters_ex against the formula in 64 bits, and its gradient-free linearity: what it leaves alone, its forms and lengths.

How far: a low number is a sum of n products of float32 values, held to 2^-22 each and added in float32 (a random walk of
sqrt(n) roundings with a margin of 4); a row's number adds `rank` products of these the same way, times a scale, to `from`."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32


def half(rng, form, *shape, spread=1.0):
    """(float16 or bfloat16 bits, their float64 values)"""
    import torch
    t = torch.from_numpy((rng.standard_normal(shape) * spread).astype(F)).to(torch.float16 if form == "f16" else torch.bfloat16)
    return t, t.double().numpy()


def wanted(x, a, b, base, scales, which, starts):
    """(y, how far a float32 kernel may be from it) in float64; rows that no sequence has: NaN"""
    y = np.full((len(x), b.shape[1]), np.nan)
    far = np.zeros_like(y)
    for s, w in enumerate(which):
        rows = slice(max(starts[s], 0), max(starts[s + 1], 0))
        y[rows] = base[rows]
        if not 0 <= w < len(a):
            continue
        xs, scale = x[rows].astype(np.float64), abs(float(scales[w]))
        low, size = xs @ a[w].T, np.abs(xs) @ np.abs(a[w]).T
        off = size * (2.0 ** -22 + 4 * np.sqrt(a.shape[2]) * 2.0 ** -24)
        add, most = low @ b[w].T, np.abs(low) @ np.abs(b[w]).T
        y[rows] += float(scales[w]) * add
        far[rows] = scale * (off @ np.abs(b[w]).T + most * (2.0 ** -22 + 4 * np.sqrt(a.shape[1]) * 2.0 ** -24))
        far[rows] += 2.0 ** -22 * (np.abs(base[rows]) + scale * np.abs(add))
    return y, far


class Call:
    def __init__(self, pkg, rng, form, n, rows, rank, adapters, fresh, which, with_scales=True, with_from=True, in_place=False, pad=0,
                 spread=1.0, x_size=1.0, behind=2, longest=None, packed=False):
        import torch
        self.pkg, self.form, self.n, self.rank, self.adapters = pkg, form, n, rank, adapters
        self.starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
        self.tokens, self.which = int(self.starts[-1]) + behind, which
        self.x = (rng.standard_normal((self.tokens, n)) * x_size * np.exp(0.5 * rng.standard_normal(n))).astype(F)
        self.a = [half(rng, form, adapters, rank, n, spread=spread) for _ in rows]
        self.b = [half(rng, form, adapters, r, rank, spread=spread) for r in rows]
        self.base = [rng.standard_normal((self.tokens, r)).astype(F) if with_from else np.zeros((self.tokens, r), F) for r in rows]
        self.scales = (rng.random(max(1, adapters)) + 0.5).astype(F) * np.where(np.arange(max(1, adapters)) % 3 == 1, -1, 1).astype(F)
        put = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()  # noqa: E731
        wide = np.full((self.tokens, n + pad), np.nan, F)
        wide[:, :n] = self.x
        self.dx, self.ds, self.dw, self.dstarts = put(wide), put(self.scales), put(np.asarray(which, np.int32)), put(self.starts)
        self.da, self.db = [t.cuda() for t, _ in self.a], [t.cuda() for t, _ in self.b]
        self.dfrom, self.dy = [], []
        for base, r in zip(self.base, rows):
            room = 0 if packed else -r % 4 + pad
            y = np.full((self.tokens, r + room), -9, F)
            if with_from:
                given = y.copy()
                given[:, :r] = base
                if in_place:
                    y = given
            self.dy.append(put(y))
            self.dfrom.append(None if not with_from else self.dy[-1] if in_place else put(given))
        self.in_place, self.with_from, self.rows = in_place, with_from, rows
        self.targets = (pkg.adapters.Target * len(rows))(*[
            pkg.adapters.Target(a.data_ptr(), b.data_ptr(), f.data_ptr() if f is not None else None, y.data_ptr(), r, 4 * y.shape[1],
                                4 * y.shape[1]) for a, b, f, y, r in zip(self.da, self.db, self.dfrom, self.dy, rows)])
        if longest is None:
            longest = max(fresh, default=0)
        self.batch = pkg.cache.Batch(self.dstarts.data_ptr(), None, None, len(fresh), self.tokens, longest, 0)
        lib = pkg.library()
        self.need = lib.hq_adapters_work_bytes(len(rows), rank, self.tokens)
        self.work = torch.full((max(self.need, 1) + 64,), 0xff, dtype=torch.uint8, device="cuda")
        self.arguments = (self.targets, len(rows), self.dx.data_ptr(), 4 * (n + pad), n, rank, adapters, pkg.adapters.FORMS[form],
                          self.ds.data_ptr() if with_scales else None, self.dw.data_ptr(), self.batch, self.work.data_ptr(), self.need)
        if not with_scales:
            self.scales = np.ones_like(self.scales)
        torch.cuda.synchronize()

    def run(self, stream=None):
        lib = self.pkg.library()
        status = lib.hq_adapters_ex(*self.arguments, stream)
        assert status == 0, lib.hq_last_error_message()

    def check(self):
        import torch
        torch.cuda.synchronize()
        assert (self.work[self.need:] == 0xff).all(), "wrote behind the workspace"
        for i, r in enumerate(self.rows):
            got = self.dy[i].cpu().numpy()
            want, far = wanted(self.x, self.a[i][1], self.b[i][1], self.base[i].astype(np.float64), self.scales, self.which, self.starts)
            assert (got[:, r:] == -9).all(), "wrote between the rows"
            left = np.isnan(want)
            kept = self.base[i] if self.in_place else np.full_like(self.base[i], -9)
            assert np.array_equal(got[:, :r][left], kept[left]), "touched rows that no sequence has"
            d = np.abs(got[:, :r] - want)
            assert (d[~left] <= far[~left] + 1e-30).all(), (i, np.nanmax(d / np.maximum(far, 1e-30)))
        return [y.cpu().numpy() for y in self.dy]


@pytest.mark.parametrize("form", ["f16", "bf16"])
@pytest.mark.parametrize("n, rows, rank", [
    (32, (5,), 8), (288, (288, 96), 16), (4096, (4096, 1024, 1024), 16), (1056, (33, 1, 700), 32), (96, (64,), 256), (2048, (130,), 64),
    (8192, (17, 18, 19, 20, 21, 22, 23, 24), 8), (160, (31, 1025), 40), (64, (4100,), 24), (512, (100,), 128), (448, (200, 50), 136)])
@pytest.mark.parametrize("fresh", [[1], [1] * 7, [3, 0, 1, 5], [33, 1, 70]], ids=str)
def test_forms_and_lengths(pkg, form, n, rows, rank, fresh):
    rng = np.random.default_rng(n + rank + len(fresh))
    which = [(-1 if i == 2 else i * 3 % 4) for i in range(len(fresh))]
    call = Call(pkg, rng, form, n, rows, rank, 4, fresh, which)
    call.run()
    call.check()


@pytest.mark.parametrize("fresh", [[15], [16], [17], [31, 32], [63], [64], [65], [127, 1, 129], [128], [300], [2, 255, 257], [0, 0, 9, 0], [0], [1000]], ids=str)
@pytest.mark.parametrize("rank", [8, 16, 48, 64])
def test_tiles(pkg, fresh, rank):
    rng = np.random.default_rng(sum(fresh) + rank)
    call = Call(pkg, rng, "bf16" if rank % 16 else "f16", 352, (260, 36), rank, 3, fresh, list(range(len(fresh))))
    call.run()
    call.check()


@pytest.mark.parametrize("more", [dict(with_scales=False), dict(with_from=False), dict(in_place=True), dict(pad=12), dict(pad=4, in_place=True),
                                  dict(longest=0), dict(behind=0), dict(behind=70)], ids=str)
@pytest.mark.parametrize("fresh", [[1, 1, 1], [40, 1, 0, 90]], ids=str)
def test_arguments(pkg, more, fresh):
    rng = np.random.default_rng(len(fresh))
    call = Call(pkg, rng, "bf16", 320, (70, 200), 16, 2, fresh, [1, -1, 0, 1][:len(fresh)], **more)
    call.run()
    call.check()


@pytest.mark.parametrize("which", [[-1, -1], [2, 2 ** 31 - 1], [-2 ** 31, 5]], ids=str)
@pytest.mark.parametrize("adapters", [2, 0])
def test_no_adapters(pkg, which, adapters):
    """sequences without one: y = from"""
    call = Call(pkg, np.random.default_rng(1), "f16", 64, (50,), 16, adapters, [3, 20], which)
    call.run()
    got = call.check()
    assert np.array_equal(got[0][:23, :50], call.base[0][:23])


def test_one_adapter_of_many_requests(pkg):
    rng = np.random.default_rng(5)
    call = Call(pkg, rng, "bf16", 1024, (512,), 32, 40, [1] * 300, [int(v) for v in rng.integers(-1, 40, 300)])
    call.run()
    call.check()


@pytest.mark.parametrize("x_size", [1e-30, 1e-12, 1e12, 1e30])
@pytest.mark.parametrize("form", ["f16", "bf16"])
@pytest.mark.parametrize("fresh", [[2], [77]], ids=str)
def test_inputs_of_any_size(pkg, x_size, form, fresh):
    rng = np.random.default_rng(3)
    call = Call(pkg, rng, form, 256, (64,), 16, 1, fresh, [0], x_size=x_size, with_from=False, spread=1e-3)
    call.run()
    call.check()


def test_subnormal_factors(pkg):
    """float16 factors below 2^-14 count as what they are"""
    rng = np.random.default_rng(4)
    for fresh in ([2], [60]):
        call = Call(pkg, rng, "f16", 256, (64,), 16, 2, fresh, [1], spread=2e-6, with_from=False)
        call.run()
        call.check()


@pytest.mark.parametrize("fresh", [[1, 1, 1, 1], [40, 40, 40, 40]], ids=str)
def test_infinities_stay_where_they_are(pkg, fresh):
    """a token with an infinity or NaN spoils its own row alone"""
    import torch
    rng = np.random.default_rng(6)
    call = Call(pkg, rng, "bf16", 128, (96,), 16, 2, fresh, [0, 1, 0, 1], behind=0)
    clean = Call(pkg, np.random.default_rng(6), "bf16", 128, (96,), 16, 2, fresh, [0, 1, 0, 1], behind=0)
    bad = [call.starts[1], call.starts[3]]
    call.dx[int(bad[0]), 5], call.dx[int(bad[1]), 127] = float("inf"), float("nan")
    torch.cuda.synchronize()
    for c in (call, clean):
        c.run()
    torch.cuda.synchronize()
    got, want = call.dy[0], clean.dy[0]
    keep = torch.ones(call.tokens, dtype=torch.bool)
    keep[bad] = False
    assert torch.equal(got[keep], want[keep])
    assert not torch.isfinite(got[bad, :96]).any()


def test_factors_past_4_gib(pkg):
    """the last of adapters whose a and b 32 bits cannot address"""
    import torch
    lib, n, rank, adapters = pkg.library(), 8192, 64, 5000
    a = torch.zeros(adapters, rank, n, dtype=torch.float16, device="cuda")
    b = torch.zeros(adapters, n, rank, dtype=torch.float16, device="cuda")
    a[-1].copy_(torch.randn(rank, n, device="cuda"))
    b[-1].copy_(torch.randn(n, rank, device="cuda"))
    for tokens in (1, 50):
        x, y = torch.randn(tokens, n, device="cuda"), torch.empty(tokens, n, device="cuda")
        which = torch.tensor([adapters - 1], dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
        need = lib.hq_adapters_work_bytes(1, rank, tokens)
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        target = pkg.adapters.Target(a.data_ptr(), b.data_ptr(), None, y.data_ptr(), n, 4 * n, 4 * n)
        batch = pkg.cache.Batch(starts.data_ptr(), None, None, 1, tokens, tokens, 0)
        torch.cuda.synchronize()
        assert lib.hq_adapters_ex(target, 1, x.data_ptr(), 4 * n, n, rank, adapters, 1, None, which.data_ptr(), batch, work.data_ptr(),
                                  need, torch.cuda.current_stream().cuda_stream) == 0
        low, wa, wb = x.double().cpu(), a[-1].double().cpu(), b[-1].double().cpu()
        want = (low @ wa.t()) @ wb.t()
        far = ((low.abs() @ wa.abs().t()) @ wb.abs().t()) * (2.0 ** -21 + 4 * (n ** 0.5 + rank ** 0.5) * 2.0 ** -24)
        assert ((y.double().cpu() - want).abs() <= far).all()


@pytest.mark.parametrize("fresh", [[1, 1, 1], [20, 60, 1]], ids=str)
def test_same_numbers_every_time(pkg, fresh):
    """on another stream, captured and replayed, twice: the same bits"""
    import torch
    call = Call(pkg, np.random.default_rng(7), "bf16", 1024, (300, 77), 32, 2, fresh, [0, 1, 0])
    assert pkg.library().hq_init() == 0
    call.run()
    first = call.check()
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    call.run(stream.cuda_stream)
    assert all(np.array_equal(a, b) for a, b in zip(first, call.check()))
    with torch.cuda.graph(g, stream=stream):
        call.run(stream.cuda_stream)
    for _ in range(3):
        for y in call.dy:
            y[:int(call.starts[-1])].fill_(-9)
        call.work.fill_(0xff)
        torch.cuda.synchronize()
        g.replay()
        assert all(np.array_equal(a, b) for a, b in zip(first, call.check()))


def test_a_batch_that_contradicts_itself(pkg):
    """starts that fall or pass the rows: wrong numbers, no access out of the buffers"""
    import torch
    for starts in ([0, 50, 3, 400, 9], [-5, 2 ** 31 - 1, -2 ** 31, 7, 7], [9, 9, 9, 9, 9]):
        for longest in (1, 60):
            call = Call(pkg, np.random.default_rng(8), "f16", 64, (40,), 8, 2, [15, 15, 15, 15], [0, 1, 0, 1], behind=0, longest=longest)
            call.dstarts.copy_(torch.tensor(starts, dtype=torch.int32))
            torch.cuda.synchronize()
            call.run()
            torch.cuda.synchronize()
            assert (call.dy[0][:, 40:] == -9).all() and (call.work[call.need:] == 0xff).all()


@pytest.mark.parametrize("fresh", [[1] * 7, [40, 1, 0, 17]], ids=str)
@pytest.mark.parametrize("more", [dict(), dict(in_place=True), dict(with_from=False)], ids=str)
def test_rows_that_are_not_whole_fours(pkg, fresh, more):
    """rows back to back, so that tokens begin on any float; in a batch of single tokens and in tiles"""
    rng = np.random.default_rng(len(fresh))
    for rows in ((97,), (1, 2, 3), (64, 130), (515,)):
        call = Call(pkg, rng, "bf16", 96, rows, 16, 3, fresh, (np.arange(len(fresh)) % 4).tolist(), packed=True, **more)
        call.run()
        call.check()


@pytest.mark.parametrize("rows, rank, fresh", [((0, 64), 64, [1040]), ((0, 70, 0), 64, [1000]), ((33, 0, 0), 256, [100, 28]),
                                               ((0, 50), 16, [1, 1, 1]), ((0, 0), 8, [20])], ids=str)
def test_projections_without_rows(pkg, rows, rank, fresh):
    """they are left out, and the rest, whose values more blocks may share, stays within the call's workspace"""
    call = Call(pkg, np.random.default_rng(rank), "bf16", 1056, rows, rank, 2, fresh, [1, 0, 1][:len(fresh)])
    call.run()
    call.check()


def test_most_tokens(pkg):
    """2^24 rows by the kernels of single tokens, whatever a sequence has of them"""
    import torch
    lib, n, rank, rows, tokens = pkg.library(), 32, 8, 4, 1 << 24
    a, b = torch.randn(1, rank, n, device="cuda").half(), torch.randn(1, rows, rank, device="cuda").half()
    x, y = torch.randn(tokens, n, device="cuda"), torch.full((tokens, rows), -9.0, device="cuda")
    starts, which = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, tokens - 3], [0]))
    need = lib.hq_adapters_work_bytes(1, rank, tokens)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    target = pkg.adapters.Target(a.data_ptr(), b.data_ptr(), None, y.data_ptr(), rows, 4 * rows, 4 * rows)
    batch = pkg.cache.Batch(starts.data_ptr(), None, None, 1, tokens, 1, 0)
    torch.cuda.synchronize()
    assert lib.hq_adapters_ex(target, 1, x.data_ptr(), 4 * n, n, rank, 1, 1, None, which.data_ptr(), batch, work.data_ptr(), need,
                              torch.cuda.current_stream().cuda_stream) == 0, lib.hq_last_error_message()
    assert (y[-3:] == -9).all()
    a, b = a[0].double(), b[0].double()
    for first in range(0, tokens - 3, 1 << 21):
        rows_of = slice(first, min(first + (1 << 21), tokens - 3))
        e = x[rows_of].double()
        want = (e @ a.t()) @ b.t()
        # (n and rank products and sums, a rounding each at most)
        far = (e.abs() @ a.abs().t()) @ b.abs().t() * (n + rank + 3) * 2.0 ** -24
        assert ((y[rows_of].double() - want).abs() <= far).all(), first


def test_a_row_as_long_as_can_be(pkg):
    """a token of 2^31 - 32 values (more tokens' stride would pass 2^31): factors of 32 GiB, 0 but for both ends"""
    import torch
    lib, n, rank, rows, ends = pkg.library(), 2 ** 31 - 32, 8, 5, 1024
    a, x = torch.zeros(1, rank, n, dtype=torch.float16, device="cuda"), torch.zeros(1, n, device="cuda")
    for part in (slice(0, ends), slice(n - ends, n)):
        a[0, :, part] = torch.randn(rank, ends, device="cuda").half()
        x[0, part] = torch.randn(ends, device="cuda")
    b, y = torch.randn(1, rows, rank, device="cuda").half(), torch.full((rows + 8,), -9.0, device="cuda")
    starts, which = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 1], [0]))
    need = lib.hq_adapters_work_bytes(1, rank, 1)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    target = pkg.adapters.Target(a.data_ptr(), b.data_ptr(), None, y.data_ptr(), rows, 0, 0)
    batch = pkg.cache.Batch(starts.data_ptr(), None, None, 1, 1, 0, 0)
    torch.cuda.synchronize()
    assert lib.hq_adapters_ex(target, 1, x.data_ptr(), 0, n, rank, 1, 1, None, which.data_ptr(), batch, work.data_ptr(), need,
                              torch.cuda.current_stream().cuda_stream) == 0, lib.hq_last_error_message()
    torch.cuda.synchronize()
    both = lambda t: torch.cat([t[..., :ends], t[..., n - ends:]], -1).double()  # noqa: E731
    low, size = both(x) @ both(a[0]).t(), both(x).abs() @ both(a[0]).abs().t()
    want, far = low @ b[0].double().t(), size @ b[0].double().abs().t() * (2 * ends + rank + 3) * 2.0 ** -24
    assert ((y[:rows].double() - want).abs() <= far).all() and (y[rows:] == -9).all()
