"""hq_batch_plan_ex and hq_pages_give_ex against a model that walks the sequences one by one, number for number."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
JUNK = -77


def plan(held, fresh, free, count, table, tokens, page, pages):
    """starts, lengths, table, left, missing, sequence, position, slot"""
    table, starts, lengths = table.copy(), [0], []
    sequence, position, slot = (np.full(tokens, -1, np.int64) for _ in range(3))
    count, missing = min(max(count, 0), pages), 0
    width = table.shape[1]
    for s, (h, f) in enumerate(zip(held, fresh)):
        h, f = max(int(h), 0), max(int(f), 0)
        f = min(f, tokens - starts[-1])
        for entry in range(-(-h // page), min(-(-(h + f) // page), width)):
            if count:
                count -= 1
                table[s, entry] = free[count]
            else:
                missing += 1
                table[s, entry] = -1
        for i in range(f):
            t, at = starts[-1] + i, h + i
            sequence[t], position[t] = s, at
            if at // page < width and 0 <= table[s, at // page] < pages:
                slot[t] = int(table[s, at // page]) * page + at % page
        starts.append(starts[-1] + f)
        lengths.append(h + f)
    return dict(starts=starts, lengths=lengths, table=table, left=[count], missing=[missing], sequence=sequence, position=position,
                slot=slot)


class Step:
    """a step's arrays on the device"""

    def __init__(self, pkg, held, fresh, free, count, table, tokens, page, pages, in_place=False, maps=(1, 1, 1), missing=True):
        import torch
        put = lambda a: torch.tensor(np.asarray(a, np.int32).reshape(-1), device="cuda")  # noqa: E731
        blank = lambda n, kind=torch.int32: torch.full((n,), JUNK, dtype=kind, device="cuda")  # noqa: E731
        self.pkg, n = pkg, len(held)
        self.held, self.fresh, self.free, self.count, self.table = put(held), put(fresh), put(free), put([count]), put(table)
        self.starts, self.lengths = blank(n + 1), self.held if in_place else blank(n)
        self.left, self.missing = self.count if in_place else blank(1), blank(1)
        self.sequence, self.position, self.slot = blank(tokens + 1), blank(tokens + 1), blank(tokens + 1, torch.int64)
        at = lambda t, there=True: t.data_ptr() if there else None  # noqa: E731
        self.batch = pkg.cache.Batch(at(self.starts), at(self.lengths), at(self.table), n, tokens, 0, table.shape[1])
        self.pool = pkg.cache.Pool(at(self.free), at(self.count), at(self.left), at(self.missing, missing), pages, page)
        self.rest = (at(self.held), at(self.fresh), *(at(t, m) for t, m in zip((self.sequence, self.position, self.slot), maps)))
        torch.cuda.synchronize()

    def run(self, stream=None):
        status = self.pkg.library().hq_batch_plan_ex(self.batch, self.pool, *self.rest, stream)
        assert status == 0, self.pkg.library().hq_last_error_message()

    def check(self, want, skip=()):
        import torch
        torch.cuda.synchronize()
        for name, value in want.items():
            got = getattr(self, name).cpu().numpy()
            value = np.asarray(value).reshape(-1)
            if name in skip:
                assert (got == JUNK).all(), name
                continue
            assert np.array_equal(got[:len(value)], value), (name, got[:len(value)][got[:len(value)] != value][:5])
            assert (got[len(value):] == JUNK).all(), f"{name}: wrote past its end"


def case(rng, sequences, most, page, spare=3, slack=4, width_less=0):
    held = rng.integers(0, 5 * page, sequences) * (rng.random(sequences) < 0.8)
    held = np.where(rng.random(sequences) < 0.2, held // page * page, held)
    fresh = rng.integers(0, most + 1, sequences) * (rng.random(sequences) < 0.9)
    had, need = -(-held // page), -(-(held + fresh) // page)
    pages = int(need.sum()) + 6
    width = max(1, int(need.max(initial=0)) + 2 - width_less)
    order = rng.permutation(pages)
    table = rng.integers(-5, 3, (sequences, width))  # (stale entries behind a row's pages)
    for s, n in enumerate(had):
        table[s, :min(n, width)] = order[:n][:width]
        order = order[n:]
    free = np.concatenate([order, np.full(pages - len(order), JUNK)])
    count = min(len(order), max(0, int((need - had).sum()) + spare))
    return dict(held=held, fresh=fresh, free=free, count=count, table=table, tokens=int(fresh.sum()) + slack, page=page, pages=pages)


def both(pkg, c, **more):
    step = Step(pkg, **c, **more)
    want = plan(**{k: c[k] for k in ("held", "fresh", "free", "count", "table", "tokens", "page", "pages")})
    step.run()
    return step, want


@pytest.mark.parametrize("sequences", [1, 2, 31, 64, 65, 255, 256, 257, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("most, page", [(1, 64), (5, 16), (200, 32)])
def test_plans(pkg, sequences, most, page):
    c = case(np.random.default_rng(sequences + most), sequences, most, page)
    step, want = both(pkg, c)
    step.check(want)


@pytest.mark.parametrize("sequences, most", [(3, 5000), (1, 40000), (40, 3000), (9000, 3)])
def test_long_prompts_and_many_sequences(pkg, sequences, most):
    c = case(np.random.default_rng(sequences), sequences, most, 16)
    step, want = both(pkg, c)
    step.check(want)


@pytest.mark.parametrize("sequences", [5, 300, 1500])
@pytest.mark.parametrize("page", [16, 128, 256])
def test_in_place(pkg, sequences, page):
    """lengths over held, what is left over the count: a serving loop's arrays, several steps"""
    rng = np.random.default_rng(sequences + page)
    c = case(rng, sequences, 30, page, spare=400)
    step = Step(pkg, **c, in_place=True)
    for _ in range(4):
        want = plan(**c)
        step.run()
        step.check(want)
        c.update(held=np.array(want["lengths"]), count=want["left"][0], table=want["table"])


@pytest.mark.parametrize("spare", [-1, -7, -10 ** 6])
@pytest.mark.parametrize("sequences", [1, 40, 1200])
def test_a_stack_that_runs_out(pkg, spare, sequences):
    c = case(np.random.default_rng(sequences - spare), sequences, 60, 16, spare=spare)
    step, want = both(pkg, c)
    step.check(want)


def test_tokens_that_do_not_fit(pkg):
    """more new tokens than the batch has rows: the last sequences' are left out; negative numbers count as none"""
    rng = np.random.default_rng(2)
    for less in (1, 50, 10 ** 6):
        c = case(rng, 70, 40, 16, slack=-less)
        c["tokens"] = max(c["tokens"], 0)
        c["fresh"][::7], c["held"][::9] = -3, -(2 ** 31)
        step, want = both(pkg, c)
        step.check(want)
    c["fresh"][:] = 2 ** 31 - 1
    step, want = both(pkg, c)
    step.check(want)


def test_a_table_that_is_too_narrow(pkg):
    """positions past the table take no page and have no slot"""
    c = case(np.random.default_rng(4), 50, 100, 16, width_less=5)
    step, want = both(pkg, c)
    step.check(want)
    c["table"] = np.zeros((50, 0), int)
    step, want = both(pkg, c)
    step.check(want)


def test_counts_and_pages_that_are_none(pkg):
    """a count past the stack, and a negative one; numbers on the stack that are no page go into the table and have no slot"""
    c = case(np.random.default_rng(5), 20, 60, 16)
    for count in (-5, 2 ** 31 - 1):
        c["count"] = count
        c["free"][::3] = 2 ** 30
        step, want = both(pkg, c)
        step.check(want)
    c["pages"], c["free"] = 0, np.zeros(0, int)
    step, want = both(pkg, c)
    step.check(want)


@pytest.mark.parametrize("maps", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1)])
def test_maps_that_are_not_wanted(pkg, maps):
    c = case(np.random.default_rng(6), 33, 40, 32)
    step, want = both(pkg, c, maps=maps, missing=False)
    step.check(want, skip=[n for n, m in zip(("sequence", "position", "slot"), maps) if not m] + ["missing"])


def test_no_sequences(pkg):
    c = dict(held=np.zeros(0, int), fresh=np.zeros(0, int), free=np.arange(4), count=3, table=np.zeros((0, 5), int), tokens=9, page=16, pages=4)
    step, want = both(pkg, c)
    step.check(want)
    c["tokens"] = 0
    step, want = both(pkg, c)
    step.check(want)


def test_far_positions(pkg):
    """positions up to the end of a table of 2^30, and slots past 32 bits"""
    held = np.array([2 ** 30 - 3, 2 ** 28 + 1])
    c = dict(held=held, fresh=np.array([3, 5]), free=np.array([2 ** 26 - 1, 7, 2 ** 26 - 2]), count=3, tokens=8, page=256, pages=2 ** 26)
    import torch
    width = 2 ** 22
    table = torch.full((2, width), 2 ** 26 - 5, dtype=torch.int32, device="cuda")
    want_slot = [(2 ** 26 - 5) * 256 + (h + i) % 256 for h, f in zip(held, c["fresh"]) for i in range(f)]
    small = dict(c, table=np.zeros((2, 1), int), pages=3, free=np.array([0, 1, 2]))
    step = Step(pkg, **small)
    free = torch.tensor(c["free"], dtype=torch.int32, device="cuda")
    # (the stack's memory is as large as its few numbers: count says 3 of 2^26 pages)
    step.batch = pkg.cache.Batch(step.starts.data_ptr(), step.lengths.data_ptr(), table.data_ptr(), 2, 8, 0, width)
    step.pool = pkg.cache.Pool(free.data_ptr(), step.count.data_ptr(), step.left.data_ptr(), step.missing.data_ptr(), 2 ** 26, 256)
    step.run()
    step.check(dict(lengths=held + c["fresh"], position=[2 ** 30 - 3, 2 ** 30 - 2, 2 ** 30 - 1] + [2 ** 28 + 1 + i for i in range(5)],
                    slot=want_slot, left=[3], missing=[0]))


def give(table, free, count, pages, first, last):
    table, free = table.copy(), free.copy()
    count = min(max(count, 0), pages)
    for s in range(len(table)):
        for e in range(max(first[s], 0) if first is not None else 0, min(last[s], table.shape[1]) if last is not None else table.shape[1]):
            if 0 <= table[s, e] < pages:
                if count < pages:
                    free[count] = table[s, e]
                count = min(count + 1, pages)
                table[s, e] = -1
    return table, free, count


@pytest.mark.parametrize("sequences, width", [(1, 1), (3, 7), (40, 64), (64, 1030), (1500, 5), (700, 70), (2, 5000)])
@pytest.mark.parametrize("ranges", ["all", "from", "to", "both"])
def test_pages_given_back(pkg, sequences, width, ranges):
    import torch
    rng = np.random.default_rng(sequences + width)
    pages = sequences * width + 10
    table = rng.permutation(pages)[:sequences * width].reshape(sequences, width)
    table[rng.random(table.shape) < 0.3] = -1
    table[rng.random(table.shape) < 0.05] = pages
    count = int(rng.integers(0, 10))
    free = np.full(pages + 1, JUNK)
    free[:count] = 5
    first = rng.integers(-2, width + 2, sequences) if ranges in ("from", "both") else None
    last = rng.integers(-2, width + 3, sequences) if ranges in ("to", "both") else None
    put = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    for left_is_count in (False, True):
        at, af, ac, al = put(table), put(free), put([count]), put([JUNK])
        a, b = (None if v is None else put(v) for v in (first, last))
        torch.cuda.synchronize()
        pool = pkg.cache.Pool(af.data_ptr(), ac.data_ptr(), (ac if left_is_count else al).data_ptr(), None, pages, 16)
        status = pkg.library().hq_pages_give_ex(pool, at.data_ptr(), sequences, width, a.data_ptr() if a is not None else None,
                                                b.data_ptr() if b is not None else None, None)
        assert status == 0
        torch.cuda.synchronize()
        want = give(table, free, count, pages, first, last)
        assert np.array_equal(at.cpu().numpy(), want[0]) and np.array_equal(af.cpu().numpy(), want[1])
        assert int((ac if left_is_count else al)) == want[2]


def test_a_full_stack_drops_pages(pkg):
    """a page that two entries hold is put on the stack twice, and what does not fit is dropped"""
    import torch
    put = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table, free, count = put([[0, 1, 1, 2], [3, -1, 0, 9]]), put([7, JUNK, JUNK, JUNK, JUNK]), put([1])
    pool = pkg.cache.Pool(free.data_ptr(), count.data_ptr(), count.data_ptr(), None, 4, 16)
    torch.cuda.synchronize()
    assert pkg.library().hq_pages_give_ex(pool, table.data_ptr(), 2, 4, None, None, None) == 0
    torch.cuda.synchronize()
    assert table.tolist() == [[-1, -1, -1, -1], [-1, -1, -1, 9]] and free.tolist() == [7, 0, 1, 1, JUNK] and count.item() == 4


def test_replayed(pkg):
    """a captured plan in place: every replay is a step further"""
    import torch
    rng = np.random.default_rng(12)
    c = case(rng, 200, 1, 16, spare=4000)
    c["tokens"] = 200
    c["table"] = np.concatenate([c["table"], np.full((200, 30), -1)], 1)
    pages = c["pages"] + 4000
    c["free"] = np.concatenate([c["free"][:c["count"]], np.arange(c["pages"], pages), np.full(pages - c["count"] - 4000, JUNK)])
    c["count"], c["pages"] = c["count"] + 4000, pages
    step = Step(pkg, **c, in_place=True)
    assert pkg.library().hq_init() == 0
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        step.run(stream.cuda_stream)
    for replay in range(5):
        c["fresh"] = rng.integers(0, 3, 200) * (replay % 2) + 1 - replay % 2
        step.fresh.copy_(torch.tensor(c["fresh"], dtype=torch.int32))
        torch.cuda.synchronize()
        want = plan(**c)
        g.replay()
        step.check(want)
        c.update(held=np.array(want["lengths"]), count=want["left"][0], table=want["table"])
