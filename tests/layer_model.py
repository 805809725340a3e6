"""Plain models, in 64 bits where they compute, of the operators between a layer's products: the norm that readies
activations, the paged cache as it is written and read, and attention over it; and a Paged cache on the device with
its host copy, whose unwritten places hold NaN."""
import ctypes

import numpy as np

F = np.float32
SMALLEST = F(2.0 ** -100)
FORMS = {"int8": (0, np.int8), "f16": (1, np.float16)}


def norm(x, d, w, eps):
    """(r, y) of hq_norm_ready_ex: r in float32, y in float64"""
    r = x if d is None else (x + d).astype(F)
    r64 = r.astype(np.float64)
    ss = (r64 * r64).sum(-1, keepdims=True)
    with np.errstate(all="ignore"):
        inv = 1.0 / np.sqrt(ss / x.shape[-1] + float(F(eps)))
        return r, r64 * inv * w.astype(np.float64)


def quantized(x, form):
    """(elements, scales) of float32 vectors (.., dim) as a cache stores them"""
    x = np.asarray(x, F)
    with np.errstate(all="ignore"):
        most = np.max(np.abs(x), -1)
        bad = ~np.isfinite(x).all(-1)
        if form == "int8":
            scale = most / F(127)
        else:
            scale = np.where(most > 0, np.ldexp(F(1), np.frexp(most)[1] - 15), F(0)).astype(F)
        scale = np.where(scale < SMALLEST, F(0), scale).astype(F)
        inv = np.where(scale > 0, F(1) / scale, F(0)).astype(F)
        e = np.where((bad | (inv == 0))[..., None], F(0), x) * np.where(bad, F(0), inv)[..., None]
        e = np.rint(e).astype(np.int8) if form == "int8" else e.astype(np.float16)
        return e, np.where(bad, F(np.nan), scale).astype(F)


class Paged:
    """a cache of `pages` pages on the device and its host copy (k, v, ks, vs as hq.h lays them out), for sequences of
    `lengths` positions of which the last `new` are new tokens; `gone`: (sequence, page index) entries of the table that
    are no page, set to `gone_as`"""

    def __init__(self, pkg, arena, rng, form, heads, dim, page, lengths, new, gone=(), gone_as=-1, spare=2, extra_width=1,
                 longest=0):
        self.pkg, self.arena, self.form, self.heads, self.dim, self.page = pkg, arena, form, heads, dim, page
        self.lengths, self.new = list(lengths), list(new)
        counts = [-(-n // page) for n in lengths]
        self.width = max(counts, default=0) + extra_width
        self.pages = sum(counts) + spare
        order = list(rng.permutation(self.pages))
        self.table = np.full((len(lengths), self.width), gone_as, np.int32)
        for s, n in enumerate(counts):
            for i in range(min(n, self.width)):
                self.table[s, i] = order.pop()
        for s, i in gone:
            self.table[s, i] = gone_as
        code, kind = FORMS[form]
        # every place that is not written: NaN scales, and elements that are NaN (float16) or -128
        junk = np.int8(-128) if form == "int8" else np.float16(np.nan)
        self.k = np.full((self.pages, heads, page, dim), junk, kind)
        self.v = np.full((self.pages, heads, dim, page), junk, kind)
        self.ks = np.full((self.pages, heads, page), np.nan, F)
        self.vs = np.full((self.pages, heads, page), np.nan, F)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.at = {n: arena.put(getattr(self, n)) for n in ("k", "v", "ks", "vs")}
        self.cache = pkg.cache.Cache(self.at["k"], self.at["v"], self.at["ks"], self.at["vs"], code, self.pages, page,
                                     heads, dim)
        self.tokens = int(self.starts[-1])
        self.batch = pkg.cache.Batch(arena.put(self.starts), arena.put(np.asarray(lengths, np.int32)),
                                     arena.put(self.table), len(lengths), self.tokens, longest, self.width)

    def place(self, s, position):
        """(page, slot) of a position, or None"""
        i = position // self.page
        if position < 0 or i >= self.width or not 0 <= self.table[s, i] < self.pages:
            return None
        return int(self.table[s, i]), position % self.page

    def positions(self):
        """(token, sequence, position) of every new token"""
        for s, (n, length) in enumerate(zip(self.new, self.lengths)):
            for i in range(n):
                yield int(self.starts[s]) + i, s, length - n + i

    def put(self, s, position, k, v):
        """store float32 vectors (heads, dim) on the host copy"""
        at = self.place(s, position)
        if at is None:
            return
        page, slot = at
        self.k[page, :, slot], self.ks[page, :, slot] = quantized(k, self.form)
        self.v[page, :, :, slot], self.vs[page, :, slot] = quantized(v, self.form)

    def fill(self, rng, spread=0.5, every=True):
        """random vectors at every position of every sequence, on the host copy and the device"""
        gain = np.exp(spread * rng.standard_normal((self.heads, self.dim))).astype(F)
        for s, length in enumerate(self.lengths):
            for first in range(0, length, 512):  # (vectorised: the sequence's positions at once)
                at = [self.place(s, p) for p in range(first, min(first + 512, length))]
                k, ks = quantized(rng.standard_normal((len(at), self.heads, self.dim)).astype(F) * gain, self.form)
                v, vs = quantized(rng.standard_normal((len(at), self.heads, self.dim)).astype(F), self.form)
                keep = [i for i, a in enumerate(at) if a is not None]
                pages, slots = [at[i][0] for i in keep], [at[i][1] for i in keep]
                self.k[pages, :, slots], self.ks[pages, :, slots] = k[keep], ks[keep]
                self.v[pages, :, :, slots], self.vs[pages, :, slots] = v[keep], vs[keep]
        self.send()

    def send(self):
        for n, at in self.at.items():
            self.arena.write(at, getattr(self, n))

    def fetch(self, name):
        a = getattr(self, name)
        return self.arena.get(self.at[name], a.dtype, a.size).reshape(a.shape)

    def vectors(self, s, positions):
        """the float64 (keys, values) (positions, heads, dim) of a sequence, and which positions are on a page"""
        at = [self.place(s, p) for p in positions]
        k = np.zeros((len(at), self.heads, self.dim))
        v = np.zeros_like(k)
        for i, a in enumerate(at):
            if a is not None:
                k[i] = self.k[a[0], :, a[1]].astype(np.float64) * self.ks[a[0], :, a[1], None].astype(np.float64)
                v[i] = self.v[a[0], :, :, a[1]].astype(np.float64) * self.vs[a[0], :, a[1], None].astype(np.float64)
        return k, v, np.array([a is not None for a in at], bool)

    def attention(self, q, scale, window=0, cap=0.0):
        """(out, bound) in float64 of q (tokens, query heads, dim): the formula's output and how far a float32 kernel may
        be from it (see `bound` below)"""
        heads = q.shape[1]
        group = heads // self.heads
        out = np.zeros(q.shape)
        far = np.zeros(q.shape)
        held = {}
        for t, s, position in self.positions():
            if s not in held:
                held[s] = self.vectors(s, range(self.lengths[s]))
            k, v, there = held[s]
            lo = max(0, position + 1 - window) if window else 0
            seen = np.arange(lo, position + 1)
            seen = seen[there[lo:position + 1]] if position >= 0 else seen[:0]
            if not seen.size:
                continue
            for h in range(heads):
                kk, vv = k[seen, h // group], v[seen, h // group]
                qq = q[t, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    a = kk @ qq * float(F(scale))
                    # a score's error: its operands' 22 bits and its sum's roundings, over the sum of the products' sizes
                    size = np.max(np.abs(kk) @ np.abs(qq)) * float(F(scale))
                    if cap:
                        a = float(F(cap)) * np.tanh(a / float(F(cap)))
                    e = np.exp(a - np.max(a))
                    out[t, h] = (e[:, None] * vv).sum(0) / e.sum()
                    ds = size * (2.0 ** -21 + np.sqrt(self.dim) * 2.0 ** -23) + np.max(np.abs(a)) * 2.0 ** -22
                    # a weight's relative error is its score's (twice: numerator and sum), its own 22 bits, and the roundings
                    # of a sum over the positions as a random walk with a margin of 4
                    far[t, h] = np.max(np.abs(vv)) * (2 * ds + 2.0 ** -20 + np.sqrt(seen.size) * 2.0 ** -22)
        return out, far

    def run_attention(self, q, scale, window=0, cap=0.0, pad=0, stream=None):
        """hq_attention_ex of q (tokens, query heads, dim): rows `pad` bytes further apart than they are long"""
        lib, heads = self.pkg.library(), q.shape[1]
        row = heads * self.dim
        wide = np.full((max(1, self.tokens), row + pad // 4), 7, F)
        wide[:self.tokens, :row] = q.reshape(self.tokens, row)
        aq, ao = self.arena.put(wide), self.arena.put(np.full_like(wide, -5))
        need = lib.hq_attention_work_bytes(ctypes.byref(self.cache), ctypes.byref(self.batch), heads)
        assert need >= 0, lib.hq_last_error_message()
        work = self.arena.alloc(max(need, 256), fill=np.full(max(need, 256), 0xff, np.uint8))  # of any content
        stride = wide.shape[1] * 4
        status = lib.hq_attention_ex(ao, aq, heads, stride, stride, ctypes.byref(self.cache), ctypes.byref(self.batch),
                                     scale, window, cap, work, need, stream)
        assert status == 0, lib.hq_last_error_message()
        got = self.arena.get(ao, F, wide.size).reshape(wide.shape)
        assert (got[:, row:] == -5).all(), "wrote between the rows"
        return got[:self.tokens, :row].reshape(q.shape)
