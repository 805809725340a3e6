"""A checkpoint's layers over a paged cache (pyodide-llm_amd/forward.py), every call on what the calls before it gave: the
products and the activations readied for them by the oracle, to the bit; residual sums to the bit; norms, rotation, gate and
attention in 64 bits.  (What a whole step gives is not compared with 64 bits: a quantized activation that lies between two
steps goes either way by a float32's last bit, and a softmax of large scores makes that any size.)

How far: a norm is the 64-bit one rounded once, 2^-24 of a value, and as readied at most a step of some element from it;
rotation and gate are a few float32 roundings (2^-20 of the largest); a score's error is (dim + 4) 2^-22 of sum |q k|, dim
products held to 22 bits and their sum, and a weight's twice that, relative; beside it 2^-18 of the largest value."""
import numpy as np
import pytest

import checkpoints
from gpu_util import same_bits
from layer_model import norm, quantized
from test_gpu_checkpoint import activations, file_tensor, product

pytestmark = pytest.mark.gpu
F = np.float32
EPS = 1e-5


def turned(x, position):
    """pairs of neighbouring values by their position's angles, in 64 bits"""
    heads, dim = x.shape
    angle = position * 10000.0 ** -(np.arange(0, dim, 2) / dim)
    pairs = x.astype(np.float64).reshape(heads, -1, 2)
    z = (pairs[..., 0] + 1j * pairs[..., 1]) * np.exp(1j * angle)
    return np.stack([z.real, z.imag], -1).reshape(heads, dim)


def near(got, want, far):
    assert (np.abs(got - want) <= far).all(), np.abs(got - want).max()


def watched(forward, oracle, data, where):
    """a Forward that checks each of its calls when it is made; .new: the step's (sequence, position) of each row"""
    class Watched(forward.Forward):
        def __init__(self, ck, **sizes):
            super().__init__(ck, **sizes)
            self.tensors = {name: file_tensor(data, where, name) for name in ck.matrices}
            self.cached, self.seen, self.calls = {}, {}, 0

        def host(self, t, count):
            self.torch.cuda.synchronize()
            return t[:count].cpu().numpy().copy()

        def norm(self, x, given, weight, count, stream, y=None):
            before = self.host(x, count), given is not None and self.host(given, count)
            super().norm(x, given, weight, count, stream, y)
            r, want = norm(before[0], before[1] if given is not None else None, self.host(weight, len(weight)), EPS)
            assert same_bits(self.host(x, count), r)
            if y is not None:
                near(self.host(y, count), want, 2.0 ** -23 * np.abs(want))
            else:
                self.normed = want.astype(F)

        def readied(self, n, count):
            frames = self.host(self.xq, count * self.frames[n]).reshape(count, -1)
            return [(f[:n], f[n:n + (n // 4 if self.ready == 2 else n // 8)].view(F)) for f in frames]

        def products(self, names, layer, x, outs, count, stream, readied):
            if names[0] == "wo":
                self.attended(layer, x, count)
            if names[0] == "w2":
                a, b = (self.seen[name].astype(np.float64) for name in ("w1", "w3"))
                want = a / (1 + np.exp(-a)) * b
                near(self.host(x, count), want, 2.0 ** -20 * np.abs(want) + 1e-30)
            super().products(names, layer, x, outs, count, stream, readied)
            n = self.ck.matrices[names[0]].n
            took = self.readied(n, count)
            rows = self.normed if readied else self.host(x, count)
            for row, (xq, xs) in zip(rows.reshape(count, n), took):
                want = activations(oracle, row, self.ck.dtype)
                if readied:  # (the norm's last bit)
                    assert np.abs(want[0].view(np.int8).astype(int) - xq.view(np.int8)).max() <= 1
                    near(xs[:n // 32], want[1][:n // 32], 2.0 ** -22 * want[1][:n // 32])
                else:
                    assert np.array_equal(want[0].view(np.uint8), xq.view(np.uint8)) and same_bits(xs, want[1])
            for name, out in zip(names, outs):
                m = self.ck.matrices[name]
                values, scales = (t.reshape(m.layers, -1)[layer] for t in self.tensors[name])
                got = self.host(out, count).reshape(count, -1)
                for row, (xq, xs) in zip(got, took):
                    xq = xq.view(np.int8) if self.ready == 2 else xq
                    assert same_bits(row, product(oracle, self.ck.dtype, xq, xs, values, scales, n)), name
                self.seen[name] = got
                self.calls += 1

        def attended(self, layer, x, count):
            s = self.ck.shape
            q, k, v, out = (self.host(t, count) for t in (self.q, self.k, self.v, x))
            for row, (sequence, position) in enumerate(self.new):
                for t, name in ((q, "wq"), (k, "wk")):
                    was = self.seen[name][row].reshape(-1, s.head_size)
                    near(t[row], turned(was, position), 2.0 ** -20 * np.abs(was).max())
                keys, values = self.cached.setdefault((sequence, layer), ([], []))
                for held, t in ((keys, k), (values, v)):
                    e, scale = quantized(t[row], self.form)
                    held.append(e.astype(np.float64) * scale[:, None].astype(np.float64))
                assert len(keys) == position + 1
                for h in range(s.heads):
                    kv = h // (s.heads // s.kv_heads)
                    ks, vs = np.array([t[kv] for t in keys]), np.array([t[kv] for t in values])
                    u = ks @ q[row, h].astype(np.float64) / np.sqrt(s.head_size)
                    p = np.exp(u - u.max())
                    off = (np.abs(ks) @ np.abs(q[row, h].astype(np.float64))).max() / np.sqrt(s.head_size)
                    near(out[row, h], p @ vs / p.sum(),
                         (2 * (s.head_size + 4) * 2.0 ** -22 * off + 2.0 ** -18) * np.abs(vs).max())
    return Watched


@pytest.mark.parametrize("dtype, header, form", [
    ("int8", (288, 768, 2, 6, 6, 100, 64), "int8"), ("int8", (512, 1024, 2, 8, 2, 100, 64), "f16"),
    ("int6", (256, 768, 2, 4, 2, 100, 64), "int8"), ("ternary", (256, 768, 2, 4, 4, 100, 64), "int8"),
    ("binary", (384, 1024, 2, 6, 2, 100, 64), "f16")])
def test_steps(pkg, oracle, dtype, header, form):
    import torch
    from pyodide_llm_amd import checkpoint, forward
    rng = np.random.default_rng(header[0] + len(dtype))
    data, where = checkpoints.write(header, dtype, rng)
    ck = checkpoint.Checkpoint(data)
    page, width = 16, 5
    model = watched(forward, oracle, data, where)(ck, tokens=64, sequences=3, pages=16, width=width, page=page, form=form)
    table = torch.from_numpy(rng.permutation(16)[:3 * width].reshape(3, width).astype(np.int32)).cuda()
    held = [0, 0, 0]
    # prompts together, then a token each, then a mixture: a few tokens, none, a longer piece
    for new in ([33, 1, 7], [1, 1, 1], [3, 0, 20]):
        x = (rng.standard_normal((sum(new), header[0])) * 0.5).astype(F)
        held = [a + b for a, b in zip(held, new)]
        starts = np.cumsum([0] + new).astype(np.int32)
        model.new = [(s, held[s] - new[s] + i) for s in range(3) for i in range(new[s])]
        y = model.step(torch.from_numpy(x.copy()).cuda(), torch.from_numpy(starts).cuda(),
                       torch.tensor(held, dtype=torch.int32, device="cuda"), table, max(new))
        assert tuple(y.shape) == x.shape and bool(torch.isfinite(y).all())
    assert model.calls == 3 * 2 * 7


def test_refused(pkg, oracle):
    import torch
    from pyodide_llm_amd import checkpoint, forward
    rng = np.random.default_rng(1)
    ck = checkpoint.Checkpoint(checkpoints.write((256, 768, 1, 4, 2, 100, 64), "int8", rng)[0])
    model = forward.Forward(ck, tokens=4, sequences=2, pages=4, width=2, page=16)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    x, table = torch.zeros(2, 256, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for bad in ((torch.zeros(5, 256, device="cuda"), ints(0, 4, 5), ints(4, 1), table), (x, ints(0, 1), ints(1, 1), table),
                (x, ints(0, 1, 2), ints(1, 1), table[:, :1]), (x, ints(0, 1, 2).long(), ints(1, 1), table),
                (x[:, :128], ints(0, 1, 2), ints(1, 1), table)):
        with pytest.raises(ValueError, match="refused"):
            model.step(*bad)
