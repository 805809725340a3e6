"""Requests served step by step (pyodide-llm_amd/serve.py): places and pages, embeddings, layers with adapters, the classifier and
the drawn tokens together, over steps of prompts and single tokens, requests that end and pages that other requests get.

Each step's logits are compared, to the bit, with a Forward of its own driven by hand (its starts, lengths, positions and table made
on the host, other pages); every call of adapters with the formula in 64 bits: an output is off by the roundings of n and of
`rank` products and sums, (n + rank + 3) 2^-24 of the sum of their sizes; the drawn tokens with a plain draw in 64 bits."""
import numpy as np
import pytest

import checkpoints
from gpu_util import same_bits
from test_gpu_checkpoint import file_tensor
from test_gpu_sample import model as drawn
from test_gpu_sample import near

pytestmark = pytest.mark.gpu
F = np.float32


def factors(torch, ck, rng, count, rank, names, kind):
    made = {}
    for name in names:
        m = ck.matrices[name]
        a = rng.standard_normal((m.layers, count, rank, m.n)) / np.sqrt(m.n)
        b = rng.standard_normal((m.layers, count, m.rows, rank)) / np.sqrt(rank)
        made[name] = tuple(torch.from_numpy(t.astype(F)).to(kind).cuda() for t in (a, b))
    return made


def watched(forward):
    class Watched(forward.Forward):
        seen = 0

        def adapt(self, adapters, names, layer, x, outs, batch, which, stream):
            host = lambda t: t.detach().float().cpu().numpy().astype(np.float64)
            before = [t.clone() for t in outs]
            super().adapt(adapters, names, layer, x, outs, batch, which, stream)
            starts, whose = self.starts, which.cpu().numpy()
            for name, was, now in zip(names, before, outs):
                was, now = (t.reshape(t.shape[0], -1) for t in (was, now))
                for s, w in enumerate(whose):
                    rows = slice(starts[s], starts[s + 1])
                    if name not in adapters.factors or not 0 <= w < adapters.count:
                        assert same_bits(now[rows].cpu().numpy(), was[rows].cpu().numpy())
                        continue
                    a, b = (host(t[layer, w]) for t in adapters.factors[name])
                    scale = 1.0 if adapters.scales is None else float(adapters.scales[w])
                    e = host(x[rows]).reshape(starts[s + 1] - starts[s], a.shape[1])
                    want = host(was[rows]) + scale * (e @ a.T) @ b.T
                    size = np.abs(host(was[rows])) + abs(scale) * (np.abs(e) @ np.abs(a).T) @ np.abs(b).T
                    far = (a.shape[1] + a.shape[0] + 3) * 2.0 ** -24 * size
                    assert (np.abs(host(now[rows]) - want) <= far).all(), name
                    self.seen += 1
    return Watched


@pytest.mark.parametrize("dtype, header, kind", [
    ("int8", (288, 768, 2, 6, 6, 1000, 64), None), ("int8", (256, 768, 2, 4, 2, 9000, 64), "bfloat16"),
    ("ternary", (256, 768, 2, 4, 4, 300, 64), "float16"), ("int6", (256, 768, 1, 4, 2, 300, 64), "float16"),
    ("binary", (384, 1024, 1, 6, 2, 300, 64), None)])
def test_requests(pkg, dtype, header, kind):
    import torch
    from pyodide_llm_amd import adapters, checkpoint, forward, serve
    rng = np.random.default_rng(header[0] + len(dtype))
    norm = 1 + rng.standard_normal(header[0]).astype(F) * 0.1
    norm[[3, 17, 100]] = 40.0  # (a classifier with channels apart)
    data, where = checkpoints.write(header, dtype, rng, norm)
    ck = checkpoint.Checkpoint(data)
    vocab, n, page, width, pages = header[5], 4, 16, 4, 9
    sizes = dict(tokens=48, sequences=n, pages=pages, width=width, page=page)
    model = watched(forward)(ck, **sizes)
    beside = None
    if kind:
        beside = adapters.Adapters(factors(torch, ck, rng, 3, 16, ("wq", "wv", "wo", "w1", "w3", "w2"), getattr(torch, kind)),
                                   torch.tensor([1.0, -0.5, 2.0], device="cuda"))
    serving = serve.Serving(model, beside)
    plain = forward.Forward(ck, **{**sizes, "pages": n * width})
    table = torch.from_numpy(rng.permutation(n * width).reshape(n, width).astype(np.int32)).cuda()
    assert ck.channels
    which = np.array([0, -1, 2, 7], np.int32)
    serving.which.copy_(torch.from_numpy(which))
    setting = dict(temperature=[0.0, 1.0, 0.7, 1.3], top_k=[0, 0, 20, 0], top_p=[1.0, 0.9, 1.0, 0.8], min_p=[0.0, 0.0, 0.05, 0.0])
    for name, v in setting.items():
        getattr(serving, name).copy_(torch.tensor(v))
    held = np.zeros(n, int)
    last = np.full(n, -1)
    steps = [([33, 1, 0, 7], []), ([1, 1, 0, 1], []), ([1, 0, 40, 1], [0]), ([20, 1, 1, 1], [2, 3]), ([1, 1, 15, 2], [])]
    for new, ends in steps:
        ids = np.concatenate([[last[s]] if k == 1 and last[s] >= 0 else rng.integers(0, vocab, k) for s, k in enumerate(new)])
        ids = ids.astype(np.int32)
        u = rng.random(n).astype(F)
        model.starts = np.cumsum([0] + new)
        held += new
        longest = max(new)
        got = serving.step(torch.from_numpy(ids).cuda(), torch.tensor(new, dtype=torch.int32, device="cuda"),
                           torch.from_numpy(u).cuda(), longest).cpu().numpy()
        assert serving.missing.item() == 0 and (serving.lengths.cpu().numpy() == held).all()
        assert serving.left.item() == pages - sum(-(-h // page) for h in held)
        t = serving.table.cpu().numpy()
        used = np.concatenate([t[s, :-(-held[s] // page)] for s in range(n)])
        assert len(set(used)) == len(used) and (0 <= used).all() and (used < pages).all()
        # by hand: embeddings on the host (where the file's int8 rows are read easily), places and pages of its own
        x = torch.empty(len(ids), header[0], device="cuda")
        if dtype == "int8":
            values, scales = file_tensor(data, where, "token_embedding_table")
            rows = (values.view(np.int8).reshape(-1, 32).astype(F) * scales.view(F)[:, None]).reshape(vocab, -1)
            x.copy_(torch.from_numpy(rows[ids]))
        else:
            plain.embed(torch.from_numpy(ids).cuda(), x)
        starts = torch.from_numpy(model.starts.astype(np.int32)).cuda()
        lengths = torch.from_numpy(held.astype(np.int32)).cuda()
        extra = () if beside is None else (None, beside, serving.which)
        y = plain.step(x, starts, lengths, table, longest, *extra)
        scores = serving.scores.cpu().numpy()
        chance = serving.chance.cpu().numpy()
        for s in range(n):
            if not new[s]:
                assert got[s] == -1
                continue
            row, logits = y[model.starts[s + 1] - 1].clone(), torch.empty(vocab, device="cuda")
            ck.classify(row.data_ptr(), logits.data_ptr(), plain.xq.data_ptr(), torch.cuda.current_stream())
            assert same_bits(logits.cpu().numpy(), scores[s])
            want, share = drawn(scores[s], u=u[s], **{k: v[s] for k, v in setting.items()})
            assert got[s] == want and near(chance[s], share)
        last = np.where(np.array(new) > 0, got, last)
        if ends:
            done = torch.zeros(n, dtype=torch.bool, device="cuda")
            done[ends] = True
            serving.finish(done)
            held[ends], last[ends] = 0, -1
            assert serving.left.item() == pages - sum(-(-h // page) for h in held)
    assert not kind or model.seen


def test_pages_that_lack(pkg):
    """a step that needs more pages than there are says so; the others' answers are theirs"""
    import torch
    from pyodide_llm_amd import checkpoint, forward, serve
    rng = np.random.default_rng(3)
    ck = checkpoint.Checkpoint(checkpoints.write((256, 768, 1, 4, 2, 300, 64), "int8", rng)[0])
    ids = torch.from_numpy(rng.integers(0, 300, 40).astype(np.int32)).cuda()
    fresh, u = torch.tensor([10, 30], dtype=torch.int32, device="cuda"), torch.full((2,), 0.5, device="cuda")
    first = []
    for pages in (3, 2):
        serving = serve.Serving(forward.Forward(ck, tokens=40, sequences=2, pages=pages, width=4, page=16))
        for t in serving.forward.held[0]:
            t.zero_()
        first.append(serving.step(ids, fresh, u, 30)[0].item())
        assert serving.missing.item() == 3 - pages and serving.left.item() == 0
    assert first[0] == first[1]


@pytest.mark.parametrize("kind", [None, "float16"])
def test_steps_replayed(pkg, kind):
    """single tokens by a captured step, each replay's answers the eager steps' to the bit"""
    import torch
    from pyodide_llm_amd import adapters, checkpoint, forward, serve
    rng = np.random.default_rng(4)
    ck = checkpoint.Checkpoint(checkpoints.write((256, 768, 2, 4, 2, 9000, 64), "int8", rng)[0])
    beside = adapters.Adapters(factors(torch, ck, rng, 2, 8, ("wq", "w2"), getattr(torch, kind))) if kind else None
    n, prompts = 3, [5, 1, 30]
    serves = [serve.Serving(forward.Forward(ck, tokens=36, sequences=n, pages=12, width=4, page=16), beside) for _ in range(2)]
    ids = torch.from_numpy(rng.integers(0, 9000, 36).astype(np.int32)).cuda()
    fresh, ones = torch.tensor(prompts, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
    u = torch.rand(n, device="cuda")
    tokens = []
    for serving in serves:
        serving.which.copy_(torch.tensor([0, 1, -1]))
        serving.step(ids, fresh, u, 30)
        serving.step(serving.tokens.clone(), ones, u, 1)  # (a step of these sizes has run)
        tokens.append(serving.tokens.clone())
    assert torch.equal(*tokens)
    eager, other = serves
    taken, numbers = tokens[1].clone(), u.clone()
    torch.cuda.synchronize()
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        taken.copy_(other.step(taken, ones, numbers, 1))
    for _ in range(5):
        u = torch.rand(n, device="cuda")
        eager.step(eager.tokens.clone(), ones, u, 1)
        numbers.copy_(u)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.tokens, taken) and torch.equal(eager.scores, other.scores)
        assert torch.equal(eager.lengths, other.lengths) and torch.equal(eager.table, other.table)


def test_a_captured_step_keeps_its_workspace(pkg):
    """a longer step of many more tokens, which needs a larger workspace, runs between a captured step's replays; a step whose
    workspace is not there is not captured"""
    import torch
    from pyodide_llm_amd import checkpoint, forward, serve
    rng = np.random.default_rng(6)
    ck = checkpoint.Checkpoint(checkpoints.write((256, 768, 1, 4, 2, 300, 64), "int8", rng)[0])
    n = 2
    serves = [serve.Serving(forward.Forward(ck, tokens=1500, sequences=n, pages=64, width=30, page=64)) for _ in range(2)]
    ids = torch.from_numpy(rng.integers(0, 300, 1400).astype(np.int32)).cuda()
    ones, u = torch.ones(n, dtype=torch.int32, device="cuda"), torch.rand(n, device="cuda")
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    eager, other = serves
    for serving in serves:
        serving.step(ids[:2], ones, u, 1)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        other.step(ids[:2], ones, u, 1)
    was = other.forward.work.numel()
    for many in (900, 1, 200):
        eager.step(ids[:2], ones, u, 1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.scores, other.scores) and torch.equal(eager.tokens, other.tokens)
        fresh = torch.tensor([many, 100], dtype=torch.int32, device="cuda")
        for serving in serves:
            serving.step(ids[:many + 100], fresh, u, max(many, 100))
        if many == 900:
            held = [torch.full((was,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]  # (what a freed one would become)
        assert torch.equal(eager.scores, other.scores)
        serves[0].finish(torch.ones(n, dtype=torch.bool, device="cuda"))
        serves[1].finish(torch.ones(n, dtype=torch.bool, device="cuda"))
    assert other.forward.work.numel() > was and all((t == 255).all() for t in held)


@pytest.mark.parametrize("kind", [None, "bfloat16"])
def test_a_first_step_is_captured(pkg, kind):
    """a step whose workspace is not there yet makes it in its graph; larger steps between its replays"""
    import torch
    from pyodide_llm_amd import adapters, checkpoint, forward
    rng = np.random.default_rng(8)
    ck = checkpoint.Checkpoint(checkpoints.write((256, 768, 2, 4, 2, 300, 64), "int8", rng)[0])
    beside = adapters.Adapters(factors(torch, ck, rng, 2, 64, ("wq", "w2"), getattr(torch, kind))) if kind else None
    eager, other = (forward.Forward(ck, tokens=1500, sequences=2, pages=64, width=32, page=64) for _ in range(2))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, which = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32), ints(1, 0)
    starts, lengths, x = ints(0, 1, 2), ints(1, 1), torch.zeros(2, 256, device="cuda")
    extra = (None, beside, which) if kind else ()
    eager.step(torch.zeros_like(x), starts, lengths, table, 1, *extra)  # (the library has run; `other` has not)
    torch.cuda.synchronize()
    assert other.work.numel() == 0
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        taken = other.step(x, starts, lengths, table, 1, *extra)
    first = other.work
    held = np.zeros(2, int)
    for many in (0, 700, 3, 1100):
        held += 1
        new = torch.from_numpy(rng.standard_normal((2, 256)).astype(F)).cuda()
        x.copy_(new)
        lengths.copy_(ints(*held))
        want = eager.step(new, starts, lengths, table, 1, *extra).clone()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, taken)
        if many:
            rows = torch.from_numpy(rng.standard_normal((many + 1, 256)).astype(F)).cuda()
            held += [many, 1]
            got = [m.step(rows.clone(), ints(0, many, many + 1), ints(*held), table, many, *extra) for m in (eager, other)]
            assert torch.equal(*got)
    assert other.work is not first and any(t is first for t in other.older)


def test_workspaces_are_what_steps_need(pkg):
    """a workspace that no captured step uses is not kept, and none is larger than a step needed"""
    import torch
    from pyodide_llm_amd import checkpoint, forward
    rng = np.random.default_rng(9)
    ck = checkpoint.Checkpoint(checkpoints.write((256, 768, 1, 4, 2, 300, 64), "int8", rng)[0])
    model = forward.Forward(ck, tokens=1500, sequences=1, pages=32, width=32, page=64)
    table, most = torch.arange(32, dtype=torch.int32, device="cuda")[None], 0
    for many in (1, 500, 600, 1500, 20):
        starts, lengths = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, many], [many]))
        model.step(torch.zeros(many, 256, device="cuda"), starts, lengths, table, many)
        batch = pkg.cache.Batch(starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), 1, many, many, 32)
        most = max(most, pkg.library().hq_attention_work_bytes(model.caches[0], batch, 4))
        assert model.work.numel() == most and not model.older


def test_steps_run_on_their_device(pkg, monkeypatch):
    """every call of the library is made with the buffers' device as the current one, whichever the caller's is"""
    import torch
    from pyodide_llm_amd import checkpoint, forward, serve
    rng = np.random.default_rng(10)
    ck = checkpoint.Checkpoint(checkpoints.write((256, 768, 1, 4, 2, 300, 64), "int8", rng)[0])
    model = forward.Forward(ck, tokens=4, sequences=2, pages=4, width=2, page=16)
    serving = serve.Serving(model)
    inside, calls = [], []

    class Entered(torch.cuda.device):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *error):
            inside.pop()
            return super().__exit__(*error)

    class Watched:
        def __getattr__(self, name):
            calls.append((name, list(inside)))
            return getattr(pkg.library(), name)

    monkeypatch.setattr(torch.cuda, "device", Entered)
    model.lib = serving.lib = Watched()
    ids, ones = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([1, 2], [1, 1]))
    serving.step(ids, ones, torch.rand(2, device="cuda"), 1)
    serving.finish(torch.ones(2, dtype=torch.bool, device="cuda"))
    x = torch.empty(2, 256, device="cuda")
    model.embed(ids, x)
    model.logits(model.step(x, serving.starts, ones, serving.table, 1), torch.empty(2, 300, device="cuda"))
    names = {name for name, _ in calls}
    assert {"hq_batch_plan_ex", "hq_embed_ex", "hq_attention_ex", "hq_sample_ex", "hq_pages_give_ex"} <= names
    assert all(at and at[-1] == model.y.device.index for _, at in calls)


def test_adapters_of_one_and_two_projections(pkg):
    """a model whose attention needs less workspace than the adapters, of which one or two projections may need more than three"""
    import torch
    from pyodide_llm_amd import adapters, checkpoint, forward
    rng = np.random.default_rng(7)
    ck = checkpoint.Checkpoint(checkpoints.write((512, 768, 1, 8, 8, 100, 64), "int8", rng)[0])
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    x = torch.from_numpy(rng.standard_normal((128, 512)).astype(F)).cuda()
    for names in (("wo", "w2"), ("w1", "w3"), ("wq", "wk", "wv", "w1")):
        model = watched(forward)(ck, tokens=128, sequences=4, pages=8, width=2, page=16)
        model.starts = np.arange(0, 129, 32)
        held = adapters.Adapters(factors(torch, ck, rng, 1, 256, names, torch.float16))
        batch = pkg.cache.Batch(4096, 4096, 4096, 4, 128, 32, 2)
        assert pkg.library().hq_attention_work_bytes(model.caches[0], batch, 8) < pkg.library().hq_adapters_work_bytes(2, 256, 128)
        model.step(x.clone(), ints(*model.starts), ints(32, 32, 32, 32), ints(*range(8)).view(4, 2), 32, None, held, ints(0, 0, 0, 0))
        assert model.seen == 4 * len(names)


def test_refused(pkg):
    import torch
    from pyodide_llm_amd import adapters, checkpoint, forward, serve
    rng = np.random.default_rng(1)
    ck = checkpoint.Checkpoint(checkpoints.write((256, 768, 1, 4, 2, 100, 64), "int8", rng)[0])
    model = forward.Forward(ck, tokens=4, sequences=2, pages=4, width=2, page=16)
    serving = serve.Serving(model)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    u = torch.zeros(2, device="cuda")
    for bad in ((ints(1, 2).long(), ints(1, 1), u), (ints(1, 2), ints(1, 1, 0), u), (ints(1, 2), ints(1, 1), u.double()),
                (ints(1, 2, 3, 4, 5), ints(4, 1), u), (ints(1, 2, 3, 4)[::2], ints(1, 1), u), (ints(), ints(0, 0), u),
                (ints(1, 2).cpu(), ints(1, 1), u)):
        with pytest.raises(ValueError, match="refused"):
            serving.step(*bad)
    for bad in (torch.zeros(3, dtype=torch.bool, device="cuda"), ints(1, 1), torch.zeros(2, dtype=torch.bool)):
        with pytest.raises(ValueError, match="refused"):
            serving.finish(bad)
    with pytest.raises(ValueError, match="refused"):
        model.embed(ints(1, 2), torch.empty(2, 64, device="cuda"))
    with pytest.raises(ValueError, match="refused"):
        model.logits(torch.empty(2, 256, device="cuda"), torch.empty(2, 99, device="cuda"))
    one = factors(torch, ck, rng, 2, 8, ("wq",), torch.float16)
    fit = adapters.Adapters(one)
    other = adapters.Adapters({"wq": (one["wq"][0][..., :128].contiguous(), one["wq"][1])})
    x, starts, lengths = torch.zeros(2, 256, device="cuda"), ints(0, 1, 2), ints(1, 1)
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for at, held, which in ((None, fit, None), (None, None, ints(0, 0)), (None, fit, ints(0)), (None, other, ints(0, 0)),
                            (ints(0), None, None), (None, fit, ints(0, 0).long()),
                            (None, adapters.Adapters({"rope": one["wq"]}), ints(0, 0))):
        with pytest.raises(ValueError, match="refused"):
            model.step(x, starts, lengths, table, 1, at, held, which)
