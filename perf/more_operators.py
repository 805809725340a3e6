"""What a serving step does around its layers, as cases that can be timed and checked: the embeddings of token ids from a
packed table, a batch's starts, lengths, page table and token maps from the requests' lengths, the low-rank adapters of many
requests beside a shared projection, and the next tokens drawn from logits with given random numbers.

`run` computes a case in its plain form (elementary torch operations) or, where `own` is true, through libhq.so's entry
points.  Activations and logits are float32, as the products take and give them; adapters are float16 or bfloat16.
"""
import importlib
import math

import torch

own = False
DEV = "cuda:0"
PACK = {"int8": 0, "int6": 1, "ternary": 2, "binary": 3, "Q4_K": 256 + 12}
GROUP = {"int8": 32, "int6": 32, "ternary": 128, "binary": 128, "Q4_K": 256}
ROW = {"int8": 1.125, "int6": 0.875, "ternary": 0.265625, "binary": 0.140625, "Q4_K": 0.5625}  # bytes a weight
FORM = {"f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}


def _embed(name, packing, vocab, dim, tokens, scale=1.0):
    return {"name": name, "op": "embed", "packing": packing, "vocab": vocab, "dim": dim, "tokens": tokens, "scale": scale}


def _plan(name, sequences, page, tokens, context, spare=1.0):
    return {"name": name, "op": "plan", "sequences": sequences, "page": page, "tokens": tokens, "context": context,
            "spare": spare}


def _sample(name, rows, vocab, kind, masked=0.0):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "kind": kind, "masked": masked}


def _adapters(name, form, n, rows, rank, adapters, sequences, tokens):
    return {"name": name, "op": "adapters", "form": form, "n": n, "rows0": rows[0], "rows1": rows[1] if len(rows) > 1 else 0,
            "rows2": rows[2] if len(rows) > 2 else 0, "rank": rank, "adapters": adapters, "sequences": sequences,
            "tokens": tokens}


def listed():
    return [
        # a story model's token looked up: a row of 288 int8 values, where the launch is everything
        _embed("embed_15m_token", "int8", 32000, 288, 1),
        # a ternary 1B model's prompts, their rows scaled by the root of the width
        _embed("embed_1b_ternary", "ternary", 128256, 2048, 511, 45.25483399593904),
        # an 8B model's long prompt
        _embed("embed_8b_2048_tokens", "int8", 128256, 4096, 2048),
        # a decode step of 32 conversations: a token each, here and there a new page
        _plan("plan_32_tokens", 32, 64, 1, 8000),
        # a server's large step: 1024 requests, prompts and turns of up to 512 tokens arriving together
        _plan("plan_1024_requests", 1024, 16, 512, 3000),
        # a story model's next token as llama2.c draws it: temperature 1, top-p 0.9
        _sample("sample_15m_token", 1, 32000, "top_p"),
        # 8 constrained answers of a 350M chat model: a grammar has masked most of the vocabulary
        _sample("sample_350m_constrained", 8, 65536, "mixed", 0.9),
        # a decode step of 32 conversations, each with its own settings
        _sample("sample_8b_32_tokens", 32, 128256, "mixed"),
        # a decode step of 256 requests, each with its own settings: the largest
        _sample("sample_8b_256_tokens", 256, 128256, "mixed"),
        # a decode step of 32 conversations over 24 adapters of rank 16, beside an 8B model's q, k and v
        _adapters("adapters_8b_32_tokens", "bf16", 4096, (4096, 1024, 1024), 16, 24, 32, 1),
        # five ragged prompts beside a 1B model's gate and up product, rank 32
        _adapters("adapters_1b_prompts", "f16", 2048, (8192, 8192), 32, 4, 5, 411),
        # a long prompt of one adapter of rank 64 beside an 8B model's output product
        _adapters("adapters_8b_2048_tokens", "bf16", 4096, (4096,), 64, 3, 1, 2048),
    ]


def draw(rng):
    """One more case: any of the operators, packings and settings, a token, a few or many"""
    def log(lo, hi):
        return math.exp(rng.uniform(math.log(lo), math.log(hi)))

    op = rng.choice(["embed", "plan", "sample", "sample", "adapters", "adapters"])
    if op == "embed":
        packing = rng.choice(["int8", "int8", "int6", "ternary", "binary", "Q4_K"])
        unit = GROUP[packing]
        dim = max(1, round(log(256, 6144) / unit)) * unit
        case = _embed("", packing, rng.choice([32000, 50257, 65536, 128256]), dim,
                      1 if rng.random() < 0.3 else min(round(log(2, 4096)) | 1, 2048 * 4096 // dim), rng.choice([1.0, dim ** 0.5]))
    elif op == "plan":
        tokens = rng.choice([1, rng.randint(2, 16), round(log(17, 1024)) | 1])
        sequences = min(round(log(1, 1500)), 1024 * 512 // tokens + 1)
        case = _plan("", sequences, rng.choice([16, 32, 64, 128, 256]), tokens, tokens + round(log(1, 8000)),
                     rng.choice([1.0, 1.0, 0.6]))
    elif op == "sample":
        vocab = rng.choice([32000, 50257, 65536, 128256, rng.randint(300, 20000) | 1])
        rows = min(round(log(1, 256)), 256 * 128256 // vocab)
        case = _sample("", rows, vocab, rng.choice(["mixed", "mixed", "top_p", "top_k", "min_p", "all", "greedy"]),
                       rng.choice([0.0, 0.0, 0.0, 0.5, 0.99]))
    else:
        n = rng.choice([288, 1024, 2048, 4096, round(log(256, 8192) / 32) * 32])
        rows = rng.choice([(n,), (n, 96), (n, max(1, n // 4), max(1, n // 4)), (round(log(96, 8192)),), (rng.choice([768, 4608, 8192]),) * 2])
        sequences = round(log(1, 48))
        tokens = rng.choice([1, 1, rng.randint(2, 16), round(log(17, 2048)) | 1])
        rank = rng.choice([8, 16, 16, 32, 64, 128])
        most = 2048 * 4096 * 2 * 64  # the largest listed case's products
        while sequences * tokens * (n + sum(rows)) * rank > most:
            sequences, tokens = max(1, sequences // 2), tokens if sequences > 1 else max(1, tokens // 2)
        case = _adapters("", rng.choice(["f16", "bf16"]), n, rows, rank, rng.randint(1, 32), sequences, tokens)
        while case["adapters"] * rank * (n + sum(rows)) > 3 * 64 * 3 * 8192:
            case["adapters"] = case["adapters"] // 2 if case["adapters"] > 1 else 1
            if case["adapters"] == 1:
                break
    del case["name"]
    return case


# ---- what a case's batch is ---------------------------------------------------------------------------------------
def _part(i):
    return (i * 0.6180339887) % 1.0 if i else 1.0


def _fresh(case):
    """the new tokens of every sequence: the first the most, others of a prompt's batch spread over the range, some with
    one and some with none"""
    tokens = case["tokens"]
    if tokens == 1:
        return [1] * case["sequences"]
    return [max(1, round(tokens * _part(i))) if i % 5 != 3 else i // 5 % 2 for i in range(case["sequences"])]


def _held(case):
    """the positions that a sequence has already: some fill their last page, some requests are new"""
    page, got = case["page"], []
    for i in range(case["sequences"]):
        held = max(0, round(case["context"] * _part(i + 7)) - 1) if i % 6 != 5 else 0
        got.append(held // page * page if i % 8 == 2 else held)
    return got


def _wanted(case):
    """the pages that the new tokens need"""
    page = case["page"]
    return sum(-(-(h + f) // page) - -(-h // page) for h, f in zip(_held(case), _fresh(case)))


def _targets(case):
    return [r for r in (case["rows0"], case["rows1"], case["rows2"]) if r]


def _which(case):
    """the adapter of every sequence: every seventh has none"""
    return [-1 if i % 7 == 6 else i * 5 % case["adapters"] for i in range(case["sequences"])]


def work(case):
    if case["op"] == "embed":
        return {"bytes": round(case["tokens"] * (case["dim"] * (ROW[case["packing"]] + 4) + 4)),
                "flops": 2 * case["tokens"] * case["dim"]}
    if case["op"] == "plan":
        # fresh, held, starts and lengths a sequence; a page read and written; sequence, position and slot a token
        return {"bytes": 16 * case["sequences"] + 8 * _wanted(case) + 16 * sum(_fresh(case)), "flops": 0}
    if case["op"] == "sample":
        # (an exponential in 64 bits a value, where a row's sum has to be known)
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": 20 * case["rows"] * case["vocab"]}
    rows, n, rank = sum(_targets(case)), case["n"], case["rank"]
    fresh, which = _fresh(case), _which(case)
    used = len({w for w, f in zip(which, fresh) if w >= 0 and f})
    busy = sum(f for w, f in zip(which, fresh) if w >= 0)
    return {"bytes": 2 * used * rank * (n * len(_targets(case)) + rows) + 4 * busy * n + 8 * sum(fresh) * rows,
            "flops": 2 * busy * rank * (n * len(_targets(case)) + rows)}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def _ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind, device=DEV)


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _bytes(gen, *shape):
    return torch.randint(0, 256, shape, dtype=torch.uint8, device=DEV, generator=gen)


def _table(case, gen):
    """(values, scales) of a packed table as a checkpoint's file has them"""
    packing, vocab, dim = case["packing"], case["vocab"], case["dim"]
    if packing == "Q4_K":
        blocks = _bytes(gen, vocab, dim // 256, 144)
        ends = (torch.rand(vocab, dim // 256, 2, device=DEV, generator=gen) * 4e-3 + 1e-4).half()
        blocks[..., :4] = ends.view(torch.uint8)
        return blocks, torch.zeros(34992, dtype=torch.uint8, device=DEV)  # (a K type's block needs no grid)
    scale = torch.rand(vocab, dim // GROUP[packing], device=DEV, generator=gen) * 1e-3 + 1e-4
    if packing in ("ternary", "binary"):
        return _bytes(gen, vocab, dim // (4 if packing == "ternary" else 8)), scale.half()
    return _bytes(gen, vocab, dim if packing == "int8" else dim * 3 // 4), scale


def _logits(case, gen):
    """rows of very different sharpness over a vocabulary whose first words are the frequent ones: a few words stand out
    of each row, by little or by much; a grammar's mask hides the rest of the words where one is at work"""
    rows, vocab = case["rows"], case["vocab"]
    x = 2.0 * _randn(gen, rows, vocab) - 0.6 * torch.log1p(torch.arange(vocab, device=DEV) / 50.0)
    words = (vocab * torch.rand(rows, 24, device=DEV, generator=gen) ** 3).long().clamp_(max=vocab - 1)
    lift = 5.0 + 8.0 * torch.rand(rows, 1, device=DEV, generator=gen)
    x.scatter_add_(1, words, lift * torch.rand(rows, 24, device=DEV, generator=gen))
    if case["masked"]:
        x[torch.rand(rows, vocab, device=DEV, generator=gen) < case["masked"]] = -math.inf
        x[:, vocab // 3] = 1.0  # (one word at least is free)
    return x


def _settings(case, gen):
    """(temperature, top_k, top_p, min_p) of every row, as requests send them"""
    rows, kind = case["rows"], case["kind"]
    i = torch.arange(rows, device=DEV)
    pick = lambda *v: _ints(v, torch.float32)[i % len(v)]  # noqa: E731
    off = torch.zeros(rows, device=DEV)
    if kind == "mixed":
        return (pick(0.7, 1.0, 0.0, 0.8, 1.2, 0.6), pick(40, 0, 0, 50, 20, 0, 1000).int(), pick(0.95, 0.9, 1.0, 0.8),
                pick(0.0, 0.05, 0.0, 0.0, 0.1))
    temperature = {"greedy": off, "all": pick(1.0, 0.8)}.get(kind, pick(1.0, 0.8, 0.6))
    top_k = pick(40, 1, 64, 200).int() if kind == "top_k" else off.int()
    top_p = pick(0.9, 0.95, 0.5) if kind == "top_p" else off + 1
    return temperature, top_k, top_p, pick(0.05, 0.1, 0.02) if kind == "min_p" else off


def _inputs(case, seed):
    gen = _generator(seed)
    op = case["op"]
    if op == "embed":
        values, scales = _table(case, gen)
        ids = torch.randint(0, case["vocab"], (case["tokens"],), dtype=torch.int32, device=DEV, generator=gen)
        return {"values": values, "scales": scales, "ids": ids}
    if op == "sample":
        temperature, top_k, top_p, min_p = _settings(case, gen)
        return {"logits": _logits(case, gen), "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
                "u": torch.rand(case["rows"], device=DEV, generator=gen)}
    if op == "plan":
        page, held, fresh = case["page"], _held(case), _fresh(case)
        wanted, had = _wanted(case), sum(-(-h // page) for h in held)
        pages, spare = had + wanted + 5, max(1, round(wanted * case["spare"])) + (3 if case["spare"] >= 1 else 0)
        width = max(-(-(h + f) // page) for h, f in zip(held, fresh)) + 2
        order = torch.randperm(pages, device=DEV, generator=gen).int()
        # a row's pages, and -1 behind them
        kept, e = -(-_ints(held) // page), torch.arange(width, device=DEV)[None]
        at = (torch.cumsum(kept, 0) - kept)[:, None] + e
        return {"held": _ints(held), "fresh": _ints(fresh), "free": order[had:].contiguous(),
                "count": _ints([min(spare, pages - had)]), "pages": pages, "width": width, "tokens": sum(fresh),
                "before": torch.where(e < kept[:, None], order[at.clamp(max=pages - 1)], -1).int()}
    n, rank, adapters, kind = case["n"], case["rank"], case["adapters"], FORM[case["form"]][1]
    fresh = _fresh(case)
    total = sum(fresh)
    got = {"fresh": fresh, "tokens": total, "which": _ints(_which(case)),
           "starts": _ints([sum(fresh[:i]) for i in range(len(fresh) + 1)]),
           "x": _randn(gen, total, n) * torch.exp(0.5 * _randn(gen, n)),
           "scales": 0.5 + torch.rand(adapters, device=DEV, generator=gen)}
    got["a"] = [(_randn(gen, adapters, rank, n) / n ** 0.5).to(kind) for _ in _targets(case)]
    got["b"] = [(_randn(gen, adapters, rows, rank) * 0.1).to(kind) for rows in _targets(case)]
    got["base"] = [_randn(gen, total, rows) for rows in _targets(case)]
    return got


def prepare(case, seed):
    state = {"case": dict(case), **_inputs(case, seed)}
    op = case["op"]
    if op == "embed":
        state["out"] = torch.empty(case["tokens"], case["dim"], device=DEV)
    elif op == "sample":
        state["token"] = torch.empty(case["rows"], dtype=torch.int32, device=DEV)
        state["chance"] = torch.empty(case["rows"], device=DEV)
    elif op == "plan":
        sequences, tokens = case["sequences"], state["tokens"]
        state["starts"], state["lengths"] = _ints([0] * (sequences + 1)), _ints([0] * sequences)
        state["left"], state["missing"] = _ints([0]), _ints([0])
        state["table"] = state["before"].clone()
        state["sequence"], state["position"] = (torch.empty(tokens, dtype=torch.int32, device=DEV) for _ in range(2))
        state["slot"] = torch.empty(tokens, dtype=torch.int64, device=DEV)
    else:
        state["y"] = [torch.empty_like(t) for t in state["base"]]
        # where each row is, for the plain form: its sequence and its place there
        at = torch.tensor([(s, i) for s, t in enumerate(state["fresh"]) for i in range(t)], device=DEV).view(-1, 2)
        state["seq"], state["place"], state["longest"] = at[:, 0], at[:, 1], max(state["fresh"])
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _plain_embed(s):
    case = s["case"]
    packing, dim, ids = case["packing"], case["dim"], s["ids"].long()
    rows, t = s["values"][ids], ids.numel()
    if packing == "Q4_K":
        ends = rows[..., :4].contiguous().view(torch.float16).float()
        sc = rows[..., 4:16].int()
        low, mid, high = sc[..., :4], sc[..., 4:8], sc[..., 8:]
        scale = torch.cat([low & 63, (high & 15) | (low >> 6 << 4)], -1)
        least = torch.cat([mid & 63, (high >> 4) | (mid >> 6 << 4)], -1)
        q = rows[..., 16:].view(t, -1, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], 3).view(t, -1, 8, 32)
        value = (ends[..., :1] * scale)[..., None] * q - (ends[..., 1:] * least)[..., None]
        return value.view(t, dim) * case["scale"]
    if packing == "int8":
        value = rows.view(torch.int8).float()
    elif packing == "int6":
        group = rows.view(t, -1, 24)
        low = torch.cat([group[..., :16] & 15, group[..., :16] >> 4], -1)
        high = torch.cat([(group[..., 16:] >> shift) & 3 for shift in (0, 2, 4, 6)], -1)
        value = ((low | (high << 4)) << 2).view(torch.int8).float()
    elif packing == "ternary":
        value = torch.stack([(rows >> shift) & 3 for shift in (0, 2, 4, 6)], -1).float() - 1
    else:
        group = rows.view(t, -1, 1, 16, 1) >> torch.arange(8, device=DEV, dtype=torch.uint8).view(2, 1, 4)
        value = (group & 1).float() * 2 - 1
    value = value.reshape(t, -1, GROUP[packing]) * s["scales"][ids].float()[..., None]
    return value.view(t, dim) * case["scale"]


def _plain_plan(s):
    page, held, fresh = s["case"]["page"], s["held"].long(), s["fresh"].long()
    lengths = held + fresh
    starts = torch.cat([torch.zeros_like(held[:1]), torch.cumsum(fresh, 0)])
    first, last = (held + page - 1) // page, (lengths + page - 1) // page
    wanted = last - first
    e = torch.arange(s["width"], device=DEV)
    k = (torch.cumsum(wanted, 0) - wanted)[:, None] + e - first[:, None]
    page_of = torch.where(k < s["count"], s["free"][(s["count"] - 1 - k).clamp(0, s["free"].numel() - 1)], -1)
    table = torch.where((e >= first[:, None]) & (e < last[:, None]), page_of, s["before"])
    rows = torch.arange(s["tokens"], device=DEV)
    sequence = torch.searchsorted(starts[1:], rows, right=True)
    position = held[sequence] + rows - starts[sequence]
    there = table[sequence, position // page].long()
    slot = torch.where(there >= 0, there * page + position % page, -1)
    left = s["count"] - wanted.sum()
    return {"starts": starts.int(), "lengths": lengths.int(), "table": table, "left": left.clamp(min=0).int(),
            "missing": (-left).clamp(min=0).int(), "sequence": sequence.int(), "position": position.int(), "slot": slot}


def _plain_sample(s):
    logits = s["logits"]
    vocab = logits.shape[1]
    greedy = s["temperature"] <= 0
    x = logits.double()
    x = (x - x.amax(-1, keepdim=True)) / torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    w = torch.exp(x)
    k = torch.where(greedy, 1, torch.where(s["top_k"] <= 0, vocab, s["top_k"]))[:, None]
    order = torch.sort(logits, dim=-1, descending=True, stable=True)[1]
    rank = torch.arange(vocab, device=DEV)
    sorted_w = torch.where(rank < k, w.gather(1, order), 0.0)
    cumulative = torch.cumsum(sorted_w, -1)
    p = torch.where(s["top_p"] < 1, s["top_p"].double(), math.inf)[:, None]
    kept = (rank < k) & ((cumulative - sorted_w < p * cumulative[:, -1:]) | (rank == 0)) & (sorted_w >= s["min_p"].double()[:, None])
    w = w * torch.zeros_like(kept).scatter_(1, order, kept)
    cumulative = torch.cumsum(w, -1)
    total = cumulative[:, -1:]
    token = torch.searchsorted(cumulative, s["u"].double()[:, None] * total, right=True).clamp_(max=vocab - 1)
    return {"token": token[:, 0].int(), "chance": (w.gather(1, token) / total)[:, 0].float()}


def _plain_adapters(s):
    which, sequences, longest = s["which"].long(), s["which"].numel(), s["longest"]
    x = torch.zeros(sequences, longest, s["case"]["n"], device=DEV)
    x[s["seq"], s["place"]] = s["x"]
    scale = torch.where(which >= 0, s["scales"][which.clamp(min=0)], 0.0)[s["seq"], None]

    def target(a, b, base):
        a, b = (m[which.clamp(min=0)].float().transpose(1, 2).contiguous() for m in (a, b))
        return base + scale * torch.matmul(torch.matmul(x, a), b)[s["seq"], s["place"]]

    return [target(*t) for t in zip(s["a"], s["b"], s["base"])]


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _at(*tensors):
    return [t.data_ptr() for t in tensors]


def _call(s):
    """what a program keeps beside its tensors: the library's function and its arguments but for the stream"""
    case, op = s["case"], s["case"]["op"]
    hq = importlib.import_module("pyodide-llm_amd")
    s["check"] = hq.check
    lib = hq.library()
    if op == "embed":
        return lib.hq_embed_ex, (*_at(s["out"], s["ids"], s["values"], s["scales"]), PACK[case["packing"]], case["vocab"], case["dim"],
                                 case["scale"], case["tokens"], 4 * case["dim"])
    if op == "sample":
        need = lib.hq_sample_work_bytes(case["rows"], case["vocab"])
        s["work"] = torch.empty(need, dtype=torch.uint8, device=DEV)
        names = ("token", "chance", "logits", "u", "temperature", "top_k", "top_p", "min_p")
        return lib.hq_sample_ex, (*_at(*(s[name] for name in names)), case["rows"], case["vocab"], 4 * case["vocab"],
                                  s["work"].data_ptr(), need)
    if op == "plan":
        batch = hq.cache.Batch(*_at(s["starts"], s["lengths"], s["table"]), case["sequences"], s["tokens"], 0, s["width"])
        pool = hq.cache.Pool(*_at(s["free"], s["count"], s["left"], s["missing"]), s["pages"], case["page"])
        return lib.hq_batch_plan_ex, (batch, pool, *_at(s["held"], s["fresh"], s["sequence"], s["position"], s["slot"]))
    batch = hq.cache.Batch(s["starts"].data_ptr(), None, None, case["sequences"], s["tokens"], s["longest"], 0)
    targets = [hq.adapters.Target(*_at(a, b, base, y), y.shape[1], 4 * y.shape[1], 4 * y.shape[1])
               for a, b, base, y in zip(s["a"], s["b"], s["base"], s["y"])]
    need = lib.hq_adapters_work_bytes(len(targets), case["rank"], s["tokens"])
    s["work"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    return lib.hq_adapters_ex, ((hq.adapters.Target * len(targets))(*targets), len(targets), s["x"].data_ptr(), 4 * case["n"],
                                case["n"], case["rank"], case["adapters"], FORM[case["form"]][0], *_at(s["scales"], s["which"]),
                                batch, s["work"].data_ptr(), need)


def _own(s):
    if "call" not in s:
        s["call"] = _call(s)
    function, arguments = s["call"]
    status = function(*arguments, torch.cuda.current_stream().cuda_stream)
    if status:
        s["check"](status)
    op = s["case"]["op"]
    if op == "embed":
        return s["out"]
    if op == "sample":
        return {"token": s["token"], "chance": s["chance"]}
    if op == "plan":
        return {name: s[name] for name in ("starts", "lengths", "table", "left", "missing", "sequence", "position", "slot")}
    return s["y"]


def run(state):
    """Embeddings; a plan's whole batch (starts, lengths, table, what is left of the pool, the token maps); the drawn tokens
    with their chances; every projection with its adapters' part"""
    if own:
        return _own(state)
    return {"embed": _plain_embed, "plan": _plain_plan, "sample": _plain_sample, "adapters": _plain_adapters}[state["case"]["op"]](state)


# ---- the results in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = _inputs(case, seed)
    if case["op"] == "embed":
        return _exact_embed(case, s)
    if case["op"] == "sample":
        chances = [_exact_row(s, r) for r in range(case["rows"])]
        return {"token": None, "chance": torch.tensor(chances, dtype=torch.float64, device=DEV)}
    out = []
    for a, b, base in zip(s["a"], s["b"], s["base"]):
        y, at = base.double(), 0
        for fresh, which in zip(s["fresh"], _which(case)):
            if fresh and which >= 0:
                low = s["x"][at:at + fresh].double() @ a[which].double().t()
                y[at:at + fresh] += low @ b[which].double().t() * s["scales"][which].double()
            at += fresh
        out.append(y)
    return out


def _exact_embed(case, s):
    packing, dim, ids = case["packing"], case["dim"], s["ids"].long()
    raw, j = s["values"][ids].long(), torch.arange(dim, device=DEV)  # (weight j of a row)
    if packing == "int8":
        value = torch.where(raw > 127, raw - 256, raw).double()
    elif packing == "int6":
        k = j % 32
        low = raw[:, j // 32 * 24 + k % 16] >> (k // 16 * 4) & 15
        top = raw[:, j // 32 * 24 + 16 + k % 8] >> (k // 8 * 2) & 3
        value = (4 * torch.where(top >= 2, low + 16 * top - 64, low + 16 * top)).double()
    elif packing == "ternary":
        value = (raw[:, j // 4] // 4 ** (j % 4) % 4 - 1).double()
    elif packing == "binary":
        k = j % 128
        value = 2.0 * (raw[:, j // 128 * 16 + k // 4 % 16] // 2 ** (k // 64 * 4 + k % 4) % 2).double() - 1
    else:
        block, k = j // 256, j % 256
        raw = raw.view(ids.numel(), -1, 144)
        ends = s["values"][ids][..., :4].contiguous().view(torch.float16).double()
        part = k // 32
        sixes = 4 + part % 4
        scale = torch.where(part < 4, raw[:, block, sixes] % 64, raw[:, block, sixes + 8] % 16 + raw[:, block, sixes] // 64 * 16)
        least = torch.where(part < 4, raw[:, block, sixes + 4] % 64,
                            raw[:, block, sixes + 8] // 16 + raw[:, block, sixes + 4] // 64 * 16)
        q = raw[:, block, 16 + k // 64 * 32 + k % 32] // 16 ** (part % 2) % 16
        return (ends[:, block, 0] * scale * q - ends[:, block, 1] * least) * case["scale"]
    return value * s["scales"][ids].double()[:, j // GROUP[packing]] * case["scale"]


def _exact_row(s, r):
    """the chance of the token that a row's number draws"""
    x = s["logits"][r].double()
    temperature, top_k, top_p, min_p, u = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    if temperature <= 0:
        return 1.0
    value, index = torch.sort(x, descending=True, stable=True)
    if top_k > 0:
        value, index = value[:int(top_k)], index[:int(top_k)]
    weight = torch.exp((value - value[0]) / temperature)
    if top_p < 1:
        reached = torch.nonzero(torch.cumsum(weight, 0) >= top_p * weight.sum())
        most = int(reached[0]) + 1 if len(reached) else len(weight)
        weight, index = weight[:most], index[:most]
    weight = torch.where(weight >= min_p, weight, 0.0)
    back = torch.argsort(index)
    above = torch.nonzero(torch.cumsum(weight[back], 0) > u * weight.sum())
    return float(weight[back][int(above[0])] / weight.sum())
