"""A layer's operators between its products, as cases that can be timed and checked: the norm that takes the residual in
and readies the products' int8 activations, the paged key/value cache as it is written and read back, and the attention
of new tokens over it.

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, where `own` is true, through
libhq.so's entry points.  All inputs are float32, as the products give them; the cache's elements are int8 or float16,
with a float32 scale a (position, head).
"""
import importlib
import math
import random

import torch

own = False
DEV = "cuda:0"
EPS = 1e-5
FORMS = {"int8": 0, "f16": 1}
READY = {"biased": 0, "plain": 1, "planes": 2, "sums": 3}
UNIT = {"biased": 32, "plain": 32, "planes": 128, "sums": 256}
SMALLEST = 2.0 ** -100  # a vector whose scale would be smaller is stored as zeros


def _norm(name, n, tokens, ready):
    return {"name": name, "op": "norm", "n": n, "tokens": tokens, "ready": ready}


def _cache(name, part, form, heads, dim, page, sequences, tokens, context):
    return {"name": name, "op": "cache", "part": part, "form": form, "heads": heads, "dim": dim, "page": page,
            "sequences": sequences, "tokens": tokens, "context": context, "ragged": sequences > 1}


def _attention(name, form, heads, kv, dim, page, sequences, tokens, context, ragged=False, window=0, cap=0.0):
    return {"name": name, "op": "attention", "form": form, "heads": kv, "queries": heads, "dim": dim, "page": page,
            "sequences": sequences, "tokens": tokens, "context": context, "ragged": ragged, "window": window,
            "cap": cap}


def listed():
    return [
        # a story model's token: one row of 288 values, where the launch is everything
        _norm("norm_15m_token", 288, 1, "plain"),
        # an 8B model's long prompt, before every projection of every layer
        _norm("norm_8b_2048_tokens", 4096, 2048, "biased"),
        # a decode step of 32 sequences of an 8B model: a key and a value of every head each, at 32 odd places
        _cache("cache_8b_32_tokens", "write", "int8", 8, 128, 64, 32, 1, 8000),
        # a 1B model's prompts of several lengths arriving together, kept in 16 bits
        _cache("cache_1b_prompts", "write", "f16", 8, 64, 32, 5, 2048, 2048),
        # a conversation's whole cache read back (to be kept, or laid out anew)
        _cache("cache_8b_read", "read", "int8", 8, 128, 64, 1, 8192, 8192),
        # a 350M chat model's turn read back: 777 positions
        _cache("cache_350m_read", "read", "f16", 4, 64, 16, 1, 777, 777),
        # a story model's token, 200 positions in: latency
        _attention("attention_15m_token", "int8", 6, 6, 48, 16, 1, 1, 200),
        # a decode step of 32 conversations of 1200 to 8000 positions
        _attention("attention_8b_32_tokens", "int8", 32, 8, 128, 64, 32, 1, 8000, ragged=True),
        # a token of one very long document, in 16 bits
        _attention("attention_8b_long_token", "f16", 32, 8, 128, 64, 1, 1, 131072),
        # a decode step of 8 sequences with 4 drafted tokens each
        _attention("attention_8b_drafts", "int8", 32, 8, 128, 64, 8, 5, 4100),
        # the last quarter of a prompt of 8192 tokens, 2048 tokens a step: the largest call
        _attention("attention_8b_chunk", "int8", 32, 8, 128, 64, 1, 2048, 8192),
        # a server's mixed step: prompts, turns and single tokens of a 1B model, one sequence without new tokens
        _attention("attention_1b_mixed", "f16", 32, 8, 64, 32, 7, 511, 3000, ragged=True),
    ]


def draw(rng):
    """One more case: any of the operators, forms and head layouts, a token, a few or a prompt"""
    def log(lo, hi):
        return math.exp(rng.uniform(math.log(lo), math.log(hi)))

    op = rng.choice(["norm", "cache", "attention", "attention"])
    if op == "norm":
        ready = rng.choice(["biased", "biased", "plain", "planes", "sums"])
        n = (round(log(288, 8192) / UNIT[ready]) | 1) * UNIT[ready]  # (an odd number of groups)
        case = _norm("", n, 1 if rng.random() < 0.35 else round(log(2, 2048)), ready)
        case["tokens"] = min(case["tokens"], 4096 * 2048 // n)
    else:
        dim, queries, kv = rng.choice([(48, 6, 6), (64, 16, 4), (64, 32, 8), (80, 20, 20), (96, 24, 8), (128, 32, 8),
                                       (128, 40, 8), (256, 24, 4)])
        form, page = rng.choice(["int8", "int8", "f16"]), rng.choice([16, 32, 64, 128, 256])
        sequences = round(log(1, 32))
        if op == "cache":
            part = rng.choice(["write", "read"])
            tokens = 1 if part == "write" and rng.random() < 0.4 else round(log(2, 4096))
            context = tokens if part == "read" else tokens + rng.randint(0, 4000)
            case = _cache("", part, form, kv, dim, page, sequences, tokens, context)
            most, cells = 8192 * 8 * 128, context * sequences * kv * dim
        else:
            tokens = rng.choice([1, 1, rng.randint(2, 16), round(log(17, 2048))])
            context = tokens + round(log(1, 16000))
            window = rng.choice([0, 0, 0, round(log(32, 4096))])
            case = _attention("", form, queries, kv, dim, page, sequences, tokens, context, rng.random() < 0.5, window,
                              rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]))
            most, cells = 32 * 128 * 2048 * 7168, queries * dim * tokens * context * sequences
            # (the plain form holds every score and every key at once)
            most = min(most, cells * 32 * 2048 * 8192 // (queries * tokens * context * sequences) + 1,
                       cells * 131072 * 8 * 128 // (context * sequences * kv * dim) + 1)
        while cells > most and case["sequences"] > 1:
            case["sequences"] -= 1
            cells = cells * case["sequences"] // (case["sequences"] + 1)
        while cells > most:
            case["tokens"], case["context"] = max(1, case["tokens"] // 2), max(1, case["context"] // 2)
            cells //= 2 if op == "cache" or case["tokens"] == 1 else 4
        # odd counts: nothing is a whole number of tiles
        case["tokens"] |= 1
        case["context"] = max(case["context"], case["tokens"]) | 1
        if case["sequences"] == 1:
            case["ragged"] = False
    del case["name"]
    return case


# ---- what a case's batch is ---------------------------------------------------------------------------------------
def _batch(case):
    """(new tokens, length with them) of every sequence: the first the longest, the others of a ragged batch spread
    over the range, some with one new token and some with none"""
    got = []
    for i in range(case["sequences"]):
        part = (i * 0.6180339887) % 1.0 if i else 1.0
        tokens, length = case["tokens"], case["context"]
        if case["ragged"] and i:
            length = max(1, round(length * (0.15 + 0.85 * part)))
            if case["op"] == "cache" and case["part"] == "read":
                tokens = length
            elif tokens > 1:
                tokens = (1, max(1, round(tokens * part)), 0, max(1, round(tokens * 0.5 * part)))[i % 4]
            length = max(length, tokens)
        got.append((tokens, length))
    return got


def _first_seen(case, new, length):
    """the first position that the first of a sequence's new tokens sees"""
    window = case.get("window", 0)
    return max(0, length - new + 1 - window) if window else 0


def _pairs(case):
    """(token, position) pairs that see each other, and positions seen, over all sequences"""
    pairs = positions = 0
    for new, length in _batch(case):
        window = case.get("window", 0) or length
        pairs += sum(min(length - new + i + 1, window) for i in range(new))
        positions += length - _first_seen(case, new, length) if new else 0
    return pairs, positions


def work(case):
    if case["op"] == "norm":
        n, t = case["n"], case["tokens"]
        scales = {"biased": n // 8, "plain": n // 8, "planes": n // 4, "sums": n // 2}[case["ready"]]
        return {"bytes": t * (12 * n + n + scales) + 4 * n, "flops": 10 * t * n}
    vector = case["dim"] * (1 if case["form"] == "int8" else 2) + 4  # a head's stored vector with its scale
    new = sum(t for t, _ in _batch(case))
    if case["op"] == "cache":
        # the float32 vectors and the stored ones, each read or written (a written batch is read back as well)
        once = 2 * new * case["heads"] * (4 * case["dim"] + vector)
        return {"bytes": once * (2 if case["part"] == "write" else 1), "flops": 6 * new * case["heads"] * case["dim"]}
    pairs, positions = _pairs(case)
    return {"bytes": 2 * positions * case["heads"] * vector + 8 * new * case["queries"] * case["dim"],
            "flops": 4 * pairs * case["queries"] * case["dim"]}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _stored(x, form):
    """(elements, scale) of the vectors x (.., dim) as the cache holds them: value = element * scale"""
    most = x.abs().amax(-1, keepdim=True)
    if form == "int8":
        scale = most / torch.full_like(most, 127.0)  # (a division by a number may be a product with its inverse)
    else:
        scale = torch.ldexp(torch.ones_like(most), torch.frexp(most)[1] - 15)
    scale = torch.where(scale < SMALLEST, torch.zeros_like(scale), scale)
    inverse = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    elements = torch.round(x * inverse).to(torch.int8) if form == "int8" else (x * inverse).half()
    return elements, scale[..., 0]


def _inputs(case, seed):
    gen = _generator(seed)
    if case["op"] == "norm":
        n, t = case["n"], case["tokens"]
        # a residual stream: channels of very different sizes, a block's output to add, a norm's weights about 1
        return {"x": _randn(gen, t, n) * torch.exp(_randn(gen, n)), "d": _randn(gen, t, n) * 0.3,
                "w": 1 + 0.3 * _randn(gen, n)}
    heads, dim, page = case["heads"], case["dim"], case["page"]
    batch = _batch(case)
    new = [t for t, _ in batch]
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    counts = [-(-length // page) for _, length in batch]
    width, pages = max(counts) + 1, sum(counts) + 3  # (a table has room to grow, a pool pages to spare)
    order = random.Random(seed).sample(range(pages), sum(counts))
    table = []
    for count, (t, length) in zip(counts, batch):
        row = [order.pop() for _ in range(count)]
        # a windowed layer has given back the pages that no token sees any more
        gone = _first_seen(case, t, length) // page if case.get("window") else 0
        table.append([-1] * gone + row[gone:] + [-1] * (width - count))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    # keys with channels of different sizes
    spread = torch.exp(0.5 * _randn(gen, heads, 1, dim))
    got = {"starts": ints(starts), "lengths": ints([length for _, length in batch]), "table": ints(table),
           "pages": pages, "width": width, "tokens": starts[-1]}
    if case["op"] == "cache" and case["part"] == "write":
        got["new_k"] = _randn(gen, starts[-1], heads, dim) * spread[:, 0]
        got["new_v"] = _randn(gen, starts[-1], heads, dim)
        elements = torch.int8 if case["form"] == "int8" else torch.float16
        got["k"] = torch.zeros(pages, heads, page, dim, dtype=elements, device=DEV)
        got["v"] = torch.zeros(pages, heads, dim, page, dtype=elements, device=DEV)
        got["ks"], got["vs"] = (torch.zeros(pages, heads, page, device=DEV) for _ in range(2))
        return got
    got["k"], got["ks"] = _stored(_randn(gen, pages, heads, page, dim) * spread, case["form"])
    v, got["vs"] = _stored(_randn(gen, pages, heads, page, dim), case["form"])
    got["v"] = v.transpose(-1, -2).contiguous()
    if case["op"] == "attention":
        got["q"] = _randn(gen, starts[-1], case["queries"], dim) * 2
    return got


def _frame(case):
    """the bytes of a token's readied activations, and of its scales (and sums) after the n int8 values"""
    n = case["n"]
    scales = {"biased": n // 8, "plain": n // 8, "planes": n // 4, "sums": n // 2}[case["ready"]]
    return (n + scales + 15) // 16 * 16, scales


def prepare(case, seed):
    state = {"case": dict(case), **_inputs(case, seed)}
    if case["op"] == "norm":
        n, t = case["n"], case["tokens"]
        frame, scales = _frame(case)
        acts = torch.zeros(t, frame, dtype=torch.uint8, device=DEV)
        state["acts"], state["r"] = acts, torch.empty(t, n, device=DEV)
        state["q8"] = acts[:, :n].view(torch.int8)
        state["scales"] = acts[:, n:n + n // 8].view(torch.float32)
        state["values"] = torch.empty(t, n, dtype=torch.float16, device=DEV)
        after = acts[:, n + n // 8:n + scales]
        state["sums"] = after.view(torch.int32 if case["ready"] == "planes" else torch.int16)
    elif case["op"] == "cache":
        shape = (state["tokens"], case["heads"], case["dim"])
        state["out_k"], state["out_v"] = (torch.empty(shape, device=DEV) for _ in range(2))
    else:
        state["out"] = torch.empty_like(state["q"])
    if case["op"] != "norm":
        # where each new token is, for the plain forms: its sequence, its place there and its position
        new = [t for t, _ in _batch(case)]
        at = torch.tensor([(s, i) for s, t in enumerate(new) for i in range(t)], device=DEV).view(-1, 2)
        state["seq"], state["place"] = at[:, 0], at[:, 1]
        batch = torch.tensor(_batch(case), device=DEV)
        state["position"] = (batch[:, 1] - batch[:, 0])[at[:, 0]] + at[:, 1]
        state["longest"] = max(new)
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _plain_norm(s):
    case = s["case"]
    n, t, ready = case["n"], case["tokens"], case["ready"]
    r = s["x"] + s["d"]
    y = r * (1 / torch.sqrt(torch.mean(r * r, -1, keepdim=True) + EPS)) * s["w"]
    groups = y.view(t, n // 32, 32)
    scale = groups.abs().amax(-1, keepdim=True) / (63.0 if ready == "biased" else 127.0)
    q = torch.round(groups * (1 / scale))
    out = {"r": r, "values": (q * scale).view(t, n).half(), "scales": scale[..., 0]}
    if ready == "planes":
        out["sums"] = (-q.sum(-1) * scale[..., 0]).half()
    if ready == "sums":
        out["sums"] = torch.cat([q.view(t, -1, 16).sum(-1), q.view(t, -1, 8).sum(-1)], -1).half()
    return out


def _plain_write(s):
    case, page = s["case"], s["case"]["page"]
    pages, slot = s["table"][s["seq"], s["position"] // page].long(), s["position"] % page
    k, s["ks"][pages, :, slot] = _stored(s["new_k"], case["form"])
    v, s["vs"][pages, :, slot] = _stored(s["new_v"], case["form"])
    s["k"][pages, :, slot] = k
    s["v"][pages, :, :, slot] = v


def _plain_read(s):
    page = s["case"]["page"]
    pages, slot = s["table"][s["seq"], s["position"] // page].long(), s["position"] % page
    return {"k": s["k"][pages, :, slot].float() * s["ks"][pages, :, slot, None],
            "v": s["v"][pages, :, :, slot].float() * s["vs"][pages, :, slot, None]}


def _plain_attention(s):
    case = s["case"]
    kv, dim, group = case["heads"], case["dim"], case["queries"] // case["heads"]
    sequences, most, reach = s["lengths"].numel(), s["longest"], s["width"] * case["page"]
    pages = s["table"].clamp(min=0).long()
    k = s["k"][pages].float() * s["ks"][pages][..., None]
    k = k.permute(0, 2, 4, 1, 3).reshape(sequences, kv, dim, reach)
    v = s["v"][pages].float() * s["vs"][pages][..., None, :]
    v = v.permute(0, 2, 1, 4, 3).reshape(sequences, kv, reach, dim)
    q = torch.zeros(sequences, most, kv, group, dim, device=DEV)
    q[s["seq"], s["place"]] = s["q"].view(-1, kv, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(sequences, kv, most * group, dim)
    scores = torch.matmul(q, k).mul_(1 / math.sqrt(dim)).view(sequences, kv, most, group, reach)
    if case["cap"]:
        scores = torch.tanh(scores / case["cap"]) * case["cap"]
    ends = torch.zeros(sequences, most, dtype=torch.long, device=DEV)
    ends[s["seq"], s["place"]] = s["position"] + 1
    j = torch.arange(reach, device=DEV)
    seen = (j < ends[..., None]) & (s["table"] >= 0).repeat_interleave(case["page"], 1)[:, None]
    if case["window"]:
        seen &= j >= ends[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp(min=-3e38)
    weights = scores.exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(sequences, kv, most * group, reach), v).view(sequences, kv, most, group, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.permute(0, 2, 1, 3, 4)[s["seq"], s["place"]].reshape(-1, kv * group, dim)


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _handles(s):
    """what a program keeps beside its tensors: the library, its descriptions of the cache and the batch, a workspace"""
    if "hq" not in s:
        case, hq = s["case"], importlib.import_module("pyodide-llm_amd")
        s["hq"] = hq
        s["lib"] = hq.library()
        if case["op"] != "norm":
            s["cache"] = hq.cache.Cache(s["k"].data_ptr(), s["v"].data_ptr(), s["ks"].data_ptr(), s["vs"].data_ptr(),
                                        FORMS[case["form"]], s["pages"], case["page"], case["heads"], case["dim"])
            s["batch"] = hq.cache.Batch(s["starts"].data_ptr(), s["lengths"].data_ptr(), s["table"].data_ptr(),
                                        s["lengths"].numel(), s["tokens"], s["longest"], s["width"])
        if case["op"] == "attention":
            s["bytes"] = s["lib"].hq_attention_work_bytes(s["cache"], s["batch"], case["queries"])
            s["work"] = torch.empty(s["bytes"], dtype=torch.uint8, device=DEV)
    return s["lib"], torch.cuda.current_stream().cuda_stream


def _ok(s, status):
    if status:
        s["hq"].check(status)


def _own_norm(s):
    lib, stream = _handles(s)
    case, acts = s["case"], s["acts"]
    n, t, ready = case["n"], case["tokens"], case["ready"]
    at, stride = acts.data_ptr(), 4 * n
    _ok(s, lib.hq_norm_ready_ex(at, at + n, None, s["r"].data_ptr(), s["x"].data_ptr(), s["d"].data_ptr(),
                                s["w"].data_ptr(), n, EPS, READY[ready], t, acts.stride(0), stride, stride, stride,
                                stream))
    q, scales, values = s["q8"], s["scales"], s["values"]
    out = {"r": s["r"], "values": values, "scales": scales}
    # the int8 values as the numbers they stand for
    if ready == "planes":  # byte 16 p + c of 64 is value 4 c + p
        torch.mul(q.view(t, n // 64, 4, 2, 8).permute(0, 1, 3, 4, 2), scales.view(t, n // 64, 2, 1, 1),
                  out=values.view(t, n // 64, 2, 8, 4))
        out["sums"] = (s["sums"] * scales).half()
    else:
        torch.mul((q - 64 if ready == "biased" else q).view(t, n // 32, 32), scales[..., None],
                  out=values.view(t, n // 32, 32))
        if ready == "sums":
            out["sums"] = s["sums"].half()
    return out


def _own_write(s):
    lib, stream = _handles(s)
    stride = s["new_k"].stride(0) * 4
    _ok(s, lib.hq_cache_write_ex(s["cache"], s["batch"], s["new_k"].data_ptr(), s["new_v"].data_ptr(), stride, stride,
                                 stream))


def _own_read(s):
    lib, stream = _handles(s)
    stride = s["out_k"].stride(0) * 4
    _ok(s, lib.hq_cache_read_ex(s["cache"], s["batch"], s["out_k"].data_ptr(), s["out_v"].data_ptr(), stride, stride,
                                stream))
    return {"k": s["out_k"], "v": s["out_v"]}


def _own_attention(s):
    lib, stream = _handles(s)
    case, stride = s["case"], s["q"].stride(0) * 4
    _ok(s, lib.hq_attention_ex(s["out"].data_ptr(), s["q"].data_ptr(), case["queries"], stride, stride, s["cache"],
                               s["batch"], 1 / math.sqrt(case["dim"]), case["window"], case["cap"],
                               s["work"].data_ptr(), s["bytes"], stream))
    return s["out"]


def run(state):
    """A norm gives the new residual, the int8 activations as the numbers they stand for (in 16 bits: where a value lies
    half-way between two steps, a last bit of the norm decides), their scales and sums; a cache's case the vectors of
    the batch's tokens read back (after they were written, where it writes); attention its output."""
    case = state["case"]
    if case["op"] == "norm":
        return (_own_norm if own else _plain_norm)(state)
    if case["op"] == "attention":
        return (_own_attention if own else _plain_attention)(state)
    if case["part"] == "write":
        (_own_write if own else _plain_write)(state)
    return (_own_read if own else _plain_read)(state)


# ---- the results in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    heads, dim, page = case["heads"], case["dim"], case["page"]
    batch, table = _batch(case), s["table"].tolist()
    if case["op"] == "cache" and case["part"] == "write":
        # the steps (a vector's scale, an int8's inverse) are the format's own float32 numbers
        got = {}
        for name in ("k", "v"):
            x = s["new_" + name]
            most = x.abs().amax(-1, keepdim=True)
            if case["form"] == "int8":
                scale = most / torch.tensor(127.0, device=DEV).expand_as(most)
                steps = torch.round(x * scale.reciprocal()).double()
            else:
                scale = torch.exp2(torch.floor(torch.log2(most.double())) - 14)
                steps = (x.double() / scale).half().double()
            got[name] = steps * scale.double()
        return got
    out = []
    for (new, length), row in zip(batch, table):
        pages = torch.tensor([max(p, 0) for p in row[:-(-length // page)]], device=DEV)
        k = (s["k"][pages].double() * s["ks"][pages].double().unsqueeze(-1)).transpose(0, 1).reshape(heads, -1, dim)
        v = (s["v"][pages].double() * s["vs"][pages].double().unsqueeze(-2)).permute(1, 0, 3, 2).reshape(heads, -1, dim)
        k, v = k[:, :length], v[:, :length]
        if case["op"] == "cache":
            out.append((k.transpose(0, 1), v.transpose(0, 1)))
            continue
        begin = sum(t for t, _ in batch[:len(out)])
        q = s["q"][begin:begin + new].double()
        last = torch.arange(length - new, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)[None]
        hidden = j > last
        if case["window"]:
            hidden = hidden | (j <= last - case["window"])
        group, rows = case["queries"] // heads, torch.empty(new, case["queries"], dim, dtype=torch.float64, device=DEV)
        for h in range(case["queries"] if new else 0):
            a = q[:, h] @ k[h // group].t().contiguous() / math.sqrt(dim)
            if case["cap"]:
                a = case["cap"] * torch.tanh(a / case["cap"])
            rows[:, h] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v[h // group]
        out.append(rows)
    if case["op"] == "cache":
        return {"k": torch.cat([k for k, _ in out]), "v": torch.cat([v for _, v in out])}
    return torch.cat(out)


def _exact_norm(case, s):
    n, t, most = case["n"], case["tokens"], 63 if case["ready"] == "biased" else 127
    r = s["x"].double() + s["d"].double()
    y = s["w"].double() * r * torch.rsqrt((r ** 2).sum(-1, keepdim=True) / n + EPS)
    y = y.view(t, n // 32, 32)
    scale = y.abs().amax(-1, keepdim=True) / most
    q = torch.round(y / scale)
    out = {"r": r, "values": (q * scale).view(t, n), "scales": scale.squeeze(-1)}
    if case["ready"] == "planes":
        out["sums"] = -q.sum(-1) * scale.squeeze(-1)
    if case["ready"] == "sums":
        out["sums"] = torch.cat([q.view(t, n // 16, 16).sum(-1), q.view(t, n // 8, 8).sum(-1)], -1)
    return out
