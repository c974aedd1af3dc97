"""The operators of a serving step over a paged key-value cache: how they are called, what they compute, and
cases of real sizes to time them on.

    plan       lengths and free pages of the requests -> block tables, slot map, positions (whole numbers)
    qkv        QK-norm, rotary embedding, and the append of keys and values to their pages
    attention  one new token of every request over its pages
    sample     ids from logits by temperature, top-k, top-p and min-p, from given uniform numbers

`run` computes them in elementary torch operations, or, with `own` set, through the package's entry points
(include/plamo_kernels.h). A case is a dict of plain values; `prepare` makes its inputs from a seed.
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TYPE_CODES = {"bf16": 0, "f16": 1, "f32": 2}
EPS = 1e-6
WORKSPACE_BYTES = 16 << 20
ROPE_THETA = 1e6

_package = None


def package():
    """This repository's package (its folder's name is no Python name, so it is loaded by its path)."""
    global _package
    if _package is None:
        name, home = "plamo_b200", Path(__file__).resolve().parents[1] / "plamo3-0.8b-runtime_b200"
        if name not in sys.modules:
            spec = importlib.util.spec_from_file_location(name, home / "__init__.py", submodule_search_locations=[str(home)])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _package = sys.modules[name].runtime
    return _package


def listed():
    return [
        # One request being answered, a few hundred tokens in: a call whose latency is what counts.
        dict(name="attention 1 x 700", op="attention", rows=1, heads=16, kv_heads=1, head_dim=128, page=16, shortest=700,
             longest=700, window=0, dtype="bf16"),
        # A batch of mixed ages under grouped-query heads, one slot of it without tokens yet.
        dict(name="attention 32 x 0-2048 gqa", op="attention", rows=32, heads=16, kv_heads=4, head_dim=128, page=16,
             shortest=0, longest=2048, window=0, dtype="bf16"),
        # A sliding-window layer: every request sees its last 2048 tokens of up to 8000.
        dict(name="attention 48 window 2048", op="attention", rows=48, heads=16, kv_heads=1, head_dim=128, page=16,
             shortest=100, longest=8000, window=2048, dtype="bf16"),
        # Few long documents: rows alone cannot fill the GPU.
        dict(name="attention 3 x 9001-32767 f16", op="attention", rows=3, heads=16, kv_heads=1, head_dim=128, page=32,
             shortest=9001, longest=32767, window=0, dtype="f16"),
        # The largest batch at the longest context.
        dict(name="attention 64 x 32768", op="attention", rows=64, heads=16, kv_heads=1, head_dim=128, page=64,
             shortest=32768, longest=32768, window=0, dtype="bf16"),
        # The decode step of 32 requests.
        dict(name="qkv 32 decode", op="qkv", tokens=32, heads=16, kv_heads=1, head_dim=128, page=16, context=32768,
             consecutive=False, skipped=0, dtype="bf16"),
        # Prompts of many requests in one call, with a few tokens whose request got no page.
        dict(name="qkv 8191 prefill gqa", op="qkv", tokens=8191, heads=16, kv_heads=4, head_dim=128, page=16, context=32768,
             consecutive=True, skipped=5, dtype="bf16"),
        # Bookkeeping of one decode step of 32 requests.
        dict(name="plan 32 decode", op="plan", rows=32, page=16, width=2048, longest=32000, most=1, ended=2, short=False),
        # A large server's step: prompt chunks of a thousand requests, some ended, and too few pages for all.
        dict(name="plan 1000 prefill", op="plan", rows=1000, page=16, width=2048, longest=32000, most=512, ended=40, short=True),
        # One request's next token under the usual controls.
        dict(name="sample 1", op="sample", rows=1, vocab=107520, filters="all", dtype="bf16"),
        # A batch in which every request brings its own controls, greedy ones among them.
        dict(name="sample 32 mixed", op="sample", rows=32, vocab=107520, filters="mixed", dtype="bf16"),
        # The largest batch, at an odd vocabulary, in 32 bits, by temperature alone.
        dict(name="sample 64 f32", op="sample", rows=64, vocab=80001, filters="none", dtype="f32"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "qkv", "plan", "sample", "sample"])
    if op == "attention":
        kv = rng.choice([1, 1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 7, 8, 16] if kv > 1 else [4, 8, 12, 16, 16, 20, 32])
        rows, dim = _spread(rng, 1, 128), rng.choice([64, 128, 128])
        # at most 64 x 32768 keys of one 128-wide head
        longest = min(_spread(rng, 1, 32768), (64 * 32768 * 128) // (rows * kv * dim))
        shortest = rng.choice([longest, rng.randint(0, longest), rng.randint(0, min(longest, 64))])
        window = rng.choice([0, 0, _spread(rng, 1, 4096)])
        return dict(op=op, rows=rows, heads=heads, kv_heads=kv, head_dim=dim, page=rng.choice([1, 8, 16, 16, 24, 32, 64, 128]),
                    shortest=shortest, longest=longest, window=window, dtype=rng.choice(["bf16", "bf16", "f16"]))
    if op == "qkv":
        tokens, kv = _spread(rng, 1, 8000), rng.choice([1, 2, 4])
        return dict(op=op, tokens=tokens, heads=kv * rng.choice([1, 3, 4] if kv > 1 else [8, 12, 16]), kv_heads=kv,
                    head_dim=rng.choice([64, 128, 128]), page=rng.choice([1, 8, 16, 24, 64]), context=_spread(rng, 8192, 65536),
                    consecutive=rng.random() < 0.5, skipped=rng.randint(0, min(7, tokens - 1)), dtype=rng.choice(["bf16", "bf16", "f16"]))
    if op == "plan":
        rows, page = _spread(rng, 1, 1000), rng.choice([1, 8, 16, 24, 64])
        longest = _spread(rng, 16, 32000)
        most = rng.choice([1, _spread(rng, 2, 512)])
        return dict(op=op, rows=rows, page=page, width=min(2048, -(-(longest + most) // page) + rng.randint(0, 3)), longest=longest,
                    most=most, ended=rng.randint(0, rows // 4), short=rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    return dict(op=op, rows=_spread(rng, 1, 64), vocab=_spread(rng, 1000, 80001 if dtype == "f32" else 107520),
                filters=rng.choice(["none", "top-k", "top-p", "min-p", "all", "mixed"]), dtype=dtype)


def _lengths(rows, shortest, longest):
    """Lengths of `rows` requests from the longest to the shortest, most of them short, as ages in a batch are."""
    if rows == 1 or shortest == longest:
        return [longest] * rows
    low = max(1, shortest)
    got = [round(longest * (low / longest) ** (i / (rows - 1))) for i in range(rows)]
    got[-1] = shortest
    return got


def _requests(case):
    """The plan's requests as (length, append) pairs, and its numbers of held, freed, needed and free pages."""
    rows, page, most = case["rows"], case["page"], case["most"]
    lens = [min(n, case["width"] * page - most) for n in _lengths(rows, 0, case["longest"])]
    adds = [1] * rows if most == 1 else [most - (i * 37) % (most + 1) for i in range(rows)]
    for i in range(min(case["ended"], rows)):
        adds[(i * rows) // case["ended"]] = -1
    held = [-(-n // page) for n in lens]
    need = [max(0, -(-(n + a) // page) - h) if a > 0 else 0 for n, a, h in zip(lens, adds, held)]
    freed = sum(h for h, a in zip(held, adds) if a < 0)
    wanted = max(0, sum(need) - freed)
    free = (9 * wanted) // 10 if case["short"] else wanted + 8
    return list(zip(lens, adds)), held, freed, sum(need), free


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _ints(values, perm=None):
    t = torch.tensor(values, dtype=torch.int32, device=DEVICE)
    return t if perm is None else t[perm].contiguous()


def _fill_table(held, width, pages):
    """A block table [rows, width] whose row r holds the next held[r] of `pages`, the rest -1."""
    table = torch.full((held.numel(), width), -1, dtype=torch.int32, device=DEVICE)
    mask = torch.arange(width, device=DEVICE) < held[:, None]
    return table.masked_scatter_(mask, pages)


def _rope_table(rows, head_dim):
    """cos and sin of every position and frequency, as bf16 bits in one word: cos | sin << 16."""
    freq = ROPE_THETA ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=DEVICE) / head_dim)
    angle = torch.arange(rows, dtype=torch.float64, device=DEVICE)[:, None] * freq
    bits = [t.to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xFFFF for t in (angle.cos(), angle.sin())]
    return bits[0] | (bits[1] << 16)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case["op"]
    s = dict(case)
    if op == "attention":
        rows, page, kv, dim, dt = case["rows"], case["page"], case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]
        perm = torch.randperm(rows, generator=gen, device=DEVICE)
        lens = _lengths(rows, case["shortest"], case["longest"])
        held = [-(-n // page) for n in lens]
        s["width"] = max(1, max(held))
        s["pages"] = sum(held) + 3
        s["lens"] = _ints(lens, perm)
        s["table"] = _fill_table(_ints(held, perm), s["width"],
                                 torch.randperm(s["pages"], generator=gen, device=DEVICE).to(torch.int32))
        s["keys"] = _normal(gen, s["pages"], page, kv, dim).to(dt)
        s["values"] = _normal(gen, s["pages"], page, kv, dim).to(dt)
        s["q"] = (2.0 * _normal(gen, rows, case["heads"], dim)).to(dt)
        s["scale"] = dim ** -0.5
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(rows, case["heads"], device=DEVICE)
        s["workspace"] = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device=DEVICE)
    elif op == "qkv":
        n, page, kv, dim, dt = case["tokens"], case["page"], case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]
        s["pages"] = 2 * -(-n // page) + 1
        total = s["pages"] * page
        s["qkv"] = _normal(gen, n, (case["heads"] + 2 * kv) * dim).to(dt)
        s["q_norm"], s["k_norm"] = ((0.1 * _normal(gen, dim)).to(dt) for _ in range(2))
        s["rope"] = _rope_table(case["context"], dim)
        if case["consecutive"]:  # whole prompts: runs of slots in pages of any order
            start = int(torch.randint(0, max(1, case["context"] - n), (1,), generator=gen, device=DEVICE))
            s["positions"] = start % case["context"] + torch.arange(n, dtype=torch.int32, device=DEVICE)
            s["positions"] %= case["context"]
            at = torch.arange(n, device=DEVICE)
            order = torch.randperm(s["pages"], generator=gen, device=DEVICE)
            slots = order[at // page] * page + at % page
        else:
            s["positions"] = torch.randint(0, case["context"], (n,), generator=gen, device=DEVICE, dtype=torch.int32)
            slots = torch.randperm(total, generator=gen, device=DEVICE)[:n]
        if case["skipped"]:
            slots[torch.randperm(n, generator=gen, device=DEVICE)[:case["skipped"]]] = -1
        s["slots"] = slots.to(torch.int32)
        # one slot more than the cache has, where the plain form puts what has no slot
        s["keys"], s["values"] = (_normal(gen, total + 1, kv, dim).to(dt) for _ in range(2))
        s["q"] = torch.empty(n, case["heads"], dim, dtype=dt, device=DEVICE)
    elif op == "plan":
        rows, page, width = case["rows"], case["page"], case["width"]
        pairs, held, freed, need, free = _requests(case)
        perm = torch.randperm(rows, generator=gen, device=DEVICE)
        s["lens"], s["append"] = _ints([n for n, _ in pairs], perm), _ints([a for _, a in pairs], perm)
        s["pages"] = sum(held) + free + 8
        s["capacity"] = max(1, sum(max(0, a) for _, a in pairs)) + 5
        order = torch.randperm(s["pages"], generator=gen, device=DEVICE).to(torch.int32)
        s["table"] = _fill_table(_ints(held, perm), width, order)
        # the free list's end past `pages` takes what the plain form does not push
        s["free_list"] = torch.full((s["pages"] + 1,), -1, dtype=torch.int32, device=DEVICE)
        s["free_list"][:free] = order[sum(held):sum(held) + free]
        s["free_count"] = _ints([free])
        s["new_lens"], s["row_start"] = _ints([0] * rows), _ints([0] * (rows + 1))
        s["slots"], s["positions"] = (torch.empty(s["capacity"], dtype=torch.int32, device=DEVICE) for _ in range(2))
        s["counts"] = _ints([0] * 4)
    else:
        rows, vocab = case["rows"], case["vocab"]
        # a background of unlikely words and a head of likely ones, as a language model's logits have
        logits = 2.5 * _normal(gen, rows, vocab)
        head = min(300, vocab)
        at = torch.rand(rows, vocab, generator=gen, device=DEVICE).topk(head, dim=1).indices
        likely = 18.0 - 1.6 * torch.arange(1, head + 1, device=DEVICE).log() + _normal(gen, rows, head)
        s["logits"] = logits.scatter_(1, at, likely).to(TYPES[case["dtype"]])
        kind = [(["none", "top-k", "top-p", "min-p", "all", "greedy"][i % 6] if case["filters"] == "mixed" else case["filters"])
                for i in range(rows)]
        perm = torch.randperm(rows, generator=gen, device=DEVICE)
        floats = lambda v: torch.tensor(v, dtype=torch.float32, device=DEVICE)[perm].contiguous()  # noqa: E731
        s["temperature"] = floats([0.0 if k == "greedy" else 0.7 + 0.05 * (i % 9) for i, k in enumerate(kind)])
        s["top_k"] = _ints([(20 + 15 * (i % 7) if k in ("top-k", "all") else 0) for i, k in enumerate(kind)], perm)
        s["top_p"] = floats([(0.8 + 0.03 * (i % 6) if k in ("top-p", "all") else 1.0) for i, k in enumerate(kind)])
        s["min_p"] = floats([(0.02 + 0.01 * (i % 4) if k in ("min-p", "all") else 0.0) for i, k in enumerate(kind)])
        s["u"] = torch.rand(rows, generator=gen, device=DEVICE)
        s["ids"], s["kept"] = _ints([0] * rows), _ints([0] * rows)
        s["logprobs"] = torch.empty(rows, device=DEVICE)
    return s


def run(state):
    return {"attention": _attention, "qkv": _qkv, "plan": _plan, "sample": _sample}[state["op"]](state)


def _cache(s):
    """The cache's descriptor, which a program makes once beside the cache."""
    if "cache" not in s:
        kv, dim, page = s["kv_heads"], s["head_dim"], s["page"]
        s["cache"] = package().PagedCache(s["keys"].data_ptr(), s["values"].data_ptr(), TYPE_CODES[s["dtype"]], s["pages"], page,
                                          kv, dim, page * kv * dim, kv * dim, dim)
    return s["cache"]


def _attention(s):
    rows, heads, dim = s["q"].shape
    if own:
        package().k_paged_attention(_cache(s), s["q"].data_ptr(), heads * dim, rows, heads, s["table"].data_ptr(), s["width"],
                                    s["lens"].data_ptr(), rows, 0, s["longest"], s["window"], s["scale"], s["out"].data_ptr(),
                                    heads * dim, s["lse"].data_ptr(), s["workspace"].data_ptr(), WORKSPACE_BYTES)
        return {"out": s["out"], "lse": s["lse"]}
    page, kv = s["page"], s["kv_heads"]
    at = torch.arange(s["width"] * page, device=DEVICE)
    held = s["table"].long()[:, at // page]
    lens = s["lens"][:, None]
    seen = (at < lens) & (held >= 0)
    if s["window"]:
        seen &= at >= lens - s["window"]
    slot = held.clamp(min=0) * page + at % page
    seen = seen[:, None, None, :]
    k = s["keys"].view(-1, kv, dim)[slot].float()
    scores = torch.matmul(s["q"].float().view(rows, kv, heads // kv, dim), k.permute(0, 2, 3, 1)) * s["scale"]
    del k
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    v = s["values"].view(-1, kv, dim)[slot].float().permute(0, 2, 1, 3)
    out = torch.matmul(p, torch.where(seen.transpose(2, 3), v, 0.0)) / torch.where(total > 0, total, 1.0)
    return {"out": out.view(rows, heads, dim).to(s["q"].dtype), "lse": (top + torch.log(total)).view(rows, heads)}


def _qkv(s):
    n, kv, dim, heads, dt = s["tokens"], s["kv_heads"], s["head_dim"], s["heads"], TYPES[s["dtype"]]
    if own:
        package().k_paged_qkv(_cache(s), s["qkv"].data_ptr(), (heads + 2 * kv) * dim, n, heads, s["q_norm"].data_ptr(),
                              s["k_norm"].data_ptr(), EPS, s["rope"].data_ptr(), s["context"], s["positions"].data_ptr(),
                              s["slots"].data_ptr(), s["q"].data_ptr(), heads * dim)
        return {"q": s["q"], "keys": s["keys"][:-1], "values": s["values"][:-1]}
    x = s["qkv"].float().view(n, heads + 2 * kv, dim)
    weight = torch.cat([s["q_norm"].float().expand(heads, dim), s["k_norm"].float().expand(kv, dim)]) + 1.0
    qk = x[:, :heads + kv]
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * weight
    angle = s["rope"][s["positions"].long()][:, None, :]
    cos, sin = (angle << 16).view(torch.float32), (angle & -65536).view(torch.float32)
    a, b = qk[..., :dim // 2], qk[..., dim // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    live = s["slots"] >= 0
    slots = torch.where(live, s["slots"].long(), s["keys"].shape[0] - 1)
    s["keys"][slots] = qk[:, heads:].to(dt)
    s["values"][slots] = s["qkv"].view(n, heads + 2 * kv, dim)[:, heads + kv:]
    q = torch.where(live[:, None, None], qk[:, :heads], 0.0).to(dt)
    return {"q": q, "keys": s["keys"][:-1], "values": s["values"][:-1]}


def _plan(s):
    rows, page, width, capacity, pages = s["rows"], s["page"], s["width"], s["capacity"], s["pages"]
    if own:
        package().k_paged_plan(s["lens"].data_ptr(), s["append"].data_ptr(), rows, page, pages, s["table"].data_ptr(), width,
                               s["free_list"].data_ptr(), s["free_count"].data_ptr(), s["new_lens"].data_ptr(),
                               s["row_start"].data_ptr(), s["slots"].data_ptr(), s["positions"].data_ptr(), capacity,
                               s["counts"].data_ptr())
        return {k: s[k] for k in ("table", "new_lens", "row_start", "slots", "positions", "counts")} | {"free_list": s["free_list"][:pages]}
    lens, add = s["lens"].long(), s["append"].long().clamp(min=0)
    ended = s["append"] < 0
    end = add.cumsum(0)
    start, want = end - add, lens + add
    held = (lens + page - 1) // page
    freed = torch.where(ended, held, 0)
    fits = (want <= width * page) & (end <= capacity)
    need = torch.where(fits & ~ended, (want + page - 1) // page - held, 0)
    free = s["free_count"].long() + freed.sum()
    upto = need.cumsum(0)
    ok = ~ended & fits & ((need == 0) | (upto <= free))
    granted = torch.where(ok, need, 0)
    # the pages of ended requests go onto the free list's end, row by row
    column = torch.arange(width, device=DEVICE)
    push = column < freed[:, None]
    to = torch.where(push, s["free_count"] + (freed.cumsum(0) - freed)[:, None] + column, pages)
    s["free_list"][to.view(-1)] = s["table"].view(-1)
    # and the new pages come off it, the last one first
    nth = column - held[:, None]
    pop = (nth >= 0) & (nth < granted[:, None])
    page_of = s["free_list"][torch.where(pop, free - 1 - (upto - need)[:, None] - nth, 0)]
    s["table"].copy_(torch.where(pop, page_of, s["table"]))
    token = torch.arange(capacity, device=DEVICE)
    row = torch.searchsorted(end, token, right=True).clamp(max=rows - 1)
    live = (token < end[-1]) & ok[row]
    position = torch.where(live, lens[row] + token - start[row], 0)
    slot = s["table"][row, position // page].long() * page + position % page
    whole = lambda t: t.to(torch.int32)  # noqa: E731
    counts = torch.stack([free[0] - granted.sum(), end[-1], granted.sum(), (~ended & ~ok).sum()])
    return {"table": s["table"], "new_lens": whole(torch.where(ended, 0, torch.where(ok, want, lens))),
            "row_start": whole(torch.cat([start, end[-1:]])), "slots": whole(torch.where(live, slot, -1)),
            "positions": whole(torch.where(live, position, -1)), "counts": whole(counts), "free_list": s["free_list"][:pages]}


def _share(fraction, total, up):
    """fraction * total / 2**24 in whole numbers, rounded down or up (fraction <= 2**24, total < 2**62)."""
    return fraction * (total >> 24) + ((fraction * (total & 0xFFFFFF) + (0xFFFFFF if up else 0)) >> 24)


def _sample(s):
    rows, vocab = s["logits"].shape
    if own:
        package().k_sample(s["logits"].data_ptr(), TYPE_CODES[s["dtype"]], rows, vocab, vocab, s["temperature"].data_ptr(),
                           s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["u"].data_ptr(),
                           s["ids"].data_ptr(), s["logprobs"].data_ptr(), s["kept"].data_ptr())
        return {"ids": s["ids"], "logprobs": s["logprobs"], "kept": s["kept"]}
    x = s["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(1, keepdim=True)
    t = s["temperature"][:, None]
    warm = t > 0
    e = torch.exp((x - top) / torch.where(warm, t, 1.0))
    e = torch.where(x == top, 1.0, e)
    e = torch.where(x == -math.inf, 0.0, e)
    # weights in fixed point, 2**40 for the most likely token: their sums are exact in any order
    w = (e * 2.0 ** 40).to(torch.int64)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    sorted_w = w.gather(1, order)
    rank = torch.arange(vocab, device=DEVICE)
    k = s["top_k"][:, None]
    k = torch.where((k <= 0) | (k > vocab), vocab, k)
    k = torch.where(warm, k, 1)
    sorted_w = torch.where(rank < k, sorted_w, 0)
    upto = sorted_w.cumsum(1)
    p = (s["top_p"].double() * 2.0 ** 24).round().clamp(0, 2 ** 24).long()[:, None]
    need = _share(p, upto[:, -1:], up=True).clamp(min=1)
    least = (s["min_p"].double().clamp(0, 1) * 2.0 ** 40).ceil().long()[:, None]
    keep = (sorted_w > 0) & (upto - sorted_w < need) & (sorted_w >= least)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, sorted_w, 0))
    total = kept.sum(1, keepdim=True)
    m = (s["u"] * 2.0 ** 24).floor().clamp(0, 2 ** 24 - 1).long()[:, None]
    ids = (kept.cumsum(1) <= _share(m, total, up=False)).sum(1, keepdim=True)
    ids = torch.where(total > 0, ids, 0)
    logprobs = torch.log(kept.gather(1, ids).double() / total.double().clamp(min=1)).float()
    return {"ids": ids.view(-1).to(torch.int32), "logprobs": logprobs.view(-1), "kept": keep.sum(1).to(torch.int32)}


def work(case):
    op = case["op"]
    if op == "attention":
        rows, heads, kv, dim = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
        window = case["window"] or case["longest"]
        keys = sum(min(n, window) for n in _lengths(rows, case["shortest"], case["longest"]))
        pages = sum(-(-min(n, window) // case["page"]) for n in _lengths(rows, case["shortest"], case["longest"]))
        return {"bytes": 4 * keys * kv * dim + 4 * pages + 4 * rows + 4 * rows * heads * dim + 4 * rows * heads,
                "flops": 4 * keys * heads * dim}
    if op == "qkv":
        n, live, heads, kv, dim = case["tokens"], case["tokens"] - case["skipped"], case["heads"], case["kv_heads"], case["head_dim"]
        return {"bytes": 4 * n * heads * dim + 8 * live * kv * dim + 2 * live * dim + 8 * n, "flops": 8 * n * (heads + kv) * dim}
    if op == "plan":
        pairs, _, freed, need, _ = _requests(case)
        tokens = sum(max(0, a) for _, a in pairs)
        return {"bytes": 16 * case["rows"] + 8 * (tokens + freed + need), "flops": 4 * (case["rows"] + tokens)}
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": case["rows"] * (size * case["vocab"] + 32), "flops": 4 * case["rows"] * case["vocab"]}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None
    if op == "attention":
        kv, page, dim = s["kv_heads"], s["page"], s["head_dim"]
        group = s["heads"] // kv
        out = torch.zeros(s["rows"], s["heads"], dim, dtype=torch.float64, device=DEVICE)
        lse = torch.full((s["rows"], s["heads"]), -math.inf, dtype=torch.float64, device=DEVICE)
        for r, n in enumerate(s["lens"].tolist()):
            first = max(0, n - s["window"]) if s["window"] else 0
            at = torch.arange(first, n, device=DEVICE)
            if not n:
                continue
            page_of = s["table"][r].long()[at // page]
            k, v = s["keys"][page_of, at % page].double(), s["values"][page_of, at % page].double()
            q = s["q"][r].double().view(kv, group, dim)
            a = torch.einsum("hgd,thd->hgt", q, k) * s["scale"]
            out[r] = torch.einsum("hgt,thd->hgd", torch.softmax(a, -1), v).reshape(-1, dim)
            lse[r] = torch.logsumexp(a, -1).view(-1)
        return {"out": out, "lse": lse}
    if op == "qkv":
        n, kv, dim, heads = s["tokens"], s["kv_heads"], s["head_dim"], s["heads"]
        x = s["qkv"].double().view(n, -1, dim)
        bits = s["rope"][s["positions"].long()].cpu().numpy().view("uint32")
        turn = [torch.from_numpy(b.astype("uint32").view("float32").astype("float64")).to(DEVICE)
                for b in (bits << 16, bits & 0xFFFF0000)]
        phase = torch.complex(*turn)[:, None, :]

        def turned(h, weight):
            h = h / (h.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * (1.0 + weight.double())
            z = torch.complex(h[..., :dim // 2], h[..., dim // 2:]) * phase
            return torch.cat([z.real, z.imag], -1)

        live = s["slots"] >= 0
        keys, values = s["keys"][:-1].double(), s["values"][:-1].double()
        at = s["slots"][live].long()
        keys[at] = turned(x[:, heads:heads + kv], s["k_norm"])[live]
        values[at] = x[:, heads + kv:][live]
        return {"q": turned(x[:, :heads], s["q_norm"]) * live[:, None, None], "keys": keys, "values": values}
    logprobs = torch.zeros(s["rows"], dtype=torch.float64, device=DEVICE)
    for r in range(s["rows"]):
        t = float(s["temperature"][r])
        if t <= 0:
            continue
        x = s["logits"][r].double()
        p = torch.softmax(x / t, 0)
        ranked, order = torch.sort(x, descending=True, stable=True)
        p_ranked = p[order]
        k = int(s["top_k"][r]) or s["vocab"]
        p_ranked[k:] = 0
        before = p_ranked.cumsum(0) - p_ranked
        keep = (p_ranked > 0) & (before < float(s["top_p"][r]) * p_ranked.sum()) & (p_ranked >= float(s["min_p"][r]) * p.max())
        kept = torch.zeros_like(p)
        kept[order[keep]] = p_ranked[keep]
        run_sum = kept.cumsum(0)
        chosen = int(torch.searchsorted(run_sum, s["u"][r].double() * run_sum[-1], right=True).clamp(max=s["vocab"] - 1))
        logprobs[r] = (kept[chosen] / kept.sum()).log()
    return {"ids": None, "logprobs": logprobs, "kept": None}
