"""The operators of a decoder's step beside its cache and attention, as cases to
measure: the plan of a ragged batch (page allocation, positions and slots from
request lengths), the norm and rotation of queries and keys, attention with a
window and sinks over the paged e4m3 cache, and the sampling of the next token.

`run` computes a case in plain torch operations (fp32 inside, 64 bits for angles
and probabilities) where `own` is false, and through luisaml_b200's entry points
where it is true.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
LEAST = 2.0 ** -1000  # weights below this share of the largest count as 0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    gqa = {"q_heads": 32, "kv_heads": 8, "dim": 128}
    rope = {"op": "rope", "rotary": 128, "interleaved": False, "far": 32768, "base": 10000.0, "norm": True, "w32": False}
    return [
        # a decode step's plan: 64 sequences bring one token each
        {"name": "plan_64x1", "op": "plan", "batch": 64, "tokens": 1, "held": 4000, "page": 64, "ended": 0.0, "chunks": 0.0},
        # continuous batching: most sequences bring a token, some a chunk of their prompt, some rows go to new requests
        {"name": "plan_256_mixed", "op": "plan", "batch": 256, "tokens": 700, "held": 2000, "page": 16, "ended": 0.1, "chunks": 0.1},
        # whole prompts of odd lengths
        {"name": "plan_9x7001", "op": "plan", "batch": 9, "tokens": 7001, "held": 0, "page": 32, "ended": 0.0, "chunks": 1.0},
        # a single chat's next token, heads of a packed projection
        dict(gqa, **rope, name="rope_1", tokens=1, dtype="bf16"),
        # prompts
        dict(gqa, **rope, name="rope_8191", tokens=8191, dtype="bf16"),
        # neighbouring pairs, a quarter of the head rotated, far positions, fp32
        dict(rope, name="rope_3001_partial", q_heads=20, kv_heads=4, dim=96, rotary=24, interleaved=True, far=1000000, tokens=3001, dtype="f32"),
        # a decode step of 64 long chats: only the window and the sinks are still in the cache
        dict(gqa, name="attend_64x1", op="attend", batch=64, tokens=1, context=30000, page=64, block=64, dtype="bf16", window=1024, sinks=4),
        # chunks of prompts behind a cached prefix
        dict(name="attend_4x1000", op="attend", batch=4, tokens=1000, context=8000, q_heads=16, kv_heads=2, dim=64, page=48, block=16, dtype="f16", window=1500, sinks=37),
        # two whole prompts in a layer with a short window
        dict(gqa, name="attend_2x4096", op="attend", batch=2, tokens=4096, context=0, page=64, block=64, dtype="bf16", window=512, sinks=16),
        # a single chat's next token: top-k and top-p together
        {"name": "sample_1x32000", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "f32", "spread": 2.5, "top_k": 50, "top_p": 0.9, "min_p": 0.0, "greedy": 0.0, "masked": 0.0},
        # a serving batch, top-p alone, odd vocabulary, some rows greedy, some restricted to few tokens
        {"name": "sample_128x128001", "op": "sample", "rows": 128, "vocab": 128001, "dtype": "f32", "spread": 2.5, "top_k": 0, "top_p": 0.92, "min_p": 0.0, "greedy": 0.1, "masked": 0.1},
        # no cut but min-p, 16-bit logits with many ties
        {"name": "sample_60x49999", "op": "sample", "rows": 60, "vocab": 49999, "dtype": "bf16", "spread": 2.0, "top_k": 0, "top_p": 1.0, "min_p": 0.01, "greedy": 0.0, "masked": 0.2},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one(rng):
    op = rng.choice(["plan", "rope", "attend", "sample", "sample"])
    if op == "plan":
        chunks = rng.choice([0.0, 0.1, 1.0])
        return {"op": op, "batch": _log(rng, 1, 512 if chunks < 1 else 32), "tokens": _log(rng, 2, 7001) if chunks else 1, "held": _log(rng, 1, 6000),
                "page": rng.choice([16, 32, 48, 64, 128]), "ended": rng.choice([0.0, 0.2]), "chunks": chunks}
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        kv = rng.choice([1, 2, 4, 5, 8])
        return {"op": op, "tokens": _log(rng, 1, 8191), "kv_heads": kv, "q_heads": kv * rng.choice([1, 2, 4, 5, 7]), "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2]), "interleaved": rng.random() < 0.4, "far": rng.choice([4096, 131072, 1000000]),
                "base": rng.choice([10000.0, 500000.0]), "norm": rng.random() < 0.8, "w32": rng.random() < 0.5, "dtype": rng.choice(["f32", "f16", "bf16"])}
    if op == "attend":
        c = {"op": op, "kv_heads": rng.choice([1, 2, 4, 5, 8]), "dim": rng.choice([64, 128]), "block": rng.choice([16, 32, 64]), "dtype": rng.choice(["f16", "bf16"]),
             "window": _log(rng, 17, 2000), "sinks": _log(rng, 1, 200)}
        c["q_heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
        c["page"] = c["block"] * rng.choice([1, 2, 3, 4])
        how = rng.choice(["decode", "verify", "prompt", "chunk"])
        if how == "decode":
            c.update(batch=_log(rng, 1, 64), tokens=1, context=_log(rng, 1, 30000))
        elif how == "verify":
            c.update(batch=_log(rng, 1, 32), tokens=rng.randint(2, 8), context=_log(rng, 1, 8000))
        elif how == "prompt":
            c.update(batch=rng.randint(1, 3), tokens=_log(rng, 16, 4096), context=0)
        else:
            c.update(batch=rng.randint(1, 6), tokens=_log(rng, 16, 1000), context=_log(rng, 16, 8000))
        return c
    return {"op": op, "rows": _log(rng, 1, 128), "vocab": _log(rng, 999, 200000), "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "spread": rng.uniform(1.0, 4.0),
            "top_k": rng.choice([0, 0, _log(rng, 1, 2000)]), "top_p": rng.choice([1.0, rng.uniform(0.3, 0.99), rng.uniform(0.8, 0.99)]),
            "min_p": rng.choice([0.0, 0.0, rng.uniform(0.005, 0.2)]), "greedy": rng.choice([0.0, 0.2]), "masked": rng.choice([0.0, 0.0, 0.3])}


def draw(rng):
    most = {}
    for c in listed():
        for k, v in work(c).items():
            most[c["op"], k] = max(most.get((c["op"], k), 0), v)
    while True:
        c = _one(rng)
        if all(v <= most[c["op"], k] for k, v in work(c).items()):
            return c


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k not in ("name", "dtype"))))


def _lengths(case):
    """New tokens and earlier tokens of each sequence: the first has the most of both, the others spread below."""
    rng = _rng(case)
    b, n, c = case["batch"], case["tokens"], case["context"]
    new = [n] + [n if n <= 8 else rng.randint((n + 1) // 2, n) for _ in range(b - 1)]
    return new, [c] + [rng.randint(c // 8, c) for _ in range(b - 1)]


def _requests(case):
    """(new tokens, held, ended) of each row of a plan: a row whose request ended takes a new one about as long."""
    rng = _rng(case)
    got = []
    for i in range(case["batch"]):
        held = rng.randint(case["held"] // 4, case["held"])
        ended = rng.random() < case["ended"]
        new = held if ended else rng.randint((case["tokens"] + 1) // 2, case["tokens"]) if rng.random() < case["chunks"] else 1
        got.append((new, held, ended))
    return got


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"plan": _plan_inputs, "rope": _rope_inputs, "attend": _attend_inputs, "sample": _sample_inputs}[case["op"]](case, g)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _plan_inputs(case, g):
    requests, page = _requests(case), case["page"]
    held = [h for _, h, _ in requests]
    cols = -(-max(n + h for n, h, _ in requests) // page) + 2
    has = _ints([-(-h // page) for h in held])
    pages = case["batch"] * cols + 5
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = order[:case["batch"] * cols].view(case["batch"], cols).clone()
    used = torch.arange(cols, device="cuda") < has[:, None]
    taken = torch.zeros(pages, dtype=torch.bool, device="cuda")
    taken[table[used].long()] = True
    free = order[~taken[order.long()]]
    table[~used] = -1
    return {"case": case, "new": _ints([n for n, _, _ in requests]), "held": _ints(held), "table": table, "free_pages": torch.cat([free, free.new_full((pages - free.numel(),), -1)]),
            "free_count": _ints([free.numel()]), "total": sum(n for n, _, _ in requests),
            "ended": torch.tensor([e for _, _, e in requests], device="cuda") if case["ended"] else None}


def _rope_inputs(case, g):
    t, hq, hk, d, dtype = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    qkv = (_normal(g, t, hq + 2 * hk, d) * torch.exp(0.3 * _normal(g, d)) * 2).to(dtype)
    first = int(torch.randint(case["far"], (1,), generator=g, device="cuda"))
    state = {"case": case, "q": qkv[:, :hq], "k": qkv[:, hq:hq + hk],
             "positions": ((first + torch.arange(t, device="cuda")) % case["far"]).to(torch.int32),
             "inv_freq": torch.tensor([case["base"] ** (-2.0 * i / case["rotary"]) for i in range(case["rotary"] // 2)], dtype=torch.float64, device="cuda")}
    for name in ("q_weight", "k_weight"):
        w = 1.0 + 0.2 * _normal(g, d)
        state[name] = (w if case["w32"] else w.to(dtype)) if case["norm"] else None
    return state


def _visible(case, n, length):
    """Positions that some query of a sequence sees: [0, a) and [b, length)."""
    first = max(0, length - n - case["window"] + 1)
    return min(case["sinks"], first), first


def _attend_inputs(case, g):
    new, old = _lengths(case)
    b, hk, d, page, block = case["batch"], case["kv_heads"], case["dim"], case["page"], case["block"]
    length = [o + n for o, n in zip(old, new)]
    cols = -(-max(length) // page)
    kept = np.zeros((b, cols * page), bool)  # slots that some query sees
    for i in range(b):
        a, first = _visible(case, new[i], length[i])
        kept[i, :a] = True
        kept[i, first:length[i]] = True
    has = kept.reshape(b, cols, page).any(2)
    pages = int(has.sum()) + 3
    table = torch.full((b, cols), -1, dtype=torch.int32, device="cuda")  # the pages between were given back
    table[torch.from_numpy(has).cuda()] = torch.randperm(pages, generator=g, device="cuda")[:pages - 3].to(torch.int32)
    held = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    held[table[table >= 0].long()] = torch.from_numpy(kept.reshape(b, cols, page)[has]).cuda()
    state = {"case": case, "table": table, "cu": _ints(np.concatenate([[0], np.cumsum(new)])), "kv_len": _ints(length), "total": sum(new), "most": max(new)}
    for name in ("k", "v"):
        channel = torch.exp(0.4 * _normal(g, hk, 1, d))  # some channels of a key are larger than others
        x = _normal(g, pages, hk, page, d) * channel
        s = x.view(pages, hk, page // block, block * d).abs().amax(-1) / 448.0
        codes = (x / s.repeat_interleave(block, 2)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        state[name + "_cache"] = torch.where(held[:, None, :, None], codes, 0x7f)  # slots that nobody sees hold anything
        state[name + "_scale"] = s
    state["q"] = (_normal(g, state["total"], case["q_heads"], d) * 1.5).to(DTYPES[case["dtype"]])
    return state


def _sample_inputs(case, g):
    rows, vocab = case["rows"], case["vocab"]
    x = _normal(g, rows, vocab) * case["spread"]
    x += 4.0 * case["spread"] * (_uniform(g, rows, vocab) < 20.0 / vocab)  # what the context asks for stands out
    if case["masked"]:  # rows whose grammar allows few tokens
        few = (_uniform(g, rows, 1) < case["masked"]) & (_uniform(g, rows, vocab) > 0.01)
        few[:, vocab // 2] = False
        x = x.masked_fill(few, float("-inf"))
    t = 0.6 + 0.7 * _uniform(g, rows)
    state = {"case": case, "logits": x.to(DTYPES[case["dtype"]]), "uniform": _uniform(g, rows),
             "temperature": torch.where(_uniform(g, rows) < case["greedy"], 0.0, t), "top_k": None, "top_p": None, "min_p": None}
    if case["top_k"]:
        state["top_k"] = torch.randint((case["top_k"] + 1) // 2, case["top_k"] + 1, (rows,), generator=g, device="cuda").to(torch.int32)
    if case["top_p"] < 1.0:
        state["top_p"] = case["top_p"] * (1.0 - 0.1 * _uniform(g, rows))
    if case["min_p"] > 0.0:
        state["min_p"] = case["min_p"] * (1.0 - 0.5 * _uniform(g, rows))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"plan": _plan, "rope": _rope, "attend": _attend, "sample": _sample}[op](state)


def _own(op, st):
    import luisaml_b200 as lb
    case = st["case"]
    if op == "plan":
        p = lb.kv_plan(st["new"], st["held"], st["table"], st["free_pages"], st["free_count"], page_size=case["page"], total=st["total"], ended=st["ended"])
        return {"cu": p.cu_tokens, "start": p.start, "kv_len": p.kv_len, "positions": p.positions, "slots": p.slots, "free_count": p.free_count,
                "table": st["table"], "free_pages": st["free_pages"]}
    if op == "rope":
        return lb.qk_norm_rope(st["q"], st["k"], st["positions"], st["inv_freq"], st["q_weight"], st["k_weight"], eps=1e-6, interleaved=case["interleaved"])
    if op == "attend":
        return lb.kv_attention(st["q"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"], st["table"], st["cu"], st["kv_len"], max_tokens=st["most"],
                               window=case["window"], sinks=case["sinks"])
    logprob = torch.empty(case["rows"], device="cuda")
    tokens = lb.sample(st["logits"], st["uniform"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"], logprob=logprob)
    return {"tokens": tokens, "logprob": logprob}


def _plan(st):
    page, total, table, free = st["case"]["page"], st["total"], st["table"], st["free_pages"]
    cols = table.shape[1]
    col = torch.arange(cols, device="cuda")
    count, held = st["free_count"], st["held"]
    start = held
    if st["ended"] is not None:  # their pages go onto the free list, in the table's order
        back = st["ended"][:, None] & (col < ((held + page - 1) // page)[:, None]) & (table >= 0)
        at = torch.where(back.view(-1), count + back.view(-1).cumsum(0) - 1, free.numel())
        free.copy_(torch.cat([free, free.new_zeros(1)]).scatter(0, at, torch.where(back, table, 0).view(-1))[:-1])
        table.masked_fill_(back, -1)
        count = count + back.sum().to(torch.int32)
        start = torch.where(st["ended"], 0, held)
    cu = torch.cat([st["new"].new_zeros(1), st["new"].cumsum(0).to(torch.int32)])
    kv_len = start + st["new"]
    had, has = (start + page - 1) // page, (kv_len + page - 1) // page
    need = has - had
    before = need.cumsum(0) - need
    take = (col >= had[:, None]) & (col < has[:, None])
    i = count - 1 - (before[:, None] + col - had[:, None])
    table.copy_(torch.where(take, torch.where(i >= 0, free[i.clamp(0, free.numel() - 1)], -1), table))
    t = torch.arange(total, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], t, right=True)
    positions = start[seq] + t - cu[seq]
    p = table[seq, positions // page]
    return {"cu": cu, "start": start, "kv_len": kv_len, "positions": positions, "slots": torch.where(p >= 0, p * page + positions % page, -1),
            "free_count": (count - need.sum()).clamp(min=0).to(torch.int32), "table": table, "free_pages": free}


def _rope(st):
    case = st["case"]
    r = case["rotary"]
    angle = st["positions"].double()[:, None, None] * st["inv_freq"]
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    got = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
        if case["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        else:
            a, b = y[..., :r // 2], y[..., r // 2:r]
            turned = torch.cat([a * c - b * s, b * c + a * s], -1)
        got.append(torch.cat([turned, y[..., r:]], -1).to(x.dtype))
    return tuple(got)


def _attend(st):
    """Queries padded to [batch, most]; keys: the sinks, and as many from the first query's window on."""
    case = st["case"]
    hk, d, page, block, window, sinks = (case[k] for k in ("kv_heads", "dim", "page", "block", "window", "sinks"))
    group, most = case["q_heads"] // hk, st["most"]
    cu, lens, table = st["cu"].long(), st["kv_len"].long(), st["table"].long()
    b = table.shape[0]
    new = cu[1:] - cu[:-1]
    first = (lens - new - window + 1).clamp(min=0)
    i = torch.arange(most, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=st["total"] - 1)
    q = st["q"].float()[at].view(b, most, hk, group, d).permute(0, 2, 1, 3, 4).reshape(b, hk, most * group, d)
    j = torch.arange(sinks, device="cuda").expand(b, sinks)
    j = torch.cat([torch.where(j < first[:, None], j, -1), first[:, None] + torch.arange(window + most - 1, device="cuda")], 1)  # [B, keys], -1: none
    j = torch.where(j < lens[:, None], j, -1)
    p = table.gather(1, j.clamp(min=0) // page).clamp(min=0)
    slot = j.clamp(min=0) % page

    def values(name):
        x = st[name + "_cache"].view(torch.float8_e4m3fn)[p, :, slot].float() * st[name + "_scale"][p, :, slot // block][..., None]  # [B, keys, H, D]
        return torch.where((j >= 0)[..., None, None], x, 0.0).transpose(1, 2)

    scores = (q @ values("k").transpose(2, 3)) / math.sqrt(d)
    pos = ((lens - new)[:, None] + i)[..., None]  # [B, most, 1]
    keys = j[:, None]
    see = (keys >= 0) & (keys <= pos) & ((keys > pos - window) | (keys < sinks))
    scores = scores.view(b, hk, most, group, -1).masked_fill(~see[:, None, :, None, :], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top > float("-inf"), top, 0.0))
    total = w.sum(-1, keepdim=True)
    o = (w.view(b, hk, most * group, -1) @ values("v")).view(b, hk, most, group, d)
    o = torch.where(total > 0, o / total, 0.0)
    t = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    return o[seq, :, t - cu[seq]].reshape(st["total"], case["q_heads"], d).to(DTYPES[case["dtype"]])


def _sample(st):
    x = st["logits"].float()
    rows, vocab = x.shape
    greedy = (st["temperature"] <= 0)[:, None]
    top = x.amax(1, keepdim=True)
    t = torch.where(greedy, 1.0, st["temperature"][:, None]).double()
    w = torch.exp((x.double() - top.double()) / t)
    w = torch.where(w < LEAST, 0.0, w)
    kept = torch.ones_like(x, dtype=torch.bool)
    if st["top_k"] is not None or st["top_p"] is not None:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        in_order = w.gather(1, order)
        rank = torch.arange(vocab, device="cuda")
        first = rank < vocab
        if st["top_k"] is not None:
            first = rank < torch.where(st["top_k"] > 0, st["top_k"], vocab)[:, None]
        if st["top_p"] is not None:
            m = torch.where(first, in_order, 0.0)
            first = first & ((m.cumsum(1) - m < st["top_p"].double()[:, None] * m.sum(1, keepdim=True)) | (rank == 0))
        kept = torch.zeros_like(kept).scatter(1, order, first.expand(rows, vocab))
    if st["min_p"] is not None:
        kept = kept & (w >= st["min_p"].double()[:, None])
    w = torch.where(kept, w, 0.0)
    c = w.cumsum(1)
    drawn = torch.searchsorted(c, st["uniform"].double()[:, None] * c[:, -1:], right=True)
    last = torch.where(w > 0, torch.arange(vocab, device="cuda"), 0).amax(1, keepdim=True)
    token = torch.where(greedy, first_of(x, top), torch.minimum(drawn, last))
    logprob = torch.where(greedy, 0.0, torch.log(w.gather(1, token) / c[:, -1:]))
    return {"tokens": token[:, 0].to(torch.int32), "logprob": logprob[:, 0].float()}


def first_of(x, top):
    """The lowest index of a row's largest value."""
    return torch.where(x == top, torch.arange(x.shape[1], device=x.device), x.shape[1]).amin(1, keepdim=True)


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "plan":
        requests, page = _requests(case), case["page"]
        total = sum(n for n, _, _ in requests)
        moved = sum(-(-h // page) for _, h, e in requests if e) + sum(-(-(n + (0 if e else h)) // page) - (0 if e else -(-h // page)) for n, h, e in requests)
        return {"bytes": case["batch"] * 20 + 8 * total + 8 * moved, "flops": 4 * total}
    size = SIZE[case["dtype"]]
    if case["op"] == "rope":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * size + 4 * case["tokens"], "flops": 8 * n}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + 28 * case["rows"], "flops": 4 * n}
    new, old = _lengths(case)
    hk, d = case["kv_heads"], case["dim"]
    pairs, tokens = 0, 0
    for n, o in zip(new, old):
        a, first = _visible(case, n, o + n)
        tokens += a + o + n - first
        pos = np.arange(o, o + n, dtype=np.int64)
        lo = np.maximum(0, pos - case["window"] + 1)
        pairs += int((pos - lo + 1 + np.minimum(lo, case["sinks"])).sum())
    total = sum(new)
    return {"bytes": 2 * tokens * hk * (d + 4 / case["block"]) + 2 * total * case["q_heads"] * d * size, "flops": 4 * d * case["q_heads"] * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    st = prepare(case, seed)
    return {"rope": _rope64, "attend": _attend64, "sample": _sample64}[case["op"]](case, st)


def _rope64(case, st):
    half = case["rotary"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(st["positions"].double(), st["inv_freq"]))[:, None]
    got = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        y = x.double().clone()
        if w is not None:
            y = w.double() * y / (y.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt()
        even, odd = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(y[..., even], y[..., odd]) * turn
        y[..., even], y[..., odd] = z.real, z.imag
        got.append(y)
    return tuple(got)


def _attend64(case, st):
    page, block, hk, dim, window, sinks = (case[k] for k in ("page", "block", "kv_heads", "dim", "window", "sinks"))
    group = case["q_heads"] // hk
    cu, lens = st["cu"].tolist(), st["kv_len"].tolist()
    out = torch.zeros(st["total"], case["q_heads"], dim, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        a, first = _visible(case, n, length)
        j = torch.cat([torch.arange(a, device="cuda"), torch.arange(first, length, device="cuda")])
        p, slot = st["table"][b].long()[j // page], j % page
        k, v = (st[x + "_cache"].view(torch.float8_e4m3fn)[p, :, slot].double() * st[x + "_scale"][p, :, slot // block].double()[..., None] for x in ("k", "v"))
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = (j > pos) | ((j <= pos - window) & (j >= sinks))
        for h in range(case["q_heads"]):
            s = st["q"][cu[b]:cu[b + 1], h].double() @ k[:, h // group].T / dim ** 0.5
            s[hidden] = -math.inf
            out[cu[b]:cu[b + 1], h] = torch.softmax(s, -1) @ v[:, h // group]
    return out


def _sample64(case, st):
    """Row by row; the tokens are whole numbers."""
    got = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    for r in range(case["rows"]):
        t = float(st["temperature"][r])
        if t <= 0:
            continue
        x = st["logits"][r].double()
        p = torch.softmax(x / t, 0)
        by_size = torch.argsort(x, descending=True, stable=True)
        if st["top_k"] is not None:
            by_size = by_size[:int(st["top_k"][r])]
        share = p[by_size] / p[by_size].sum()
        if st["top_p"] is not None:
            by_size = by_size[:1 + int((share.cumsum(0)[:-1] < float(st["top_p"][r])).sum())]
        if st["min_p"] is not None:
            by_size = by_size[p[by_size] >= float(st["min_p"][r]) * p.max()]
        left = by_size.sort().values
        c = (p[left] / p[left].sum()).cumsum(0)
        i = min(int((c <= float(st["uniform"][r])).sum()), left.numel() - 1)
        got[r] = torch.log(p[left[i]] / p[left].sum())
    return {"tokens": None, "logprob": got}
