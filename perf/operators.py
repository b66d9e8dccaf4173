"""The operators of an FP8 decoder layer, as cases to measure: RMS norm with the
residual's addition and an e4m3 output, the quantizing write into a paged e4m3
key/value cache, the read back from it, and the attention over it.

`run` computes a case in plain torch operations (fp32 inside) where `own` is
false, and through luisaml_b200's entry points where it is true.
"""
import math
import random

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -100  # the least scale of a block that is not all zeros
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    norm = {"op": "norm", "eps": 1e-6}
    gqa = {"q_heads": 32, "kv_heads": 8, "dim": 128}
    return [
        # one token of a 4096-wide decoder layer: the residual's addition, the norm and the per-token quantization
        # that feed its FP8 GEMMs; latency counts
        dict(norm, name="norm_1x4096", rows=1, cols=4096, dtype="bf16", residual=True, static=False),
        # a batch of prompts of odd length, an fp32 stream of odd width, the calibrated per-tensor scale
        dict(norm, name="norm_8191x5000", rows=8191, cols=5000, dtype="f32", residual=False, static=True),
        # one decode step of 64 sequences: one token each joins a partly filled block, whose scale may grow
        dict(gqa, name="write_64x1", op="write", batch=64, tokens=1, context=1000, page=64, block=64, dtype="bf16"),
        # prompts of 5 sequences of different lengths
        dict(gqa, name="write_5x4000", op="write", batch=5, tokens=4000, context=0, page=64, block=16, dtype="f16"),
        # a short prefix brought back as fp32
        dict(name="read_1x300", op="read", batch=1, tokens=300, context=0, q_heads=4, kv_heads=4, dim=64, page=16, block=16, dtype="f32"),
        # prefixes of 32 sequences brought back for another consumer
        dict(gqa, name="read_32x2000", op="read", batch=32, tokens=2000, context=100, page=128, block=64, dtype="bf16"),
        # a single chat's next token: the smallest call
        dict(gqa, name="decode_1x513", op="attend", batch=1, tokens=1, context=512, page=16, block=16, dtype="bf16", window=0, softcap=0.0),
        # a serving batch's decode step, contexts from short to 4096
        dict(gqa, name="decode_64x4096", op="attend", batch=64, tokens=1, context=4096, page=64, block=64, dtype="bf16", window=0, softcap=0.0),
        # one long document's next token
        dict(gqa, name="decode_1x131072", op="attend", batch=1, tokens=1, context=131071, page=256, block=64, dtype="bf16", window=0, softcap=0.0),
        # four drafted tokens of each of 16 sequences verified at once; capped scores
        dict(name="verify_16x4", op="attend", batch=16, tokens=4, context=2000, q_heads=40, kv_heads=8, dim=64, page=32, block=32, dtype="f16", window=0, softcap=30.0),
        # two whole prompts
        dict(gqa, name="prompt_2x4096", op="attend", batch=2, tokens=4096, context=0, page=64, block=64, dtype="bf16", window=0, softcap=0.0),
        # the next chunks of four prompts behind a cached prefix, in a layer with a sliding window
        dict(name="chunk_4x1000", op="attend", batch=4, tokens=1000, context=8000, q_heads=16, kv_heads=2, dim=64, page=48, block=16, dtype="f16", window=1500, softcap=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one(rng):
    op = rng.choice(["norm", "write", "read", "attend", "attend", "attend"])
    if op == "norm":
        return {"op": op, "eps": 1e-6, "rows": _log(rng, 1, 8191), "cols": _log(rng, 257, 8192), "dtype": rng.choice(["f32", "f16", "bf16"]),
                "residual": rng.random() < 0.5, "static": rng.random() < 0.3}
    c = {"op": op, "kv_heads": rng.choice([1, 2, 4, 5, 8]), "dim": rng.choice([64, 128]), "block": rng.choice([16, 32, 64])}
    c["q_heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 5, 7, 8])
    c["page"] = c["block"] * rng.choice([1, 2, 3, 4])
    if op in ("write", "read"):
        c.update(batch=_log(rng, 1, 64), tokens=_log(rng, 1, 4000), context=rng.choice([0, _log(rng, 1, 2000)]), dtype=rng.choice(["f32", "f16", "bf16"]))
        return c
    c.update(dtype=rng.choice(["f16", "bf16"]), window=rng.choice([0, 0, _log(rng, 64, 3000)]), softcap=rng.choice([0.0, 0.0, 30.0]))
    how = rng.choice(["decode", "long", "verify", "prompt", "chunk"])
    if how == "decode":
        c.update(batch=_log(rng, 1, 100), tokens=1, context=_log(rng, 1, 4096))
    elif how == "long":
        c.update(batch=1, tokens=1, context=_log(rng, 4096, 131071))
    elif how == "verify":
        c.update(batch=_log(rng, 1, 32), tokens=rng.randint(2, 8), context=_log(rng, 1, 4096))
    elif how == "prompt":
        c.update(batch=rng.randint(1, 4), tokens=_log(rng, 16, 4096), context=0)
    else:
        c.update(batch=rng.randint(1, 6), tokens=_log(rng, 16, 1000), context=_log(rng, 16, 8000))
    return c


def draw(rng):
    most = [work(c) for c in listed()]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        c = _one(rng)
        w = work(c)
        if any(w[k] > most[k] for k in w) or (c["op"] != "norm" and _slots(c) * c["kv_heads"] * c["dim"] > 64 * 4200 * 8 * 128):
            continue
        if c["op"] == "attend" and c["batch"] * c["q_heads"] * c["tokens"] * (c["context"] + c["tokens"]) > 2 * 32 * 4096 * 4096:
            continue
        return c


def _lengths(case):
    """New tokens and earlier tokens of each sequence: the first has the most of both, the others spread below."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k not in ("name", "dtype"))))
    b, n, c = case["batch"], case["tokens"], case["context"]
    one = case["op"] == "attend" and n <= 8  # a decode or verifying step brings the same number of tokens for all
    new = [n] + [n if one else rng.randint((n + 1) // 2, n) for _ in range(b - 1)]
    old = [c] + [rng.randint(c // 8, c) for _ in range(b - 1)]
    return new, old


def _pages(case):
    """Pages in a sequence's row of the block table: room for the padded grid of blocks the plain write works on."""
    return -(-(case["tokens"] + case["context"] + 2 * case["block"]) // case["page"])


def _slots(case):
    return case["batch"] * _pages(case) * case["page"]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        spread = torch.exp(0.5 * normal(cols))  # channels of different size, as a trained layer has
        state["x"] = (normal(rows, cols) * spread).to(dtype)
        state["residual"] = (normal(rows, cols) * spread * 4).to(dtype) if case["residual"] else None
        state["weight"] = (1.0 + 0.2 * normal(cols)).to(dtype)
        state["scale"] = torch.full((1,), 0.03, device="cuda") if case["static"] else None
        return state
    new, old = _lengths(case)
    b, hk, d, page, block = case["batch"], case["kv_heads"], case["dim"], case["page"], case["block"]
    cols = _pages(case)
    pages = b * cols + 3
    table = torch.randperm(pages, generator=g, device="cuda")[:b * cols].view(b, cols).to(torch.int32)
    state["table"] = table
    state["cu"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    state["start"] = torch.tensor(old, dtype=torch.int32, device="cuda")
    state["total"], state["most"] = sum(new), max(new)
    written = [o if case["op"] == "write" else o + n for o, n in zip(old, new)]  # what the cache holds before the call
    state["kv_len"] = torch.tensor([o + n for o, n in zip(old, new)], dtype=torch.int32, device="cuda")
    # which slots of which page hold a token
    position = torch.arange(cols * page, device="cuda").view(1, cols, page)
    held = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    held[table.long()] = position < torch.tensor(written, device="cuda").view(b, 1, 1)
    for name in ("k", "v"):
        channel = torch.exp(0.4 * normal(hk, 1, d))  # some channels of a key are larger than others
        cache = torch.empty(pages, hk, page, d, dtype=torch.uint8, device="cuda")
        scales = torch.empty(pages, hk, page // block, device="cuda")
        for at in range(0, pages, 2048):
            m = held[at:at + 2048]
            x = normal(m.shape[0], hk, page, d) * channel * m[:, None, :, None]
            amax = x.view(-1, hk, page // block, block * d).abs().amax(-1)
            s = amax / E4M3_MAX
            div = torch.where(s > 0, s, 1.0).repeat_interleave(block, 2)[..., None]
            cache[at:at + 2048] = (x / div).to(torch.float8_e4m3fn).view(torch.uint8)
            if case["op"] == "attend":  # slots that hold no token hold anything
                cache[at:at + 2048] = torch.where(m[:, None, :, None], cache[at:at + 2048], 0x7f)
                s = torch.where(m[:, ::block][:, None, :], s, float("nan"))
            scales[at:at + 2048] = s
        state[name + "_cache"], state[name + "_scale"] = cache, scales
    if case["op"] == "write":
        for name in ("k", "v"):
            size = torch.exp(0.4 * normal(state["total"], hk, 1))  # a token may be larger than its block so far
            state[name] = (normal(state["total"], hk, d) * size).to(dtype)
    elif case["op"] == "attend":
        state["q"] = (normal(state["total"], case["q_heads"], d) * 1.5).to(dtype)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"norm": _norm, "write": _write, "read": _read, "attend": _attend}[op](state)


def _own(op, st):
    import luisaml_b200 as lb
    case = st["case"]
    if op == "norm":
        q, s, h = lb.rmsnorm_quantize(st["x"], st["weight"], residual=st["residual"], eps=case["eps"], scale=st["scale"])
        return _norm_out(q.view(torch.float8_e4m3fn), s, h, case)
    cache = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
    if op == "write":
        lb.kv_cache_write(*cache, st["k"], st["v"], st["table"], st["cu"], st["start"])
        return _cache_out(st)
    if op == "read":
        return lb.kv_cache_read(*cache, st["table"], st["cu"], st["start"], total=st["total"], dtype=DTYPES[case["dtype"]])
    return lb.kv_attention(st["q"], *cache, st["table"], st["cu"], st["kv_len"], max_tokens=st["most"],
                           window=case["window"], softcap=case["softcap"])


def _norm_out(q, s, h, case):
    out = {"q": q}
    if not case["static"]:
        out["scale"] = s
    if case["residual"]:
        out["h"] = h
    return out


def _cache_out(st):
    return {"k": st["k_cache"].view(torch.float8_e4m3fn), "v": st["v_cache"].view(torch.float8_e4m3fn), "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _encode(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _decode(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _norm(st):
    case = st["case"]
    h = st["x"].float()
    if case["residual"]:
        h = h + st["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + case["eps"]) * st["weight"].float()
    if case["static"]:
        s = st["scale"]
        q = _encode(y / s)
    else:
        s = y.abs().amax(-1) / E4M3_MAX
        s = torch.where(s > 0, s, 1.0)
        q = _encode(y / s[:, None])
    return _norm_out(q, s, h.to(DTYPES[case["dtype"]]) if case["residual"] else None, case)


def _write(st):
    """Works on a padded grid of blocks [batch, blocks, block]; slots that nothing changes are written back as they are."""
    case = st["case"]
    page, block, d = case["page"], case["block"], case["dim"]
    start, cu, table = st["start"].long(), st["cu"].long(), st["table"].long()
    count = (st["most"] + block - 2) // block + 1
    slot = torch.arange(count * block, device="cuda")
    pos = (start // block * block)[:, None] + slot  # [B, count * block]
    t = pos - start[:, None]
    fresh = (t >= 0) & (t < (cu[1:] - cu[:-1])[:, None])
    at = (t + cu[:-1, None]).clamp(0, st["total"] - 1)
    where = table.gather(1, pos // page), pos % page
    head = pos[:, ::block]
    head = table.gather(1, head // page), head % page // block
    before = (head[0] >= 0) & (pos[:, ::block] < start[:, None])  # blocks that hold earlier tokens
    touched = fresh.view(-1, count, block).any(-1)
    for name in ("k", "v"):
        cache, scales = st[name + "_cache"], st[name + "_scale"]
        x = st[name].float()[at].view(-1, count, block, case["kv_heads"], d)
        f = fresh.view(-1, count, block, 1, 1)
        amax = torch.where(f, x.abs(), 0.0).amax((2, 4))  # [B, count, H]
        s = amax / E4M3_MAX
        s = torch.where(amax > 0, s.clamp(min=MIN_SCALE), 0.0)
        had = scales[head[0], :, head[1]]
        held = torch.where(before[..., None], had, 0.0)
        s = torch.maximum(s, held)
        div = torch.where(s > 0, s, 1.0)[:, :, None, :, None]
        codes = cache[where[0], :, where[1]].view(x.shape)
        again = _encode(_decode(codes) * held[:, :, None, :, None] / div).view(torch.uint8)
        grew = (before & touched)[:, :, None, None, None] & (s > held)[:, :, None, :, None]
        earlier = (pos < start[:, None]).view(f.shape)
        out = torch.where(f, _encode(x / div).view(torch.uint8), torch.where(grew & earlier, again, codes))
        cache[where[0], :, where[1]] = out.view(*pos.shape, case["kv_heads"], d)
        scales[head[0], :, head[1]] = torch.where(touched[..., None], s, had)
    return _cache_out(st)


def _read(st):
    case = st["case"]
    cu = st["cu"].long()
    t = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = st["start"].long()[seq] + t - cu[seq]
    p, slot = st["table"].long()[seq, pos // case["page"]], pos % case["page"]
    got = []
    for name in ("k", "v"):
        y = _decode(st[name + "_cache"][p, :, slot]) * st[name + "_scale"][p, :, slot // case["block"]][..., None]
        got.append(y.to(DTYPES[case["dtype"]]))
    return tuple(got)


def _attend(st):
    """Queries padded to [batch, most], keys to the block table's width."""
    case = st["case"]
    hk, d, page, block = case["kv_heads"], case["dim"], case["page"], case["block"]
    group, most = case["q_heads"] // hk, st["most"]
    cu, lens, table = st["cu"].long(), st["kv_len"].long(), st["table"].long()
    b, width = table.shape[0], table.shape[1] * page
    new = cu[1:] - cu[:-1]
    i = torch.arange(most, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=st["total"] - 1)
    q = st["q"].float()[at].view(b, most, hk, group, d).permute(0, 2, 1, 3, 4).reshape(b, hk, most * group, d)
    held = (torch.arange(width, device="cuda") < lens[:, None])[:, None, :, None]

    def values(name):
        x = _decode(st[name + "_cache"][table])  # [B, pages, H, page, D]
        x = x * st[name + "_scale"][table].repeat_interleave(block, 3)[..., None]
        return torch.where(held, x.permute(0, 2, 1, 3, 4).reshape(b, hk, width, d), 0.0)

    scores = (q @ values("k").transpose(2, 3)) / math.sqrt(d)
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    pos = (lens - new)[:, None] + i  # [B, most]
    j = torch.arange(width, device="cuda")
    see = (j <= pos[..., None]) & (j < lens[:, None, None])
    if case["window"]:
        see &= j > pos[..., None] - case["window"]
    see = see[:, None, :, None, :]
    scores = scores.view(b, hk, most, group, width).masked_fill(~see, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > float("-inf"), top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, most * group, width) @ values("v")).view(b, hk, most, group, d)
    o = torch.where(total > 0, o / total, 0.0)
    t = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    o = o[seq, :, t - cu[seq]]
    return o.reshape(st["total"], case["q_heads"], d).to(DTYPES[case["dtype"]])


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        per = size * (3 if case["residual"] else 1) + 1
        return {"bytes": n * per + case["cols"] * size + case["rows"] * (0 if case["static"] else 4), "flops": 6 * n}
    new, old = _lengths(case)
    hk, d, block = case["kv_heads"], case["dim"], case["block"]
    total = sum(new)
    if case["op"] in ("write", "read"):
        n = 2 * total * hk * d
        return {"bytes": n * (size + 1) + 8 * hk * sum(-(-x // block) for x in new), "flops": 2 * n}
    window = case["window"]
    pairs, tokens = 0, 0
    for n, o in zip(new, old):
        first = max(0, o - window + 1) if window else 0
        tokens += o + n - first
        seen = np.arange(o + 1, o + n + 1, dtype=np.int64)
        pairs += int((np.minimum(seen, window) if window else seen).sum())
    return {"bytes": 2 * tokens * hk * (d + 4 / block) + 2 * total * case["q_heads"] * d * size, "flops": 4 * d * case["q_heads"] * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _round64(x):
    """Nearest e4m3 value, ties to the even one, saturating."""
    x = x.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        h = st["x"].double() + (st["residual"].double() if case["residual"] else 0.0)
        y = h / torch.sqrt(torch.mean(h ** 2, 1, keepdim=True) + case["eps"]) * st["weight"].double()
        s = st["scale"].double().expand(case["rows"]) if case["static"] else y.abs().max(1).values / 448
        return _norm_out(_round64(y / s[:, None]), s, h, case)
    block, page, hk = case["block"], case["page"], case["kv_heads"]
    table, cu, start, lens = (st[k].tolist() for k in ("table", "cu", "start", "kv_len"))
    value = {n: st[n + "_cache"].view(torch.float8_e4m3fn) for n in ("k", "v")}
    if case["op"] == "write":
        value = {n: v.double() for n, v in value.items()}
        scale = {n: st[n + "_scale"].double() for n in ("k", "v")}
        for b, row in enumerate(table):
            n = cu[b + 1] - cu[b]
            for first in range(start[b] // block * block, start[b] + n, block):
                p, r = row[first // page], first % page
                lo, hi = max(first, start[b]), min(first + block, start[b] + n)
                for name in ("k", "v"):
                    x = st[name][cu[b] + lo - start[b]:cu[b] + hi - start[b]].double().transpose(0, 1)  # [H, tokens, D]
                    s = x.abs().amax((1, 2)) / 448
                    s = torch.where(s > 0, s.clamp(min=MIN_SCALE), s)
                    if lo > first:
                        was = scale[name][p, :, r // block].clone()
                        s = torch.maximum(s, was)
                        v = value[name][p, :, r:r + lo - first]
                        again = _round64(v * (was / torch.where(s > 0, s, 1.0))[:, None, None])
                        value[name][p, :, r:r + lo - first] = torch.where((s > was)[:, None, None], again, v)
                    value[name][p, :, r + lo - first:r + hi - first] = _round64(x / torch.where(s > 0, s, 1.0)[:, None, None])
                    scale[name][p, :, r // block] = s
        return {"k": value["k"], "v": value["v"], "k_scale": scale["k"], "v_scale": scale["v"]}

    def tokens(name, b, lo, hi):
        """[H, hi - lo, D] of sequence b in 64 bits"""
        rows = [table[b][i] for i in range(lo // page, -(-hi // page))]
        x = value[name][rows].double() * st[name + "_scale"][rows].double().repeat_interleave(block, 2)[..., None]
        x = x.transpose(0, 1).reshape(hk, -1, case["dim"])
        return x[:, lo - lo // page * page:][:, :hi - lo]

    if case["op"] == "read":
        got = [[tokens(n, b, start[b], lens[b]).transpose(0, 1) for b in range(case["batch"])] for n in ("k", "v")]
        return tuple(torch.cat(x) for x in got)
    group = case["q_heads"] // hk
    out = torch.zeros(st["total"], case["q_heads"], case["dim"], dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n, length = cu[b + 1] - cu[b], lens[b]
        k, v = tokens("k", b, 0, length), tokens("v", b, 0, length)
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")
        hidden = (j > pos) | ((j <= pos - case["window"]) if case["window"] else (j < 0))
        for h in range(case["q_heads"]):
            s = st["q"][cu[b]:cu[b + 1], h].double() @ k[h // group].T / case["dim"] ** 0.5
            if case["softcap"]:
                s = torch.tanh(s / case["softcap"]) * case["softcap"]
            s[hidden] = -math.inf
            out[cu[b]:cu[b + 1], h] = torch.softmax(s, -1) @ v[h // group]
    return out
