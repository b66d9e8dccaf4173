"""The decode step's operators (include/lcml_decode_step.h) against plain
implementations: the plan of a batch, row by row in Python; the norm and
rotation, attention with sinks and sampling in 64 bits.
"""
import math
import random

import numpy as np
import pytest
import torch

from test_decoder_gpu import TYPES, Cache, _attention_bound, _cu, _no_device_error

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _error_word_stays_clear(dev):
    assert _no_device_error() == 0
    yield
    assert _no_device_error() == 0


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------------------
# the plan
# ---------------------------------------------------------------------------
def _plan_of(new, held, ended, table, free, capacity, page, total):
    """The definition, row by row. table: list of lists, free: list; both are changed."""
    cols = len(table[0]) if table else 0
    columns = lambda n: min(-(-n // page), cols)  # noqa: E731
    start = []
    for b, row in enumerate(table):
        start.append(0 if ended[b] else max(0, held[b]))
        if ended[b]:
            for c in range(columns(max(0, held[b]))):
                if row[c] >= 0:
                    if len(free) < capacity:
                        free.append(row[c])
                    row[c] = -1
    cu = [0]
    for n in new:
        cu.append(min(cu[-1] + max(0, n), total))
    kv_len = [s + cu[b + 1] - cu[b] for b, s in enumerate(start)]
    for b, row in enumerate(table):
        for c in range(columns(start[b]), columns(kv_len[b])):
            row[c] = free.pop() if free else -1
    positions, slots = [-1] * total, [-1] * total
    for b, row in enumerate(table):
        for i in range(cu[b + 1] - cu[b]):
            p = start[b] + i
            positions[cu[b] + i] = p
            if p // page < cols and row[p // page] >= 0:
                slots[cu[b] + i] = row[p // page] * page + p % page
    return cu, start, kv_len, positions, slots, [len(free)]


def _pages(held, page, cols, spare, rng):
    need = [min(-(-max(0, h) // page), cols) for h in held]
    order = rng.sample(range(sum(need) + spare), sum(need) + spare)
    table = [[order.pop() if c < n else -1 for c in range(cols)] for n in need]
    return table, order


def _check_plan(dev, new, held, ended, page, cols, spare, total=None, capacity=None, stride=0, in_place=False, use_ended=None):
    import luisaml_b200 as lb
    rng = random.Random(len(new) * 7 + page)
    table, free = _pages(held, page, cols, spare, rng)
    total = sum(max(0, n) for n in new) if total is None else total
    capacity = len(free) + sum(len(r) for r in table) if capacity is None else capacity
    wide = torch.full((len(new), cols + stride), -7, dtype=torch.int32, device=dev)
    wide[:, :cols] = _ints(table, dev).view(len(new), cols)
    free_t = _ints(free + [-9] * (capacity - len(free)), dev)
    count, held_t = _ints([len(free)], dev), _ints(held, dev)
    flags = torch.tensor(ended, dtype=torch.bool, device=dev) if (any(ended) if use_ended is None else use_ended) else None
    kw = {"kv_len": held_t, "free_count_out": count} if in_place else {}
    got = lb.kv_plan(_ints(new, dev), held_t, wide[:, :cols], free_t, count, page_size=page, total=total, ended=flags, **kw)
    if in_place:
        assert got.kv_len is held_t and got.free_count is count
    before = list(free)
    want = _plan_of(new, held, ended, table, free, capacity, page, total)
    for name, w in zip(got._fields, want):
        assert getattr(got, name).tolist() == w, name
    assert wide[:, :cols].tolist() == table and (wide[:, cols:] == -7).all()
    assert free_t[:len(free)].tolist() == free  # what was handed out may be left behind them
    assert len(before) >= 0
    return got


@pytest.mark.parametrize("ended", [0.0, 0.3])
@pytest.mark.parametrize("batch,most,page,stride", [(1, 1, 16, 0), (1, 700, 16, 3), (3, 40, 64, 0), (64, 1, 64, 0), (65, 9, 48, 5), (257, 300, 32, 0), (2500, 3, 16, 1)])
def test_plan(dev, batch, most, page, stride, ended):
    rng = random.Random(batch + most)
    new = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(batch)]
    held = [rng.choice([0, page, rng.randint(0, 500)]) for _ in range(batch)]
    over = [rng.random() < ended for _ in range(batch)]
    cols = max(-(-(n + h) // page) for n, h in zip(new, held)) + 1
    _check_plan(dev, new, held, over, page, cols, spare=batch * cols, stride=stride)
    _check_plan(dev, new, held, over, page, cols, spare=batch * cols, total=sum(new) + 77, in_place=True)  # padded, in place


def test_plan_of_the_most_rows(dev):
    rng = random.Random(5)
    held = [rng.randint(0, 60) for _ in range(16384)]
    over = [rng.random() < 0.2 for _ in range(16384)]
    _check_plan(dev, [rng.choice([0, 1, 1, 1, 9]) for _ in range(16384)], held, over, 16, 6, spare=16384)
    _check_plan(dev, [1] * 16384, held, [False] * 16384, 16, 6, spare=16384, in_place=True)


@pytest.mark.parametrize("page", [1, 2, 3, 4, 5, 7, 48, 65536])
def test_plan_of_long_rows(dev, page):
    """runs of tokens of one row that begin and end inside a page, or span several"""
    rng = random.Random(page)
    new, held = [1, 700, 0, 2, 911, 1, 1301, 5], [rng.randint(0, 3 * page) for _ in range(8)]
    cols = max(-(-(n + h) // page) for n, h in zip(new, held))
    over = [False, False, True, False, True, False, False, False]
    _check_plan(dev, new, held, [False] * 8, page, cols, spare=8 * cols, total=sum(new) + 3)
    _check_plan(dev, new, held, over, page, cols, spare=8 * cols)
    _check_plan(dev, new, held, over, page, cols, spare=cols)  # the list runs out
    short = _no_device_error()
    assert short in (0, 8)
    _check_plan(dev, new, held, over, page, max(1, cols // 2), spare=8 * cols)  # rows longer than the table
    assert _no_device_error() in (0, 7)


def test_plan_of_pages_past_32_bits(dev):
    """slots that int32 does not hold are -1"""
    import luisaml_b200 as lb
    free = _ints([1, (1 << 31) // 64 - 1, (1 << 31) // 64, 0x7fffffff, 3], dev)
    p = lb.kv_plan(_ints([700], dev), _ints([0], dev), _ints([[-1] * 11], dev), free, _ints([5], dev), page_size=64, total=700)
    want = [3 * 64 + i for i in range(64)] + [-1] * 128 + [(1 << 31) - 64 + i for i in range(64)] + [64 + i for i in range(64)] + [-1] * 380
    assert p.slots.tolist() == want and p.positions.tolist() == list(range(700)) and _no_device_error() == 8


def test_plan_of_nothing(dev):
    import luisaml_b200 as lb
    none = _ints([], dev)
    p = lb.kv_plan(none, none, none.view(0, 4), _ints([5, 6], dev), _ints([2], dev), page_size=16, total=3)
    assert p.cu_tokens.tolist() == [0] and p.positions.tolist() == [-1] * 3 and p.free_count.tolist() == [2] and p.kv_len.numel() == 0
    _check_plan(dev, [0, 0], [5, 0], [True, True], 16, 2, spare=1)
    _check_plan(dev, [0, 0], [5, 0], [False, False], 16, 2, spare=1, use_ended=True)
    _check_plan(dev, [3], [0], [False], 16, 1, spare=1)


def test_an_ended_row_whose_entries_are_out_of_order(dev):
    """entries below 0 (an earlier shortage) are left out"""
    import luisaml_b200 as lb
    table = _ints([[3, -1, 4, 5], [9, 8, 7, 6]], dev)
    free = _ints([0, 0, 0, 0, 0, 0], dev)
    p = lb.kv_plan(_ints([17, 1], dev), _ints([60, 30], dev), table, free, _ints([0], dev), page_size=16, total=18, ended=torch.tensor([True, False], device=dev))
    assert table.tolist() == [[5, 4, -1, -1], [9, 8, 7, 6]] and p.free_count.tolist() == [1] and free[:1].tolist() == [3]
    assert p.positions.tolist() == list(range(17)) + [30] and p.slots.tolist() == [80 + i for i in range(16)] + [64, 8 * 16 + 14]


def test_what_does_not_fit_is_reported(dev):
    args = dict(ended=[False, False, False], page=16)
    _check_plan(dev, [40, 20, 30], [0, 0, 3], cols=4, spare=4, **args)  # the list runs out
    assert _no_device_error() == 8
    _check_plan(dev, [40, 20, 30], [0, 0, 40], cols=3, spare=20, **args)  # longer than the table
    assert _no_device_error() == 7
    _check_plan(dev, [4, 20, 30], [0, 7, 40], cols=9, spare=20, total=20, **args)  # more tokens than the maps hold
    assert _no_device_error() == 7
    _check_plan(dev, [4, -20, 30], [0, 7, -40], cols=9, spare=20, **args)  # negative lengths
    assert _no_device_error() == 7
    _check_plan(dev, [0, 0, 0], [60, 60, 60], ended=[True, False, True], page=16, cols=4, spare=1, capacity=6)  # more pages back than the list has room for
    assert _no_device_error() == 7
    _check_plan(dev, [1, 1, 1], [16, 16, 16], cols=0, spare=4, **args)
    assert _no_device_error() == 7
    import luisaml_b200 as lb
    p = lb.kv_plan(_ints([1], dev), _ints([0x7fffffff], dev), _ints([[1]], dev), _ints([2], dev), _ints([1], dev), page_size=16, total=1)
    assert p.kv_len.tolist() == [0x7fffffff] and p.slots.tolist() == [-1] and p.positions.tolist() == [0x7fffffff]
    assert _no_device_error() == 7
    p = lb.kv_plan(_ints([1], dev), _ints([0], dev), _ints([[-1]], dev), _ints([2], dev), _ints([-4], dev), page_size=16, total=1)
    assert p.free_count.tolist() == [0] and p.slots.tolist() == [-1]
    assert _no_device_error() in (7, 8)
    p = lb.kv_plan(_ints([1], dev), _ints([0], dev), _ints([[-1]], dev), _ints([2], dev), _ints([50], dev), page_size=16, total=1)
    assert p.free_count.tolist() == [0] and p.slots.tolist() == [32]
    assert _no_device_error() == 7


def test_plan_refusals(dev):
    import luisaml_b200 as lb
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    ok = dict(new_tokens=i(2), held=i(2), block_table=i(2, 3), free_pages=i(4), free_count=i(1), page_size=16, total=2)
    lb.kv_plan(**ok)
    for bad in (dict(new_tokens=i(3)), dict(held=i(2).long()), dict(block_table=i(3, 2).t()), dict(free_pages=i(8)[::2]), dict(free_count=i(2)), dict(page_size=0),
                dict(total=-1), dict(ended=i(2)), dict(ended=i(3).bool()), dict(kv_len=i(3)), dict(free_count_out=i(2)), dict(held=i(2).cpu()), dict(page_size=1 << 40),
                dict(block_table=i(1, 3).expand(2, 3))):
        with pytest.raises(ValueError):
            lb.kv_plan(**{**ok, **bad})
    with pytest.raises(lb.LcmlError):
        lb.kv_plan(**{**ok, "page_size": 65537})


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------
def _rope64(x, pos, freq, w, eps, interleaved):
    """The definition, and what its terms come to without their signs."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    r = 2 * freq.numel()
    t = pos.double()[:, None, None] * freq.double()
    c, s = torch.cos(t), torch.sin(t)
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    p, q, size = a * c - b * s, b * c + a * s, a.abs() + b.abs()
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat([u, v], -1))
    return torch.cat([join(p, q), y[..., r:]], -1), torch.cat([join(size, size), y[..., r:].abs()], -1)


def _check_rope(x, pos, freq, w, eps, interleaved, got):
    want, size = _rope64(x, pos, freq, w, eps, interleaved)
    # fp32 inside: the sum of squares, at most 16 of a lane's terms and 5 of lanes' deep, with
    # a rounding each of squares, reaches the norm by half; its root and the products take
    # 6 more; the angle's rounding to fp32 is pi 2^-25 at most and sincospi's 2 steps of
    # 2^-24; two products and a sum take 3. 32 * 2^-24 of |a| + |b| covers them. Then one
    # rounding to the type, half a step (below the normal range: 2^-25 in halves).
    half = torch.finfo(x.dtype).eps / 2
    bound = 32 * 2.0 ** -24 * size * (1 + half) + half * want.abs() + 2.0 ** -25 * (x.dtype == torch.float16) + 2.0 ** -126
    assert got.dtype == x.dtype and ((got.double() - want).abs() <= bound).all()


def _freq(rotary, dev, base=10000.0):
    return torch.tensor([base ** (-2.0 * i / rotary) for i in range(rotary // 2)], dtype=torch.float64, device=dev)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary", [(1, 32, 8, 128, 128), (1, 1, 1, 2, 2), (7, 5, 1, 64, 64), (700, 4, 4, 80, 80), (33, 20, 4, 96, 24), (5, 3, 1, 256, 64),
                                                     (3, 2, 1, 512, 512), (2, 3, 2, 130, 66), (9, 2, 1, 384, 10), (4, 4, 2, 128, 0), (6, 0, 3, 64, 32), (300, 7, 7, 16, 16)])
def test_rope(dev, dtype, tokens, hq, hk, dim, rotary, interleaved):
    import luisaml_b200 as lb
    g = torch.Generator(device=dev).manual_seed(dim + tokens)
    t = TYPES[dtype]
    q, k = ((torch.randn(tokens, h, dim, generator=g, device=dev) * 3).to(t) for h in (hq, hk))
    pos = torch.randint(0, 100000, (tokens,), generator=g, device=dev).to(torch.int32)
    freq = _freq(rotary, dev)
    for wt in {t, torch.float32}:
        qw, kw = ((1 + 0.3 * torch.randn(dim, generator=g, device=dev)).to(wt) for _ in range(2))
        a, b = lb.qk_norm_rope(q, k, pos, freq, qw, kw, eps=1e-5, interleaved=interleaved)
        _check_rope(q, pos, freq, qw, 1e-5, interleaved, a)
        _check_rope(k, pos, freq, kw, 1e-5, interleaved, b)
    f32 = freq.float()
    a, b = lb.qk_norm_rope(q, k, pos, f32, None, kw, interleaved=interleaved)  # a norm of the keys alone, frequencies in fp32
    _check_rope(q, pos, f32, None, 1e-6, interleaved, a)
    _check_rope(k, pos, f32, kw, 1e-6, interleaved, b)


@pytest.mark.parametrize("tokens", [1, 3, 200, 3000])
def test_rope_of_a_packed_projection_in_place(dev, tokens):
    """q and k as slices of one projection, turned in place; the values beside them stay"""
    import luisaml_b200 as lb
    for dim, off in ((128, 0), (64, 0), (64, 1), (64, 4)):  # starts of every alignment
        qkv = torch.randn(tokens, 13, dim + 8, device=dev).bfloat16()
        was = qkv.clone()
        q, k = qkv[:, :8, off:off + dim], qkv[:, 8:10, off:off + dim]
        w = 1 + 0.1 * torch.randn(dim, device=dev)
        pos = torch.arange(tokens, dtype=torch.int32, device=dev) + 1000
        a, b = lb.qk_norm_rope(q, k, pos, _freq(dim, dev), w, w, q_out=q, k_out=k)
        assert a is q and b is k
        _check_rope(was[:, :8, off:off + dim], pos, _freq(dim, dev), w, 1e-6, False, q)
        _check_rope(was[:, 8:10, off:off + dim], pos, _freq(dim, dev), w, 1e-6, False, k)
        qkv[:, :10, off:off + dim] = was[:, :10, off:off + dim]
        assert torch.equal(qkv, was)


def test_rope_far_positions_and_skipped_tokens(dev):
    import luisaml_b200 as lb
    pos = _ints([0, 1, -1, (1 << 20) - 1, 10 ** 7, -(1 << 31), 0x7fffffff], dev)
    q = torch.randn(7, 3, 64, device=dev)
    out = torch.full((7, 3, 64), 9.0, device=dev)
    a, b = lb.qk_norm_rope(q, q[:, :1], pos, _freq(64, dev, 500000.0), q_out=out)
    keep = torch.tensor([0, 1, 3, 4], device=dev)
    _check_rope(q[keep], pos[keep], _freq(64, dev, 500000.0), None, 1e-6, False, a[keep])
    assert (a[2] == 9).all() and (a[5] == 9).all()
    assert torch.equal(a[0], q[0])
    # 2^31 positions: 2^-53 of the turns of the product and of the frequency, 2^-21 of a turn
    want, size = _rope64(q[6:], pos[6:], _freq(64, dev, 500000.0), None, 1e-6, False)
    assert ((a[6:].double() - want).abs() <= size * (2 * math.pi * 2.0 ** -20 + 32 * 2.0 ** -24)).all()


def test_rope_strides(dev):
    """heads before tokens, and tokens further apart than 32 bits count"""
    import luisaml_b200 as lb
    pos = torch.arange(7, dtype=torch.int32, device=dev) + 50
    q, k = torch.randn(5, 7, 64, device=dev).half().transpose(0, 1), torch.randn(2, 7, 64, device=dev).half().transpose(0, 1)
    w = torch.ones(64, device=dev)
    out = torch.empty(5, 7, 64, device=dev, dtype=torch.float16).transpose(0, 1)
    a, b = lb.qk_norm_rope(q, k, pos, _freq(64, dev), w, w, q_out=out)
    assert a is out
    _check_rope(q, pos, _freq(64, dev), w, 1e-6, False, a)
    _check_rope(k, pos, _freq(64, dev), w, 1e-6, False, b)
    big = torch.empty((1 << 31) + 1024, dtype=torch.bfloat16, device=dev)
    q = big.as_strided((3, 4, 64), (1 << 30, 64, 1))
    q.copy_(torch.randn(3, 4, 64, device=dev))
    was = q.clone()
    lb.qk_norm_rope(q, q[:, :0], pos[:3], _freq(64, dev), q_out=q)
    _check_rope(was, pos[:3], _freq(64, dev), None, 1e-6, False, q)


def test_rope_special_values(dev):
    """An infinity or NaN reaches its own pair (and with a norm its head), nothing else."""
    import luisaml_b200 as lb
    q = torch.randn(4, 2, 64, device=dev).half()
    q[1, 0, 3], q[2, 1, 50] = float("nan"), float("inf")
    pos = _ints([5, 6, 7, 8], dev)
    a, _ = lb.qk_norm_rope(q, q, pos, _freq(32, dev))
    bad = torch.zeros(4, 2, 64, dtype=torch.bool, device=dev)
    bad[1, 0, [3, 19]] = True
    assert torch.equal(a.isnan(), bad) and a[2, 1, 50] == float("inf") and a[2, 1, 51].isfinite()
    a, _ = lb.qk_norm_rope(q, q, pos, _freq(32, dev), torch.ones(64, device=dev))
    assert torch.equal(a.isnan().any(-1), torch.tensor([[False, False], [True, False], [False, True], [False, False]], device=dev))
    a, _ = lb.qk_norm_rope(torch.zeros_like(q), q, pos, _freq(32, dev), torch.ones(64, device=dev))
    assert (a == 0).all()


def test_rope_refusals(dev):
    import luisaml_b200 as lb
    q, k, pos, f = torch.zeros(2, 4, 64, device=dev), torch.zeros(2, 1, 64, device=dev), _ints([0, 1], dev), _freq(64, dev)
    w = torch.ones(64, device=dev)
    lb.qk_norm_rope(q, k, pos, f)
    for a, kw in (((q, k[:1], pos, f), {}), ((q, k.half(), pos, f), {}), ((q, k, pos.long(), f), {}), ((q, k, pos[:1], f), {}), ((q, k, pos, f.half()), {}),
                  ((q, k, pos, torch.cat([f, f])), {}), ((q, k, pos, f, w[:32]), {}), ((q, k, pos, f, w.half(), w), {}), ((q, k, pos, f, w, w.bfloat16()), {}),
                  ((q, k, pos, f), {"q_out": q.half()}), ((q, k, pos, f), {"k_out": q}), ((q.transpose(1, 2), k, pos, f), {}), ((q, k, pos.cpu(), f), {}),
                  ((q, k, pos, f), {"q_out": q[:, :1].expand(2, 4, 64)}), ((q.double(), k.double(), pos, f), {})):
        with pytest.raises((ValueError, lb.LcmlError)):
            lb.qk_norm_rope(*a, **kw)
    with pytest.raises(lb.LcmlError):
        lb.qk_norm_rope(torch.zeros(2, 4, 65, device=dev), torch.zeros(2, 1, 65, device=dev), pos, f[:8])
    a, b = lb.qk_norm_rope(q[:0], k[:0], pos[:0], f)
    assert a.shape == (0, 4, 64)


# ---------------------------------------------------------------------------
# attention with sinks
# ---------------------------------------------------------------------------
def _sinks64(q, k, v, pos, length, scale, window, sinks, softcap):
    s = q @ k.T * scale
    reach = (q.abs() @ k.abs().T * scale).amax()
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    j = torch.arange(length, device=q.device)
    s = s.masked_fill((j > pos[:, None]) | ((j <= pos[:, None] - window) & (j >= sinks)), -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    return p @ v, lse, p @ v.abs(), reach


def _check_sinks(dev, new, lens, heads, group, dim, page, block, dtype, window, sinks, softcap=0.0, variant=0, seed=0):
    """Pages that nobody sees are not in the table, slots that nobody sees hold NaN."""
    import luisaml_b200 as lb
    cache = Cache(dev, lens, max(lens), heads, dim, page, block, seed=seed)
    full = cache.table.clone()
    hidden = torch.zeros(len(lens), cache.table.shape[1] * page, dtype=torch.bool, device=dev)
    for b, (n, length) in enumerate(zip(new, lens)):
        hidden[b, min(sinks, length):max(0, length - n - window + 1)] = True
    by_page = hidden.view(len(lens), -1, page)
    at, rows = cache.table.long(), by_page[..., None, :, None].expand(-1, -1, heads, -1, dim)
    codes = [x.clone() for x in (cache.k, cache.v)]
    for x in (cache.k, cache.v):
        x[at] = torch.where(rows, 0x7f, x[at])
    cache.table = torch.where(by_page.all(-1), -1, cache.table)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    q = (torch.randn(sum(new), heads * group, dim, generator=g, device=dev) * 1.5).to(TYPES[dtype])
    lse = torch.empty(sum(new), heads * group, device=dev)
    kw = dict(max_tokens=max(new), window=window, sinks=sinks, softcap=softcap, variant=variant, lse=lse)
    out = lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, **kw)
    assert torch.equal(out, lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, **kw))
    cache.table = full
    cache.k, cache.v = codes
    first = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        k, v = cache.tokens("k", b, length), cache.tokens("v", b, length)
        pos = torch.arange(length - n, length, device=dev)
        sv = cache.vs[cache.table[b].long()]
        sv = sv[sv > 0]
        for h in range(heads * group if n else 0):
            qq = q[first:first + n, h].double()
            ref, ref_lse, weighted, reach = _sinks64(qq, k[h // group], v[h // group], pos, length, dim ** -0.5, window, sinks, softcap)
            bound = _attention_bound(ref, weighted, reach, dim, length, float(v[h // group].abs().max()), float(sv.max() / sv.min()), softcap, q.dtype)
            got = out[first:first + n, h].double()
            assert ((got - ref).abs() <= bound).all(), (b, h)
            d = (lse[first:first + n, h].double() - ref_lse).abs()
            assert (d <= 2 * ((dim + 8) * 2.0 ** -24 * float(reach) + softcap * 2.0 ** -20 + 2.0 ** -18)).all()
        first += n


@pytest.mark.parametrize("window,sinks", [(1, 1), (20, 4), (128, 16), (100, 129), (300, 1000), (2000, 3), (17, 250)])
@pytest.mark.parametrize("dim,group,page,block,dtype", [(128, 4, 64, 64, "bf16"), (64, 5, 48, 16, "f16"), (256, 1, 32, 32, "bf16")])
def test_sinks_of_single_tokens(dev, dim, group, page, block, dtype, window, sinks):
    _check_sinks(dev, [1] * 6, [1, 20, 33, 500, 1300, 257], 2, group, dim, page, block, dtype, window, sinks)


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("window,sinks,softcap", [(1, 4, 0.0), (37, 17, 0.0), (200, 130, 20.0), (129, 300, 0.0), (5000, 8, 0.0)])
@pytest.mark.parametrize("dim,group,page,block,dtype", [(64, 5, 48, 16, "f16"), (128, 2, 256, 64, "bf16"), (256, 1, 32, 16, "bf16")])
def test_sinks_of_runs_of_queries(dev, dim, group, page, block, dtype, window, sinks, softcap, variant):
    if variant == 2 and dim == 256:
        pytest.skip("the tensor-core kernel serves head_dim 64 and 128")
    _check_sinks(dev, [4, 1, 130, 0, 33, 300], [700, 1, 130, 9, 1000, 901], 2, group, dim, page, block, dtype, window, sinks, softcap, variant)


def test_sinks_of_long_contexts(dev):
    """the chunks of a row are joined; long chunks over several row blocks"""
    _check_sinks(dev, [1, 1], [20011, 700], 1, 4, 128, 64, 64, "bf16", 15000, 100)
    _check_sinks(dev, [700, 513], [5000, 513], 1, 4, 128, 16, 16, "bf16", 600, 37, variant=2)


def test_no_sinks_is_the_plain_call(dev):
    import luisaml_b200 as lb
    cache = Cache(dev, [900, 300], 900, 2, 128, 64, 64)
    for n in (1, 200):
        q = torch.randn(2 * n, 4, 128, device=dev).bfloat16()
        args = (q, *cache.args(), cache.table, _cu([n, n], dev), cache.lens)
        assert torch.equal(lb.kv_attention(*args, max_tokens=n), lb.kv_attention(*args, max_tokens=n, sinks=5))
        assert torch.equal(lb.kv_attention(*args, max_tokens=n, window=50), lb.kv_attention(*args, max_tokens=n, window=50, sinks=0))
        all_seen = lb.kv_attention(*args, max_tokens=n, window=50, sinks=0x7fffffff)
        assert (all_seen.float() - lb.kv_attention(*args, max_tokens=n).float()).abs().max() < 0.05
    with pytest.raises(ValueError):
        lb.kv_attention(*args, max_tokens=n, window=50, sinks=-1)


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def _kept(x, t, k, p, m, slacks):
    """Tokens that stay, by rising index, for each of some relative slacks of what top_p compares; and all weights."""
    with np.errstate(invalid="ignore"):
        w = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / t))
    order = np.arange(len(x))
    if k > 0 or p < 1:
        order = np.argsort(-x, kind="stable")
    if k > 0:
        order = order[:k]
    cuts = {len(order)}
    if p < 1:
        c = np.cumsum(w[order])
        cuts = {1 + int((c[:-1] < p * c[-1] * (1 + slack)).sum()) for slack in slacks}
    kept = [order[:n] for n in cuts]
    return [np.sort(o[w[o] >= min(m, 1.0)] if m > 0 else o) for o in kept], w


def _check_sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    import luisaml_b200 as lb
    rows = logits.shape[0]
    logprob = torch.empty(rows, device=logits.device)
    kw = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    got = lb.sample(logits, u, logprob=logprob, **kw)
    again = lb.sample(logits, u, **kw)
    assert got.dtype == torch.int32 and torch.equal(got, again)
    get = lambda v, r, off: off if v is None else float(v[r])  # noqa: E731
    tokens = got.tolist()
    for r in range(rows):
        x = logits[r].double().cpu().numpy()
        x = np.where(np.isnan(x), -np.inf, x)
        t, k, p, m = get(temperature, r, 1.0), int(get(top_k, r, 0)), get(top_p, r, 1.0), get(min_p, r, 0.0)
        if x.max() == -np.inf:
            assert tokens[r] == -1 and logprob[r].isnan()
            continue
        if not t > 0 or x.max() == np.inf:
            assert tokens[r] == int(np.argmax(x)) and logprob[r] == 0
            continue
        p = 1.0 if math.isnan(p) else p
        # Sums of up to 2^19 weights in 64 bits, in any order, and weights good to 1e-12:
        # the border between two tokens is uncertain by less than 1e-11 of the sum.
        # Where a token hangs on that (equal weights whose sum meets top_p exactly), the
        # draw and its logprob are those of one side of the border.
        fine, wants = set(), []
        sets, w = _kept(x, t, k, p, m, (-1e-11, 0.0, 1e-11))
        for kept in sets:
            c, last = np.cumsum(w[kept]), int(np.nonzero(w[kept] > 0)[0][-1])
            share = min(max(float(u[r]), 0.0), 1.0)
            for off in (-1e-11, 0.0, 1e-11):
                i = int((c <= (share + off) * c[-1]).sum())
                i = min(i, last)
                fine.add(int(kept[i]))
                if kept[i] == tokens[r]:
                    wants.append(math.log(w[kept][i] / c[-1]))
        assert tokens[r] in fine, (r, tokens[r], fine)
        # the fp32 output: half a step, and 1e-11 of the share
        assert any(abs(float(logprob[r]) - want) <= 2.0 ** -24 * abs(want) + 1e-10 for want in wants), r
    return got


def _rows(dev, rows, vocab, dtype="f32", spread=2.5, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + vocab)
    return (torch.randn(rows, vocab, generator=g, device=dev) * spread).to(TYPES[dtype]), torch.rand(rows, generator=g, device=dev)


def _all(dev, rows, v, dtype=torch.float32):
    return torch.full((rows,), v, dtype=dtype, device=dev)


SETTINGS = [{}, {"temperature": 0.7}, {"top_k": 50}, {"top_p": 0.9}, {"min_p": 0.05}, {"temperature": 1.3, "top_k": 200, "top_p": 0.8, "min_p": 0.02}, {"top_k": 2000, "top_p": 0.95},
            {"temperature": 0.05, "top_p": 0.99}, {"temperature": 30.0, "top_p": 0.999}, {"top_k": 1}, {"top_p": 0.0}, {"min_p": 1.0}, {"temperature": 5.0, "top_p": 0.3}]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 33, 1000, 4099, 50001])
def test_sample(dev, vocab, dtype):
    x, u = _rows(dev, 5, vocab, dtype)
    for s in SETTINGS:
        _check_sample(x, u, **{k: _all(dev, 5, v, torch.int32 if k == "top_k" else torch.float32) for k, v in s.items()})


@pytest.mark.parametrize("vocab,dtype", [(128001, "f32"), (200003, "f32"), (500000, "f32"), (500001, "bf16"), (900001, "f16")])
def test_sample_of_large_vocabularies(dev, vocab, dtype):
    """rows over several CTAs, and rows that their shared memory does not hold"""
    x, u = _rows(dev, 2, vocab, dtype)
    for s in ({}, {"top_k": 40, "top_p": 0.9}, {"top_p": 0.95}, {"top_k": 100000}, {"min_p": 0.001}):
        _check_sample(x, u, **{k: _all(dev, 2, v, torch.int32 if k == "top_k" else torch.float32) for k, v in s.items()})


@pytest.mark.parametrize("rows", [1, 3, 20, 200])
def test_sample_a_batch_of_different_rows(dev, rows):
    x, u = _rows(dev, rows, 3001, seed=rows)
    g = torch.Generator(device=dev).manual_seed(rows)
    pick = lambda *v: torch.tensor(v, device=dev)[torch.randint(len(v), (rows,), generator=g, device=dev)]  # noqa: E731
    x[::3] += 8.0 * (torch.rand(x[::3].shape, generator=g, device=dev) < 0.002)
    x[1::4] = x[1::4].masked_fill(torch.rand(x[1::4].shape, generator=g, device=dev) < 0.99, -math.inf)
    _check_sample(x, u, temperature=pick(0.0, 0.5, 1.0, -1.0, math.nan, 2.0), top_k=pick(0, 1, 5, 40, 700, 5000, -3).to(torch.int32),
                  top_p=pick(0.1, 0.9, 1.0, 0.99, -1.0, 2.0, math.nan), min_p=pick(0.0, 0.1, 0.01, -1.0, math.nan, 1.5))


def test_sample_ties(dev):
    """Equal logits go by their index: all equal, a few values, a great many at the cut."""
    u = torch.linspace(0, 0.999, 9, device=dev)
    for vocab in (7, 1000, 70001):
        x = torch.zeros(9, vocab, device=dev)
        for s in ({}, {"top_k": 5}, {"top_k": vocab // 2 + 1}, {"top_p": 0.5}, {"top_p": 0.3, "top_k": 6}, {"min_p": 0.5}):
            _check_sample(x, u, **{k: _all(dev, 9, v, torch.int32 if k == "top_k" else torch.float32) for k, v in s.items()})
        g = torch.Generator(device=dev).manual_seed(vocab)
        x = torch.randint(0, 4, (9, vocab), generator=g, device=dev).float() - 1.0
        x[x == 0] = -0.0
        x[:, ::2] = torch.where(x[:, ::2] == 0, 0.0, x[:, ::2])  # both zeros are one value
        for s in ({}, {"top_k": 3}, {"top_k": vocab * 2 // 3}, {"top_p": 0.5}, {"top_p": 0.9}, {"top_p": 0.97, "top_k": vocab * 4 // 5}):
            _check_sample(x.bfloat16(), u, **{k: _all(dev, 9, v, torch.int32 if k == "top_k" else torch.float32) for k, v in s.items()})


def test_sample_one_token_that_outweighs_the_others(dev):
    """the cut far below the first bin, whose mass is almost all"""
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.rand(12, 60001, generator=g, device=dev) * 1e-3
    x[:, 777] = torch.linspace(9.0, 14.5, 12, device=dev)
    for p in (0.5, 0.8, 0.9, 0.97):
        _check_sample(x, torch.linspace(0.01, 0.99, 12, device=dev), top_p=_all(dev, 12, p))


def test_sample_special_values(dev):
    inf, nan = math.inf, math.nan
    x = torch.randn(8, 500, device=dev)
    x[0] = -inf
    x[1] = nan
    x[2, 100:] = nan
    x[3, [7, 300]] = inf
    x[4, :499] = -inf
    x[5] = x[5] * 1e30
    x[6] = x[6] * 1e-40
    x[7, 0], x[7, 1] = 3.4e38, -3.4e38
    u = torch.full((8,), 0.6, device=dev)
    for s in SETTINGS + [{"temperature": inf}, {"temperature": 1e-30, "top_p": 0.5}, {"temperature": 1e30, "top_p": 0.5}, {"temperature": 1e38, "min_p": 0.5}]:
        _check_sample(x, u, **{k: _all(dev, 8, v, torch.int32 if k == "top_k" else torch.float32) for k, v in s.items()})


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [700, 30001])
def test_sample_masks_of_the_lowest_value(dev, vocab, dtype):
    """rows whose mask is the type's lowest value: of all tokens, of all but one, of all but a few"""
    x, u = _rows(dev, 5, vocab, dtype)
    lowest = torch.finfo(x.dtype).min
    x[0] = lowest
    x[1, :vocab - 1] = lowest
    x[2, 3:] = lowest
    x[3, ::2] = lowest
    x[4] = -math.inf
    x[4, 5] = lowest
    for s in SETTINGS:
        _check_sample(x, u, **{k: _all(dev, 5, v, torch.int32 if k == "top_k" else torch.float32) for k, v in s.items()})


def test_sample_uniform_at_its_ends(dev):
    x, _ = _rows(dev, 6, 900)
    x[:, :5] = -math.inf
    u = torch.tensor([0.0, -1.0, 1.0, 2.0, math.nan, 1.0 - 2.0 ** -24], device=dev)
    import luisaml_b200 as lb
    got = lb.sample(x, u)
    assert got.tolist()[:5] == [5, 5, 899, 899, 5]
    _check_sample(x[5:], u[5:])


def test_sample_strides_streams_and_outputs(dev):
    import luisaml_b200 as lb
    for dtype in ("f32", "bf16"):
        for off in (0, 1, 3, 4):  # row starts of every alignment
            big, u = _rows(dev, 6, 2061, dtype)
            x = big[:, off:off + 2050]
            _check_sample(x, u, top_p=_all(dev, 6, 0.9))
    out = torch.full((6,), -5, dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lb.sample(x, u, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert got is out and torch.equal(out, lb.sample(x, u))
    # two captured calls, replayed in turn, on the same and on different rows
    graphs, outs = [], []
    for part in (x, x[2:], x):
        outs.append(torch.empty(part.shape[0], dtype=torch.int32, device=dev))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            lb.sample(part, u[:part.shape[0]], top_p=_all(dev, part.shape[0], 0.8), out=outs[-1])
    for _ in range(3):
        for g in graphs:
            g.replay()
    for part, o in zip((x, x[2:], x), outs):
        assert torch.equal(o, lb.sample(part, u[:part.shape[0]], top_p=_all(dev, part.shape[0], 0.8)))
    assert lb.sample(x[:0], u[:0]).shape == (0,)


def test_sample_rows_far_apart(dev):
    x, u = _rows(dev, 3, 5000)
    big = torch.empty((1 << 31) + 5000, dtype=torch.float32, device=dev)
    far = big.as_strided((3, 5000), (1 << 30, 1))
    far.copy_(x)
    _check_sample(far, u, top_p=_all(dev, 3, 0.9))


def test_sample_draws_by_the_probabilities(dev):
    """of 65536 evenly spaced numbers each token gets its share, to one"""
    import luisaml_b200 as lb
    n = 65536
    x = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.1], device=dev)
    u = (torch.arange(n, device=dev) + 0.5) / n
    got = torch.bincount(lb.sample(x.expand(n, 5).contiguous(), u).long(), minlength=5)
    assert ((got - n * torch.softmax(x.double(), 0)).abs() <= 1).all()


def test_sample_refusals(dev):
    import luisaml_b200 as lb
    x, u = torch.zeros(2, 9, device=dev), torch.zeros(2, device=dev)
    i = torch.zeros(2, dtype=torch.int32, device=dev)
    lb.sample(x, u)
    for a, kw in (((x[0], u), {}), ((x, u[:1]), {}), ((x, u.double()), {}), ((x.t(), u), {}), ((x.double(), u), {}), ((x, u), {"top_k": u}), ((x, u), {"top_k": i.long()}),
                  ((x, u), {"top_p": u[:1]}), ((x, u), {"temperature": u.half()}), ((x, u), {"min_p": u.cpu()}), ((x, u), {"out": u}), ((x, u), {"logprob": i}),
                  ((x[:1].expand(2, 9), u), {})):
        with pytest.raises(ValueError):
            lb.sample(*a, **kw)
    with pytest.raises(lb.LcmlError):
        lb.sample(x[:, :0], u)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_a_captured_step_moves_on(dev):
    """plan, norm and rotation, cache write, attention and sampling in one graph: ten replays are ten eager steps"""
    import luisaml_b200 as lb
    batch, hq, hk, dim, page, vocab, steps = 5, 4, 2, 64, 16, 1000, 40
    g = torch.Generator(device=dev).manual_seed(0)
    emb, proj = torch.randn(vocab, (hq + 2 * hk) * dim, generator=g, device=dev).half(), (torch.randn(hq * dim, vocab, generator=g, device=dev) / 8).half()
    w, freq, us = torch.ones(dim, device=dev), _freq(dim, dev), torch.rand(steps, batch, generator=g, device=dev)
    ended = [[(s + 3 * b) % 17 == 16 for b in range(batch)] for s in range(steps)]

    class State:
        def __init__(self):
            pages = 60
            self.k, self.v = (torch.zeros(pages, hk, page, dim, dtype=torch.uint8, device=dev) for _ in range(2))
            self.ks, self.vs = (torch.zeros(pages, hk, 1, device=dev) for _ in range(2))
            self.table, self.held = _ints([[-1] * 6] * batch, dev), _ints([0] * batch, dev)
            self.free, self.count = torch.arange(pages, dtype=torch.int32, device=dev), _ints([pages], dev)
            self.token, self.new, self.ended, self.u = _ints([1, 2, 3, 4, 5], dev), _ints([1] * batch, dev), torch.zeros(batch, dtype=torch.bool, device=dev), torch.zeros(batch, device=dev)

        def step(self):
            p = lb.kv_plan(self.new, self.held, self.table, self.free, self.count, page_size=page, total=batch, ended=self.ended, kv_len=self.held, free_count_out=self.count)
            qkv = emb[self.token.long()].view(batch, hq + 2 * hk, dim)
            q, k, v = qkv.split((hq, hk, hk), 1)
            q, k = lb.qk_norm_rope(q, k, p.positions, freq, w, w)
            cache = (self.k, self.v, self.ks, self.vs)
            lb.kv_cache_write(*cache, k, v, self.table, p.cu_tokens, p.start)
            o = lb.kv_attention(q, *cache, self.table, p.cu_tokens, p.kv_len, max_tokens=1, window=12, sinks=3)
            lb.sample(o.view(batch, -1) @ proj, self.u, top_p=torch.full((batch,), 0.9, device=dev), out=self.token)
            return p

    eager, seen = State(), []
    for s in range(steps):
        eager.u.copy_(us[s])
        eager.ended.copy_(torch.tensor(ended[s], device=dev))
        eager.step()
        seen.append((eager.token.tolist(), eager.held.tolist(), eager.count.item()))
    replayed = State()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        State().step()  # warm up on another state
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed.step()
    for s in range(steps):
        replayed.u.copy_(us[s])
        replayed.ended.copy_(torch.tensor(ended[s], device=dev))
        graph.replay()
        assert (replayed.token.tolist(), replayed.held.tolist(), replayed.count.item()) == seen[s], s
    assert torch.equal(eager.table, replayed.table) and torch.equal(eager.k, replayed.k)
    used = sum(-(-h // page) for h in replayed.held.tolist())
    assert replayed.count.item() == 60 - used
    pages = [int(p) for row, h in zip(replayed.table.tolist(), replayed.held.tolist()) for p in row[:-(-h // page)]] + replayed.free[:60 - used].tolist()
    assert sorted(pages) == list(range(60))  # no page lost, none twice
