"""The decoder-layer operators at the edges of what their arguments may hold:
scores far apart, padded and partial batches, in-place outputs, value scales far
apart, sequences without tokens. Plain implementations in 64 bits as in
test_decoder_gpu.py."""
import ctypes

import numpy as np
import pytest
import torch

from test_decoder_gpu import TYPES, Cache, _attend, _attention64, _check_attention, _check_norm, _check_write, _cu

pytestmark = pytest.mark.gpu


def _device_error():
    import luisaml_b200 as lb
    code = ctypes.c_int(0)
    lb.lib().lcml_device_error(ctypes.byref(code))
    return code.value


@pytest.fixture(autouse=True)
def _error_word_stays_clear(dev):
    assert _device_error() == 0
    yield
    assert _device_error() == 0


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (64, "bf16"), (128, "f16"), (128, "bf16")])
@pytest.mark.parametrize("nats", [60, 88, 95, 100, 150, 250, 400])
def test_a_score_far_above_the_earlier_ones(dev, nats, dim, dtype, variant):
    """A key of a later tile that takes the whole softmax, in each of 16 neighbouring positions (one per head), for every
    row and for one row alone"""
    import luisaml_b200 as lb
    n, length, heads = 40, 330, 16
    for rows in (slice(None), slice(21, 22)):
        cache = Cache(dev, [length], length, heads, dim, 64, 16, seed=nats)
        cache.k[cache.table[0].long()] = 0
        cache.ks.fill_(1.0)
        for h in range(heads):
            key = 192 + h  # within a tile that every row sees in full
            cache.k[int(cache.table[0, key // 64]), h, key % 64] = 0x38  # 1.0
        q = torch.zeros(n, heads, dim, device=dev, dtype=TYPES[dtype])
        q[rows] = 1.0
        lse = torch.empty(n, heads, device=dev)
        scale = nats / dim
        out = lb.kv_attention(q, *cache.args(), cache.table, _cu([n], dev), cache.lens, max_tokens=n, scale=scale, lse=lse, variant=variant)
        _check_attention(cache, q, [n], [length], out, lse, scale=scale)


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("new,total,most", [([3], 512, 512), ([5, 0, 2], 700, 300), ([100, 3], 200, 100), ([0, 0], 400, 200), ([30] * 40, 1500, 30),
                                            ([260, 40], 600, 300), ([1] * 30, 240, 8), ([1] * 64, 2000, 1)])
def test_padded_queries(dev, new, total, most, dim, dtype):
    """a packed dimension longer than cu_tokens[batch]: every query is computed, the padding is left alone"""
    import luisaml_b200 as lb
    heads, group = 8, 4
    lens = [n + 150 + 31 * (i % 5) for i, n in enumerate(new)]
    cache = Cache(dev, lens, max(lens) + 5, heads, dim, 32, 16)
    q = torch.randn(total, heads * group, dim, device=dev).to(TYPES[dtype])
    out, lse = torch.full_like(q, 7.0), torch.full((total, heads * group), 7.0, device=dev)
    lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, max_tokens=most, out=out, lse=lse)
    _check_attention(cache, q, new, lens, out, lse)
    assert (out[sum(new):] == 7).all() and (lse[sum(new):] == 7).all()


def test_a_captured_batch_replayed_with_fewer_tokens(dev):
    import luisaml_b200 as lb
    heads, group, dim = 2, 4, 128
    new = [100] * 40
    cache = Cache(dev, [300] * 40, 300, heads, dim, 32, 16)
    q = torch.randn(sum(new), heads * group, dim, device=dev).bfloat16()
    out, lse = torch.empty_like(q), torch.empty(sum(new), heads * group, device=dev)
    cu = _cu(new, dev)
    call = lambda: lb.kv_attention(q, *cache.args(), cache.table, cu, cache.lens, max_tokens=100, out=out, lse=lse, workspace=ws)  # noqa: E731
    ws = torch.empty(lb.kv_attention_workspace_size(q, *cache.args(), cache.table, cu, cache.lens, max_tokens=100), dtype=torch.uint8, device=dev)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        with torch.cuda.graph(graph, stream=side):
            call()
    torch.cuda.current_stream().wait_stream(side)
    for new, lens in (([100] * 40, [300] * 40), ([1] * 40, [300] * 40), ([(7 * i) % 30 for i in range(40)], [200 + i for i in range(40)])):
        cu.copy_(_cu(new, dev))
        cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(7.0)
        lse.fill_(7.0)
        graph.replay()
        _check_attention(cache, q, new, lens, out, lse)
        assert (out[sum(new):] == 7).all()


def test_padded_writes_and_reads(dev):
    import luisaml_b200 as lb
    start, new, total = [3, 0, 40], [20, 5, 1], 100
    cache = Cache(dev, start, 80, 2, 64, 32, 16)
    k, v = (torch.randn(total, 2, 64, device=dev).bfloat16() for _ in range(2))
    cu = _cu(new, dev)
    _check_write(cache, start, new, k, v, lambda lb: lb.kv_cache_write(*cache.args(), k, v, cache.table, cu, cache.lens))
    got = lb.kv_cache_read(*cache.args(), cache.table, cu, cache.lens, total=total, dtype=torch.float32)
    for a, which in zip(got, "kv"):
        want = torch.cat([cache.tokens(which, b, s + n)[:, s:].transpose(0, 1) for b, (s, n) in enumerate(zip(start, new))])
        assert torch.equal(a[:sum(new)], want.float())


@pytest.mark.parametrize("dtype,cols", [("bf16", 5376), ("bf16", 4104), ("bf16", 2304), ("f16", 3848), ("f32", 2304), ("f32", 5376), ("bf16", 433), ("f32", 33000)])
@pytest.mark.parametrize("rows", [3, 400])
def test_norm_in_place(dev, rows, cols, dtype):
    """h_out = x and h_out = residual, at widths whose last vectors do not fill the threads: bit for bit as with an output of its own"""
    import luisaml_b200 as lb
    g = torch.Generator(device=dev).manual_seed(cols)
    x = torch.randn(rows, cols, generator=g, device=dev)
    r = torch.randn(rows, cols, generator=g, device=dev)
    # the row's maximum lies in what the surplus threads would read, and would grow with another addition
    x[:, -32:], r[:, -32:] = 4.0, 4.0
    x, r = x.to(TYPES[dtype]), r.to(TYPES[dtype])
    w = torch.ones(cols, device=dev)
    want = lb.rmsnorm_quantize(x, w, r)
    _check_norm(x, w, r, 1e-6, *want)
    for turn in range(30):
        for alias in ("x", "residual"):
            a, b = x.clone(), r.clone()
            got = lb.rmsnorm_quantize(a, w, b, h_out=a if alias == "x" else b)
            assert all(torch.equal(p, q) for p, q in zip(got, want)), (turn, alias)


def _check_rows(cache, q, new, lens, out, dtype, share=0.05):
    """Attention against 64 bits with a bound taken row by row from the weights p and value scales s: a weight enters the
    product as a half of p_j s_j over a reference that is at most the row's largest, so beside the relative terms (fp32
    scores, 2^-11, the sum, the output's type) it is off by 2^-25 of max_j(p_j s_j), for every code it multiplies.
    `share`: the bound may not be more of the row's largest output, so a wrong value shows."""
    group, at = q.shape[1] // cache.heads, 0
    half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    for b, (n, length) in enumerate(zip(new, lens)):
        k, v = cache.tokens("k", b, length), cache.tokens("v", b, length)
        s = cache.vs[cache.table[b].long()].double().transpose(0, 1).reshape(cache.heads, -1).repeat_interleave(cache.block, 1)[:, :length]
        codes = cache.v[cache.table[b].long()].view(torch.float8_e4m3fn).double().transpose(0, 1).reshape(cache.heads, -1, cache.dim)[:, :length].abs()
        pos = torch.arange(length - n, length, device=q.device)
        for h in range(q.shape[1]):
            qq, c = q[at:at + n, h].double(), h // group
            ref, lse, weighted, reach = _attention64(qq, k[c], v[c], pos, length, cache.dim ** -0.5, True, 0, 0.0)
            x = (qq @ k[c].T * cache.dim ** -0.5).masked_fill(torch.arange(length, device=q.device) > pos[:, None], -float("inf"))
            p = torch.exp(x - lse[:, None])
            least = 2.0 ** -25 * (p * s[c]).amax(1, keepdim=True) * codes[c].sum(0)
            off = 2 * ((cache.dim + 8) * 2.0 ** -24 * float(reach) + 2.0 ** -20)
            bound = half * ref.abs() + (2.0 ** -25 if dtype == "f16" else 0.0) + (1 + half) * (weighted * (off + 2.0 ** -11 + (length + 16) * 2.0 ** -24) + least)
            assert (bound.amax(1) <= share * ref.abs().amax(1)).all(), "the bound would hide a wrong value"
            err = (out[at:at + n, h].double() - ref).abs()
            assert (err <= bound).all(), (b, h, float((err / ref.abs().amax(1, keepdim=True)).max()), float((err / bound).max()))
        at += n


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1e-2, 1e-4, 1e-8, 1.0, 100.0])
def test_a_block_of_zero_values_beside_small_ones(dev, size, dim, variant):
    """A value block of scale 0 counts in the softmax's sum and nowhere else, however small the other values are; whatever
    its codes say."""
    import luisaml_b200 as lb
    new, lens, heads, group = [1, 40], [600, 333], 2, 2
    for code in (0x00, 0x7e, 0xfe):  # the last two: what an infinity alone in its block leaves behind
        cache = Cache(dev, lens, 600, heads, dim, 32, 16)
        cache.vs *= size
        for b in range(2):
            p = int(cache.table[b, 1])
            cache.v[p, :, 16:] = code
            cache.vs[p, :, 1] = 0
        q = (torch.randn(sum(new), heads * group, dim, device=dev) * 1.5).bfloat16()
        out = lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, max_tokens=40, variant=variant)
        _check_rows(cache, q, new, lens, out, "bf16")


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16")])
def test_value_scales_far_apart(dev, dim, dtype, variant):
    """blocks 2^20 apart, zero blocks among them, several queries a sequence"""
    import luisaml_b200 as lb
    new, lens, heads, group = [30, 1], [500, 200], 2, 2
    cache = Cache(dev, lens, 500, heads, dim, 32, 16)
    g = torch.Generator(device=dev).manual_seed(11)
    cache.vs *= torch.exp2(torch.randint(-10, 11, cache.vs.shape, device=dev, generator=g).float())
    for b in range(2):
        cache.v[int(cache.table[b, 2]), :, :16], cache.vs[int(cache.table[b, 2]), :, 0] = 0, 0
    q = (torch.randn(sum(new), heads * group, dim, device=dev, generator=g) * 1.5).to(TYPES[dtype])
    out = lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, max_tokens=30, variant=variant)
    _check_rows(cache, q, new, lens, out, dtype)


def test_a_sink_without_values(dev):
    """a first block of zero values that takes nearly the whole softmax: the rest is small and still right"""
    import luisaml_b200 as lb
    for dim in (64, 128):
        for variant in (1, 2):
            cache = Cache(dev, [400], 400, 1, dim, 32, 16)
            p = int(cache.table[0, 0])
            cache.v[p, :, :16], cache.vs[p, :, 0] = 0, 0
            cache.k[p, :, :16] = 0x48  # 4.0
            cache.ks[p, :, 0] = 1.0
            cache.vs *= 1e-3
            q = (torch.randn(20, 2, dim, device=dev) * 0.3 + 8.0 / (4.0 * dim ** 0.5)).bfloat16()  # the sink's score is about 8
            out = lb.kv_attention(q, *cache.args(), cache.table, _cu([20], dev), cache.lens, max_tokens=20, variant=variant)
            _check_rows(cache, q, [20], [400], out, "bf16")


def test_sequences_without_new_tokens_are_not_touched(dev):
    """An idle sequence in the middle of a block: its table is not followed, and a page it shares with a sequence that
    writes belongs to that one alone."""
    import luisaml_b200 as lb
    start, new = [5, 21, 40], [0, 1, 0]
    cache = Cache(dev, start, 64, 2, 64, 32, 16)
    k, v = (torch.randn(1, 2, 64, device=dev) * 50 for _ in range(2))
    table = cache.table.clone()
    table[0] = -1  # no pages any more
    cache.table = cache.table[1:2]  # for the oracle: the sequence that writes, alone
    _check_write(cache, start[1:2], new[1:2], k, v, lambda lb: lb.kv_cache_write(*cache.args(), k, v, table, _cu(new, dev), cache.lens))
    lb.kv_cache_read(*cache.args(), table, _cu(new, dev), cache.lens, total=1)


def test_idle_sequences_on_a_shared_page(dev):
    start, new = [21] + [20] * 60, [1] + [0] * 60
    for turn in range(20):
        cache = Cache(dev, start, 64, 4, 64, 32, 16, seed=turn)
        cache.table[1:] = cache.table[0]
        k, v = (torch.randn(1, 4, 64, device=dev) * 50 for _ in range(2))
        _check_write(cache, start, new, k, v, lambda lb: lb.kv_cache_write(*cache.args(), k, v, cache.table, _cu(new, dev), cache.lens))


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 5000, 100])
def test_windows_longer_than_any_sequence(dev, window, variant):
    """with queries before the first token among them"""
    for new, lens in (([12], [4]), ([40, 3], [30, 200])):
        _attend(dev, new, lens, 2, 2, 64, 16, 16, "bf16", variant=variant, window=window)


def test_a_part_of_a_batch(dev):
    """cu_tokens of sequences 2 .. 4 of a longer batch: the packed tokens keep their places"""
    import luisaml_b200 as lb
    new, lens = [300, 5, 70, 0, 40, 9], [300, 50, 100, 30, 333, 60]
    heads, group, dim = 2, 4, 64
    for variant in (0, 1, 2):
        cache = Cache(dev, lens, 340, heads, dim, 32, 16)
        cu = _cu(new, dev)
        q = torch.randn(sum(new), heads * group, dim, device=dev).bfloat16()
        out = torch.full_like(q, 7.0)
        lb.kv_attention(q, *cache.args(), cache.table[2:5], cu[2:6], cache.lens[2:5], max_tokens=70, variant=variant, out=out)
        lo, hi = sum(new[:2]), sum(new[:5])
        whole = Cache(dev, lens, 340, heads, dim, 32, 16)  # the same one
        whole.table = cache.table[2:5]
        _check_attention(whole, q[lo:hi], new[2:5], lens[2:5], out[lo:hi])
        assert (out[:lo] == 7).all() and (out[hi:] == 7).all()
    start = [n - m for n, m in zip(lens, new)]
    first = torch.tensor(start, dtype=torch.int32, device=dev)
    k, v = lb.kv_cache_read(*cache.args(), cache.table[2:5], cu[2:6], first[2:5], total=sum(new), dtype=torch.float32)
    want = torch.cat([cache.tokens("k", b, lens[b])[:, start[b]:].transpose(0, 1) for b in range(2, 5)])
    assert torch.equal(k[lo:hi], want.float())
    x, y = (torch.randn(sum(new), heads, dim, device=dev) * 3 for _ in range(2))
    other = Cache(dev, start, 340, heads, dim, 32, 16, seed=1)
    twin = Cache(dev, start, 340, heads, dim, 32, 16, seed=1)
    lb.kv_cache_write(*other.args(), x, y, other.table[2:5], cu[2:6], first[2:5])
    lb.kv_cache_write(*twin.args(), x[lo:hi].clone(), y[lo:hi].clone(), twin.table[2:5], _cu(new[2:5], dev), first[2:5])
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(other.args(), twin.args()))


def test_negative_lengths_are_reported(dev):
    """and count as a sequence that holds nothing (attention) or is not followed (write, read)"""
    import luisaml_b200 as lb
    cache = Cache(dev, [20, 30], 64, 2, 64, 32, 16)
    before = [t.clone() for t in cache.args()]
    cu = _cu([1, 1], dev)
    bad = torch.tensor([-3, 30], dtype=torch.int32, device=dev)
    q = torch.randn(2, 4, 64, device=dev).half()
    for variant in (1, 2):
        out = lb.kv_attention(q, *cache.args(), cache.table, cu, bad, max_tokens=1, variant=variant)
        assert _device_error() == 7
        assert (out[0] == 0).all()
    lb.kv_cache_read(*cache.args(), cache.table, cu, bad, total=2)
    assert _device_error() == 7
    k = torch.randn(2, 2, 64, device=dev)
    lb.kv_cache_write(*cache.args(), k, k, cache.table, cu, bad)
    assert _device_error() == 7
    p = cache.table[0].long()
    assert all(torch.equal(a[p].nan_to_num(), b[p].nan_to_num()) for a, b in zip(before, cache.args()))


def test_layouts_of_the_output(dev):
    """heads first, one head, one token, rows apart"""
    import luisaml_b200 as lb
    for new, lens, heads in (([5, 1], [60, 9], 2), ([1], [40], 2), ([6], [33], 1)):
        cache = Cache(dev, lens, 60, heads, 64, 16, 16)
        n = sum(new)
        q = torch.randn(n, heads, 64, device=dev).half()
        for out in (torch.empty(heads, n, 64, device=dev).half().transpose(0, 1), torch.empty(n, heads, 64, device=dev).half(),
                    torch.empty(n, 2 * heads + 1, 70, device=dev).half()[:, ::2, 3:67][:, :heads]):
            lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, max_tokens=max(new), out=out)
            _check_attention(cache, q, new, lens, out)
        if n > 1:
            with pytest.raises(lb.LcmlError):
                lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, out=torch.empty(1, heads, 64, device=dev).half().expand(n, -1, -1))
