"""The decoder-layer operators (include/lcml_decoder.h) against plain
implementations in 64 bits: RMS norm with an e4m3 output, the paged e4m3
key/value cache's write and read, attention over it.

Codes and scales of the cache and values read back are compared bit for bit
(the oracle's encoder). The norm's codes may differ where y / s lies at a
rounding boundary, attention within the bound that _attention_bound derives.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _no_device_error():
    import luisaml_b200 as lb
    code = ctypes.c_int(0)
    lb.lib().lcml_device_error(ctypes.byref(code))
    return code.value


@pytest.fixture(autouse=True)
def _error_word_stays_clear(dev):
    assert _no_device_error() == 0
    yield
    assert _no_device_error() == 0


def _decode(codes):
    return codes.view(torch.float8_e4m3fn).double()


def _spacing(v):
    """Distance of neighbouring e4m3 values at |v|."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(2.0 ** -6, 448.0))) - 3)


# ---------------------------------------------------------------------------
# RMS norm
# ---------------------------------------------------------------------------
def _check_norm(x, w, r, eps, q, s, h, static=None):
    h64 = x.double() + (r.double() if r is not None else 0.0)
    y = h64 / torch.sqrt((h64 ** 2).mean(1, keepdim=True) + eps) * w.double()
    # The fp32 sum of squares: at most 48 additions deep plus a rounding each
    # of squares and h; half of that reaches 1 / sqrt; y takes four roundings
    # more: 40 * 2^-24 in all.
    rel = 40 * 2.0 ** -24
    if static is None:
        ref = y.abs().amax(1) / 448
        ref = torch.where(ref > 0, ref, 1.0)
        assert ((s.double() - ref).abs() <= 2 * rel * ref).all()
        v = y / s.double()[:, None]
    else:
        v = y / static
    v = v.clamp(-448, 448)
    got = _decode(q)
    # nearest e4m3 value of a v that is off by 2 rel at most
    assert ((got - v).abs() <= _spacing(v) / 2 * (1 + 2.0 ** -20) + 2 * rel * v.abs()).all()
    if r is not None:
        assert torch.equal(h, (x.float() + r.float()).to(x.dtype))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 433), (5, 5000), (700, 1024), (2, 33000), (4, 8), (400, 2052), (1, 32)])
def test_norm(dev, dtype, rows, cols):
    import luisaml_b200 as lb
    g = torch.Generator(device=dev).manual_seed(rows * 31 + cols)
    t = TYPES[dtype]
    x = (torch.randn(rows, cols, generator=g, device=dev) * 3).to(t)
    r = (torch.randn(rows, cols, generator=g, device=dev) * 5).to(t)
    for wt in {t, torch.float32}:
        w = (1 + 0.3 * torch.randn(cols, generator=g, device=dev)).to(wt)
        q, s, h = lb.rmsnorm_quantize(x, w, r, eps=1e-5)
        _check_norm(x, w, r, 1e-5, q, s, h)
        q, s, h = lb.rmsnorm_quantize(x, w, eps=1e-6)
        assert h is None
        _check_norm(x, w, None, 1e-6, q, s, h)
        fixed = torch.tensor([0.011], device=dev)
        q, s, h = lb.rmsnorm_quantize(x, w, r, scale=fixed, eps=1e-5)
        assert s is fixed
        _check_norm(x, w, r, 1e-5, q, None, h, static=fixed.double())


def test_norm_strides_aliasing_and_rows_apart(dev):
    import luisaml_b200 as lb
    g = torch.Generator(device=dev).manual_seed(5)
    for off in (0, 1, 4):  # row starts of every alignment
        big = torch.randn(37, 700, generator=g, device=dev).to(torch.bfloat16)
        x, r = big[:, off:off + 256], big[:, 300 + off:556 + off]
        w = torch.ones(256, device=dev)
        h = torch.full((37, 300), 7.0, device=dev, dtype=torch.bfloat16)
        q, s, got = lb.rmsnorm_quantize(x, w, r, h_out=h[:, 8:264])
        _check_norm(x, w, r, 1e-6, q, s, got)
        assert (h[:, :8] == 7).all() and (h[:, 264:] == 7).all()
    x, r = (torch.randn(9, 512, generator=g, device=dev) for _ in range(2))
    want = lb.rmsnorm_quantize(x, torch.ones(512, device=dev), r)
    got = lb.rmsnorm_quantize(x, torch.ones(512, device=dev), r, h_out=r)  # the residual stream in place
    assert got[2] is r and all(torch.equal(a, b) for a, b in zip(want, got))


def test_norm_zero_rows_nan_and_empty(dev):
    import luisaml_b200 as lb
    x = torch.randn(4, 640, device=dev)
    x[1] = 0
    x[2, 7] = float("nan")
    q, s, _ = lb.rmsnorm_quantize(x, torch.ones(640, device=dev))
    assert s[1] == 1 and (q[1] == 0).all()
    assert (q[2] & 0x7f == 0x7f).all()  # the row's mean square is NaN
    keep = [0, 3]
    _check_norm(x[keep], torch.ones(640, device=dev), None, 1e-6, q[keep], s[keep], None)
    q, s, _ = lb.rmsnorm_quantize(x[:0], torch.ones(640, device=dev))
    assert q.shape == (0, 640) and s.shape == (0,)


def test_norm_feeds_the_gemm(dev):
    """codes and per-row scales are the GEMM's A and scale_a"""
    import luisaml_b200 as lb
    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn(33, 512, generator=g, device=dev).bfloat16()
    q, s, _ = lb.rmsnorm_quantize(x, torch.ones(512, device=dev))
    wq, sw = lb.quantize_rows_dynamic(torch.randn(256, 512, generator=g, device=dev))
    y = lb.gemm(q, wq, s, sw, out_dtype=torch.float32)
    ref = (_decode(q) * s.double()[:, None]) @ (_decode(wq) * sw.double()[:, None]).T
    assert ((y.double() - ref).abs() <= 1e-3 + 2e-3 * ref.abs()).all()


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
class Cache:
    """A paged cache, its block table and lengths."""

    def __init__(self, dev, lens, room, heads, dim, page, block, seed=0, fill=True):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.dev, self.heads, self.dim, self.page, self.block = dev, heads, dim, page, block
        b, cols = len(lens), max(1, -(-room // page))
        pages = b * cols + 2
        self.table = torch.randperm(pages, generator=g, device=dev)[:b * cols].view(b, cols).to(torch.int32)
        # what holds no token is NaN: it must not matter
        self.k, self.v = (torch.full((pages, heads, page, dim), c, dtype=torch.uint8, device=dev) for c in (0x7f, 0xff))
        self.ks, self.vs = (torch.full((pages, heads, page // block), float("nan"), device=dev) for _ in range(2))
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        if fill:
            for i, n in enumerate(lens):
                for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
                    for first in range(0, n, block):
                        p, slot, m = int(self.table[i, first // page]), first % page, min(block, n - first)
                        x = torch.randn(heads, m, dim, generator=g, device=dev)
                        s = x.abs().amax((1, 2)) / 448 * (0.5 + torch.rand(heads, generator=g, device=dev))
                        codes[p, :, slot:slot + m] = (x / s[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                        scales[p, :, slot // block] = s

    def args(self):
        return self.k, self.v, self.ks, self.vs

    def tokens(self, which, seq, n):
        """[heads, n, dim] in 64 bits"""
        codes, scales = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        rows = self.table[seq].long()
        x = _decode(codes[rows]) * scales[rows].double().repeat_interleave(self.block, 2)[..., None]
        return x.transpose(0, 1).reshape(self.heads, -1, self.dim)[:, :n]


def _cu(lens, dev):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)


def _write_oracle(codes, scales, table, page, block, start, cu, x):
    """The write's definition, block by block, with the oracle's codec; numpy, in place."""
    heads = codes.shape[1]
    for b, s0 in enumerate(start):
        n = cu[b + 1] - cu[b]
        for first in range(s0 // block * block, s0 + n, block):
            p, slot = table[b][first // page], first % page
            lo, hi = max(first, s0), min(first + block, s0 + n)
            for h in range(heads):
                new = x[cu[b] + lo - s0:cu[b] + hi - s0, h]
                amax = np.abs(new[np.isfinite(new)]).max(initial=np.float32(0))
                s = max(amax / np.float32(448), np.float32(2.0 ** -100)) if amax > 0 else np.float32(0)
                old = scales[p, h, slot // block] if lo > first else np.float32(0)
                top = np.float32(max(s, old))
                div = top if top > 0 else np.float32(1)
                if lo > first and s > old:
                    was = oracle.e4m3_decode(codes[p, h, slot:slot + lo - first].copy()).astype(np.float32) * old
                    codes[p, h, slot:slot + lo - first] = oracle.quantize(was.astype(np.float32), div)
                codes[p, h, slot + lo - first:slot + hi - first] = oracle.quantize(np.ascontiguousarray(new), div)
                scales[p, h, slot // block] = top


def _check_write(cache, start, new, k, v, run):
    import luisaml_b200 as lb
    want = []
    cu = np.concatenate([[0], np.cumsum(new)])
    for codes, scales, x in ((cache.k, cache.ks, k), (cache.v, cache.vs, v)):
        c, s = codes.cpu().numpy().copy(), scales.cpu().numpy().copy()
        _write_oracle(c, s, cache.table.cpu().numpy(), cache.page, cache.block, start, cu, x.float().cpu().numpy())
        want += [c, s]
    run(lb)
    for name, a, b in zip(("k", "k_scale", "v", "v_scale"), (cache.k, cache.ks, cache.v, cache.vs), want):
        got = a.cpu().numpy()
        if got.dtype == np.uint8:
            assert np.array_equal(got, b), (name, np.argwhere(got != b)[:3])
        else:
            assert np.array_equal(got.view(np.uint32)[~np.isnan(b)], b.view(np.uint32)[~np.isnan(b)]) and np.isnan(got[np.isnan(b)]).all(), name


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page,block", [(64, 16, 16), (128, 48, 16), (128, 64, 64), (256, 128, 128), (64, 512, 512), (128, 256, 256)])
def test_write(dev, dtype, dim, page, block):
    heads = 3
    start = [0, 5, block, 2 * page - 1, 0, 77]
    new = [1, 40, 2 * block + 3, 2, 0, 1]
    cache = Cache(dev, start, max(a + b for a, b in zip(start, new)) + 1, heads, dim, page, block, seed=dim + block)
    g = torch.Generator(device=dev).manual_seed(3)
    k, v = (torch.randn(sum(new), heads, dim, generator=g, device=dev).mul(torch.exp(torch.randn(sum(new), heads, 1, generator=g, device=dev))).to(TYPES[dtype])
            for _ in range(2))
    _check_write(cache, start, new, k, v, lambda lb: lb.kv_cache_write(*cache.args(), k, v, cache.table, _cu(new, dev), cache.lens))


def test_write_token_by_token_and_again(dev):
    """Tokens that keep growing re-encode their block each time; a repeated call changes nothing."""
    import luisaml_b200 as lb
    heads, dim, page, block = 2, 128, 32, 32
    cache = Cache(dev, [0, 0], 100, heads, dim, page, block)
    for step in range(70):
        start = [step, step]
        k, v = (torch.randn(2, heads, dim, device=dev) * (1 + step % 37) for _ in range(2))
        lens = torch.tensor(start, dtype=torch.int32, device=dev)
        call = lambda lb: lb.kv_cache_write(*cache.args(), k, v, cache.table, _cu([1, 1], dev), lens)  # noqa: E731
        _check_write(cache, start, [1, 1], k, v, call)
        before = [t.clone() for t in cache.args()]
        call(lb)
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(before, cache.args()))


def test_write_many_sequences(dev):
    """more sequences than one search step probes, most of them without tokens"""
    rng = np.random.default_rng(0)
    start = rng.integers(0, 40, 1500).tolist()
    new = (rng.integers(0, 30, 1500) * (rng.random(1500) < 0.3)).tolist()
    cache = Cache(dev, start, 80, 1, 64, 16, 16, fill=False)
    for s in (cache.ks, cache.vs):
        s.fill_(0.01)
    cache.k.fill_(0x31)
    cache.v.fill_(0xb2)
    k, v = (torch.randn(sum(new), 1, 64, device=dev).bfloat16() for _ in range(2))
    _check_write(cache, start, new, k, v, lambda lb: lb.kv_cache_write(*cache.args(), k, v, cache.table, _cu(new, dev), cache.lens))


def test_write_strided_unaligned_and_special_values(dev):
    heads, dim, page, block = 2, 64, 32, 16
    start, new = [3, 0], [20, 17]
    for off in (0, 1):
        cache = Cache(dev, start, 60, heads, dim, page, block, seed=off)
        qkv = torch.randn(37, 5, dim + 2 * off, device=dev).half()  # as a slice of a fused projection
        k, v = qkv[:, 1:3, off:off + dim], qkv[:, 3:5, off:off + dim]
        k[4, 0, 3], k[5, 1, 0], v[30, 1, 9] = float("inf"), float("nan"), float("-inf")
        v[20:36, 0] = 0
        k[20:36, 1] = 6e-8  # a half's least value
        _check_write(cache, start, new, k, v, lambda lb: lb.kv_cache_write(*cache.args(), k, v, cache.table, _cu(new, dev), cache.lens))
    one = torch.randn(1, 1, dim, device=dev).expand(37, heads, dim)  # broadcast tokens: strides of zero
    cache = Cache(dev, start, 60, heads, dim, page, block)
    _check_write(cache, start, new, one, one, lambda lb: lb.kv_cache_write(*cache.args(), one, one, cache.table, _cu(new, dev), cache.lens))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page,block", [(64, 16, 16), (128, 48, 16), (256, 128, 128), (128, 192, 64)])
def test_read(dev, dtype, dim, page, block):
    import luisaml_b200 as lb
    lens = [1, 300, 0, 97, 2 * page]
    start = [0, 13, 0, 96, page - 1]
    cache = Cache(dev, lens, 310, 3, dim, page, block, seed=block)
    new = [n - s for n, s in zip(lens, start)]
    first = torch.tensor(start, dtype=torch.int32, device=dev)
    k, v = lb.kv_cache_read(*cache.args(), cache.table, _cu(new, dev), first, total=sum(new), dtype=TYPES[dtype])
    for got, which in ((k, "k"), (v, "v")):
        want = torch.cat([cache.tokens(which, b, lens[b])[:, start[b]:].transpose(0, 1) for b in range(5)])
        # decode * scale is one fp32 rounding of the 64-bit product, then one of the type's
        assert torch.equal(got, want.float().to(TYPES[dtype]))


def test_read_returns_what_was_written(dev):
    import luisaml_b200 as lb
    new = [100, 33]
    cache = Cache(dev, [0, 0], 100, 4, 128, 64, 64, fill=False)
    k, v = (torch.randn(133, 4, 128, device=dev).bfloat16() for _ in range(2))
    lb.kv_cache_write(*cache.args(), k, v, cache.table, _cu(new, dev), cache.lens)
    got = lb.kv_cache_read(*cache.args(), cache.table, _cu(new, dev), cache.lens, total=133, dtype=torch.float32)
    for a, b in zip((k, v), got):
        # half an e4m3 step: 2^-4 of the value, or 2^-10 of the block's scale (at most 7 / 448) for the smallest
        assert ((a.float() - b).abs() <= a.float().abs() * 2.0 ** -4 * 1.0001 + 2.0 ** -10 * 7 / 448).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attention64(q, k, v, pos, length, scale, causal, window, softcap):
    """One sequence and head in 64 bits: out, lse, and per output the bound's ingredients."""
    s = q @ k.T * scale
    reach = (q.abs() @ k.abs().T * scale).amax() if s.numel() else torch.zeros((), device=q.device)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    j = torch.arange(length, device=q.device)
    hide = (j > pos[:, None]) if causal else (j < 0).expand(len(pos), -1)
    if window:
        hide = hide | (j <= pos[:, None] - window)
    s = s.masked_fill(hide, -math.inf)
    lse = torch.logsumexp(s, -1) if length else torch.full((len(pos),), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.where(lse[:, None] > -math.inf, torch.exp(s - lse[:, None]), 0.0)
    return p @ v, lse, p @ v.abs(), reach


def _attention_bound(ref, weighted, reach, dim, keys, v_most, ratio, cap, dtype):
    """How far the kernel may be off, element by element:
    * a score: fp32 dot of dim products (any order) and a few roundings of
      products with scales, (dim + 8) 2^-24 of sum |q k| scale; the cap's tanh
      8 ulps of cap; the exponent's argument and ex2 2^-20: a weight is off by
      twice that relatively (itself and the sum);
    * each weight enters the product as a half: 2^-11 relatively, and 2^-25
      absolutely (subnormal halves) in units of the largest weight, whose
      value scale may be `ratio` times another's;
    * fp32 accumulation over the keys: keys 2^-24 (sums of positive terms),
    * one rounding to the output's type (8 significant bits: 2^-8, 11: 2^-11)."""
    off = 2 * ((dim + 8) * 2.0 ** -24 * float(reach) + cap * 2.0 ** -20 + 2.0 ** -20)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    return half * ref.abs() + 2.0 ** -24 + (1 + half) * (weighted * (off + 2.0 ** -11 + (keys + 16) * 2.0 ** -24) + keys * 2.0 ** -25 * ratio * v_most)


def _check_attention(cache, q, new, lens, out, lse=None, scale=None, causal=True, window=0, softcap=0.0):
    group = q.shape[1] // cache.heads
    at = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        k, v = cache.tokens("k", b, length), cache.tokens("v", b, length)
        pos = torch.arange(length - n, length, device=q.device)
        sv = cache.vs[cache.table[b].long()][:, :, :]
        sv = sv[sv > 0]
        ratio = float(sv.max() / sv.min()) if sv.numel() else 1.0
        for h in range(q.shape[1] if n else 0):
            qq = q[at:at + n, h].double()
            ref, ref_lse, weighted, reach = _attention64(qq, k[h // group], v[h // group], pos, length, scale or cache.dim ** -0.5, causal, window, softcap)
            most = float(v[h // group].abs().max()) if length else 0.0
            bound = _attention_bound(ref, weighted, reach, cache.dim, length, most, ratio, softcap, q.dtype)
            got = out[at:at + n, h].double()
            err = (got - ref).abs()
            assert not got.isnan().any() and (err <= bound).all(), (b, h, float((err - bound).max()), float(err.max()))
            if lse is not None:
                g = lse[at:at + n, h].double()
                empty = ref_lse == -math.inf
                assert (g[empty] == -math.inf).all()
                d = (g - ref_lse)[~empty].abs()
                assert (d <= 2 * ((cache.dim + 8) * 2.0 ** -24 * float(reach) + softcap * 2.0 ** -20 + 2.0 ** -18)).all()
        at += n


def _attend(dev, new, lens, heads, group, dim, page, block, dtype, variant=0, seed=0, spread=1.5, **kw):
    import luisaml_b200 as lb
    cache = Cache(dev, lens, max(max(lens), 1) + 3, heads, dim, page, block, seed=seed)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    q = (torch.randn(sum(new), heads * group, dim, generator=g, device=dev) * spread).to(TYPES[dtype])
    lse = torch.empty(sum(new), heads * group, device=dev)
    out = lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, max_tokens=max(new), lse=lse, variant=variant, **kw)
    _check_attention(cache, q, new, lens, out, lse, **kw)
    return cache, q, out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,group,dim,page,block", [(2, 4, 128, 16, 16), (1, 8, 64, 48, 16), (3, 1, 128, 64, 64), (1, 16, 256, 32, 32), (2, 5, 64, 128, 64),
                                                        (1, 40, 128, 64, 32)])
def test_decode(dev, dtype, heads, group, dim, page, block):
    _attend(dev, [1] * 7, [1, 2, 15, 16, 17, 500, 1300], heads, group, dim, page, block, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_split_over_many_chunks(dev, dtype):
    """long contexts: the chunks of one row are joined; and many sequences beside a long one"""
    _attend(dev, [1], [20011], 1, 4, 128, 64, 64, dtype)
    _attend(dev, [1] * 40, [9000] + [37 * i for i in range(39)], 1, 2, 64, 32, 16, dtype)


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("kw", [{}, {"window": 1}, {"window": 37}, {"window": 300, "softcap": 20.0}, {"softcap": 3.0}, {"causal": False}, {"scale": 0.3}])
@pytest.mark.parametrize("dim,group,dtype", [(64, 5, "f16"), (128, 2, "bf16"), (256, 1, "bf16")])
def test_runs_of_queries(dev, dim, group, dtype, kw, variant):
    """several queries a sequence: verifying steps, chunks behind a prefix, whole prompts"""
    if variant == 2 and dim == 256:
        pytest.skip("the tensor-core kernel serves head_dim 64 and 128")
    _attend(dev, [4, 1, 130, 0, 33, 300], [700, 1, 130, 9, 1000, 301], 2, group, dim, 48, 16, dtype, variant=variant, **kw)


@pytest.mark.parametrize("dim,page,block,group,dtype", [(128, 64, 64, 4, "bf16"), (128, 16, 16, 1, "f16"), (64, 256, 32, 8, "bf16"), (64, 80, 16, 3, "f16")])
def test_prompts(dev, dim, page, block, group, dtype):
    """the tensor-core kernel over several row blocks and key tiles, boxes of every height"""
    _attend(dev, [700, 129, 1, 385], [700, 1500, 64, 385], 2, group, dim, page, block, dtype, variant=2)
    _attend(dev, [513], [2049], 1, group, dim, page, block, dtype, variant=2, window=200, softcap=30.0)


@pytest.mark.parametrize("variant", [0, 2])
def test_rows_that_see_nothing(dev, variant):
    """more queries than tokens, and sequences that hold none"""
    cache, q, out = _attend(dev, [5, 3, 1], [2, 0, 0], 2, 2, 64, 16, 16, "bf16", variant=variant)
    assert (out[:3] == 0).all() and (out[5:] == 0).all()


def test_scales_of_very_different_size(dev):
    """value scales 2^20 apart between blocks, and blocks of zeros (scale 0)"""
    import luisaml_b200 as lb
    lens = [200, 90]
    cache = Cache(dev, lens, 200, 2, 128, 32, 16)
    cache.vs *= torch.exp2(torch.randint(-10, 11, cache.vs.shape, device=dev).float())
    p = cache.table[0, 1].long()
    cache.k[p, :, :16], cache.v[p, :, :16], cache.ks[p, :, 0], cache.vs[p, :, 0] = 0, 0, 0, 0
    q = torch.randn(2, 4, 128, device=dev).bfloat16()
    out = lb.kv_attention(q, *cache.args(), cache.table, _cu([1, 1], dev), cache.lens, max_tokens=1)
    _check_attention(cache, q, [1, 1], lens, out)


def test_large_and_small_queries(dev):
    """bf16 queries far outside fp16's range: score magnitudes from 0 to one-hot rows"""
    for spread in (1e-6, 1e6, 3e5):
        import luisaml_b200 as lb
        lens = [77, 400]
        cache = Cache(dev, lens, 400, 1, 64, 16, 16)
        q = (torch.randn(2, 3, 64, device=dev) * spread).bfloat16()
        out = lb.kv_attention(q, *cache.args(), cache.table, _cu([1, 1], dev), cache.lens, max_tokens=1, scale=1.0 / (8 * spread))
        _check_attention(cache, q, [1, 1], lens, out, scale=1.0 / (8 * spread))


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_only_where_it_is_seen(dev, dim, variant):
    """A NaN in a later token's key or value does not reach earlier queries; those that see it get NaN where the plain form does."""
    import luisaml_b200 as lb
    n, length, heads, group = 60, 333, 2, 2
    for window in (0, 20):
        cache = Cache(dev, [length], length, heads, dim, 32, 16)
        bad_v, bad_k = length - 20, length - 7
        cache.v[cache.table[0, bad_v // 32].long(), 0, bad_v % 32, 5] = 0x7f
        cache.k[cache.table[0, bad_k // 32].long(), 1, bad_k % 32, 9] = 0xff
        q = torch.randn(n, heads * group, dim, device=dev).half()
        out = lb.kv_attention(q, *cache.args(), cache.table, _cu([n], dev), cache.lens, max_tokens=n, window=window, variant=variant)
        pos = torch.arange(length - n, length, device=dev)
        sees = lambda j: (j <= pos) & ((j > pos - window) if window else True)  # noqa: E731
        want = torch.zeros(n, heads * group, dim, dtype=torch.bool, device=dev)
        want[:, :group, 5] = sees(bad_v)[:, None]
        want[:, group:] = sees(bad_k)[:, None, None]
        assert torch.equal(out.isnan(), want)


def test_strides_and_streams(dev):
    """q as a slice of a fused projection, out in a wider buffer, the call on another stream than its tensors' own"""
    import luisaml_b200 as lb
    lens, new = [100, 260], [1, 5]
    cache = Cache(dev, lens, 260, 2, 64, 16, 16)
    qkv = torch.randn(6, 8 + 2 + 2, 66, device=dev).bfloat16()
    q = qkv[:, :8, 1:65]
    buf = torch.full((6, 9, 64), 5.0, device=dev, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = lb.kv_attention(q, *cache.args(), cache.table, _cu(new, dev), cache.lens, max_tokens=5, out=buf[:, :8])
    torch.cuda.current_stream().wait_stream(side)
    _check_attention(cache, q, new, lens, out)
    assert (buf[:, 8] == 5).all()


def test_repeatable_and_in_a_graph(dev):
    import luisaml_b200 as lb
    lens = [5000, 70]
    cache = Cache(dev, lens, 5000, 2, 128, 64, 64)
    q = torch.randn(2, 8, 128, device=dev).bfloat16()
    cu = _cu([1, 1], dev)
    size = lb.kv_attention_workspace_size(q, *cache.args(), cache.table, cu, cache.lens, max_tokens=1)
    ws = torch.full((size,), 0xff, dtype=torch.uint8, device=dev)  # contents on entry do not matter
    first = lb.kv_attention(q, *cache.args(), cache.table, cu, cache.lens, max_tokens=1, workspace=ws)
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lb.kv_attention(q, *cache.args(), cache.table, cu, cache.lens, max_tokens=1, workspace=ws, out=out)
        with torch.cuda.graph(graph, stream=side):
            lb.kv_attention(q, *cache.args(), cache.table, cu, cache.lens, max_tokens=1, workspace=ws, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, first)
    cache.lens.copy_(torch.tensor([3210, 11], dtype=torch.int32))  # lengths live on the device
    graph.replay()
    _check_attention(cache, q, [1, 1], [3210, 11], out)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals(dev):
    import luisaml_b200 as lb
    cache = Cache(dev, [20, 4], 64, 2, 64, 32, 16)
    cu = _cu([1, 1], dev)
    q = torch.randn(2, 4, 64, device=dev).half()
    k = torch.randn(2, 2, 64, device=dev)
    good = (*cache.args(), cache.table, cu, cache.lens)
    call = lambda **kw: lb.kv_attention(q, *good, max_tokens=1, **kw)  # noqa: E731
    for bad in ({"window": -1}, {"softcap": -1.0}, {"window": 3, "causal": False}, {"variant": 9}, {"scale": float("nan")}):
        with pytest.raises(lb.LcmlError):
            call(**bad)
    with pytest.raises(ValueError):
        lb.kv_attention(q.float(), *good)
    with pytest.raises(ValueError):
        lb.kv_attention(q[:, :, :32], *good)
    with pytest.raises(lb.LcmlError):
        lb.kv_attention(q[:, :3], *good)  # 3 query heads over 2
    with pytest.raises(ValueError):
        lb.kv_attention(q, *cache.args(), cache.table.long(), cu, cache.lens)
    with pytest.raises(ValueError):
        lb.kv_attention(q.cpu(), *good)
    with pytest.raises(ValueError):
        lb.kv_cache_write(*cache.args(), k[:, :1], k[:, :1], cache.table, cu, cache.lens)
    with pytest.raises(ValueError):
        lb.kv_cache_write(*cache.args(), k, k.half(), cache.table, cu, cache.lens)
    with pytest.raises(lb.LcmlError):  # blocks of 8 tokens
        lb.kv_cache_write(cache.k, cache.v, *(torch.zeros(cache.k.shape[0], 2, 4, device=dev) for _ in range(2)), k, k, cache.table, cu, cache.lens)
    odd = torch.zeros(2, 2, 16, 96, dtype=torch.uint8, device=dev), torch.zeros(2, 2, 1, device=dev)
    with pytest.raises(lb.LcmlError):  # head_dim 96
        lb.kv_cache_read(odd[0], odd[0], odd[1], odd[1], cache.table, cu, cache.lens, total=2)
    with pytest.raises(ValueError):
        lb.kv_cache_read(*good, total=2, dtype=torch.float64)
    x = torch.randn(4, 64, device=dev)
    with pytest.raises(ValueError):
        lb.rmsnorm_quantize(x, torch.ones(63, device=dev))
    with pytest.raises(ValueError):
        lb.rmsnorm_quantize(x.double(), torch.ones(64, device=dev))
    with pytest.raises(ValueError):
        lb.rmsnorm_quantize(x, torch.ones(64, device=dev), x.half())
    with pytest.raises(lb.LcmlError):
        lb.rmsnorm_quantize(x, torch.ones(64, device=dev), eps=-1.0)
    assert lb.lib().lcml_rmsnorm_quantize(None, None) == 1 and b"null" in lb.lib().lcml_last_error()


def test_bad_pages_are_not_followed(dev):
    """entries outside the cache and lengths past the table: reported, never dereferenced"""
    import luisaml_b200 as lb
    cache = Cache(dev, [60, 10], 64, 2, 64, 32, 16)
    before = [t.clone() for t in cache.args()]
    cu = _cu([1, 1], dev)
    table = cache.table.clone()
    table[0, 1] = -1
    table[1, 0] = cache.k.shape[0]
    k = torch.randn(2, 2, 64, device=dev)
    lb.kv_cache_write(*cache.args(), k, k, table, cu, cache.lens)
    assert _no_device_error() == 6
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(before, cache.args()))
    lb.kv_cache_read(*cache.args(), table, cu, cache.lens, total=2)
    assert _no_device_error() == 6
    q = torch.randn(2, 4, 64, device=dev).half()
    lb.kv_attention(q, *cache.args(), table, cu, cache.lens, max_tokens=1)
    assert _no_device_error() == 6
    long = torch.tensor([100000, 10], dtype=torch.int32, device=dev)
    lb.kv_attention(q, *cache.args(), cache.table, cu, long, max_tokens=1)
    assert _no_device_error() == 7
    lb.kv_cache_write(*cache.args(), k, k, cache.table, cu, long)
    assert _no_device_error() == 6


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (64, "f16")])
def test_the_choice_of_kernel(dev, dim, dtype):
    """many sequences that the automatic choice gives to the tensor-core kernel: all of them (no streaming launch), all
    but the short ones (both launches, sequences of no query among them), and one row less than either side of the threshold"""
    rows = {128: 28, 64: 40}[dim]
    held = [200 + 3 * i for i in range(40)]
    for new in ([30] * 40, [30] * 39 + [29], [30, 1, 30, 0] * 10, [rows // 4, rows // 4 - 1, 30, 30] * 10):
        _attend(dev, new, held, 2, 4, dim, 32, 16, dtype)


def test_many_sequences_of_one_token(dev):
    """more segments than CTAs, whole and cut, and more sequences than one launch plans"""
    _attend(dev, [1] * 300, [(7 * i) % 100 for i in range(300)], 2, 4, 128, 16, 16, "bf16")
    _attend(dev, [1] * 1100, [(13 * i) % 40 for i in range(1099)] + [1500], 1, 2, 64, 16, 16, "f16")
