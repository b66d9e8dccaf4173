"""The operators of a decoder layer around the FP8 GEMMs, over the C ABI of
``include/lcml_decoder.h``: RMS norm with the residual's addition and an e4m3
output, the paged e4m3 key/value cache (quantizing write, read back) and the
attention over it.

All of them take CUDA tensors, enqueue on torch's current stream and neither
synchronise nor read lengths back: the lengths of a ragged batch stay on the
device. Codes are uint8 e4m3 as everywhere in this package.

A cache is four tensors that the caller keeps::

    k_cache, v_cache   uint8   [pages, kv_heads, page_size, head_dim]
    k_scale, v_scale   float32 [pages, kv_heads, page_size // scale_block]

and a ragged batch is three int32 tensors: ``block_table`` [batch, columns]
(position t of sequence b lives in slot t % page_size of page
block_table[b, t // page_size]), ``cu_tokens`` [batch + 1] (sequence b owns the
packed tokens cu_tokens[b] .. cu_tokens[b + 1] - 1) and a length per sequence.
"""
from __future__ import annotations

import ctypes

import torch

from . import _capi
from ._capi import DTYPE_BFLOAT16, DTYPE_FLOAT, DTYPE_FLOAT16, check

_DTYPES = {torch.float32: DTYPE_FLOAT, torch.float16: DTYPE_FLOAT16, torch.bfloat16: DTYPE_BFLOAT16}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _dtype(t, name, allowed):
    if t.dtype not in allowed:
        raise ValueError(f"{name}: unsupported dtype {t.dtype}")
    return _DTYPES[t.dtype]


def _same_device(first, *ts):
    dev = first.device
    _need(dev.type == "cuda", "luisaml_b200 ops take CUDA tensors")
    for t in ts:
        _need(t is None or t.device == dev, "tensors on different devices")


def rmsnorm_quantize(x, weight, residual=None, *, eps=1e-6, scale=None, out=None, scale_out=None, h_out=None):
    """RMS norm of ``x`` (+ ``residual``) with e4m3 codes out: the A operand of :func:`gemm`.

    x, residual: [rows, cols] float32, float16 or bfloat16 (rows may be strided);
    weight: [cols], x's type or float32. ``scale``: a calibrated float32 [1]; without
    it each row gets max|y| / 448. Returns (codes uint8 [rows, cols], scales, h):
    scales is float32 [rows] (or ``scale``), h is x + residual in x's type (None
    without a residual; ``h_out`` may be x or residual itself).
    """
    _need(x.dim() == 2, "rmsnorm_quantize: x is [rows, cols]")
    rows, cols = x.shape
    _same_device(x, weight, residual, scale, out, scale_out, h_out)
    xd = _dtype(x, "x", _DTYPES)
    wd = _dtype(weight, "weight", (x.dtype, torch.float32))
    _need(weight.shape == (cols,) and weight.is_contiguous(), "rmsnorm_quantize: weight is [cols], contiguous")
    if residual is not None and h_out is None:
        h_out = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    for name, t in (("x", x), ("residual", residual), ("h_out", h_out)):
        _need(t is None or (t.shape == x.shape and t.dtype == x.dtype and (t.stride(1) == 1 or cols <= 1)
                            and (rows <= 1 or t.stride(0) >= cols)),
              f"rmsnorm_quantize: {name} has x's shape and type, with contiguous rows that do not overlap")
    if out is None:
        out = torch.empty((rows, cols), dtype=torch.uint8, device=x.device)
    _need(out.shape == x.shape and out.dtype == torch.uint8 and out.is_contiguous(),
          "rmsnorm_quantize: out is uint8 [rows, cols], contiguous")
    if scale is None:
        if scale_out is None:
            scale_out = torch.empty(rows, dtype=torch.float32, device=x.device)
        _need(scale_out.shape == (rows,) and scale_out.dtype == torch.float32 and scale_out.is_contiguous(),
              "rmsnorm_quantize: scale_out is float32 [rows]")
    else:
        _need(scale_out is None, "rmsnorm_quantize: give scale or scale_out, not both")
        _need(scale.numel() == 1 and scale.dtype == torch.float32, "rmsnorm_quantize: scale is one float32")
    d = _capi.RmsnormDesc(rows, cols, x.data_ptr(), max(x.stride(0), cols), _ptr(residual),
                          max(residual.stride(0), cols) if residual is not None else 0, _ptr(h_out),
                          max(h_out.stride(0), cols) if h_out is not None else 0, weight.data_ptr(), xd, wd, eps,
                          _ptr(scale), _ptr(scale_out), out.data_ptr())
    check(_capi.load().lcml_rmsnorm_quantize(ctypes.byref(d), _stream()))
    return out, scale if scale is not None else scale_out, h_out


def _cache(k_cache, v_cache, k_scale, v_scale):
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype == torch.uint8
          and k_cache.is_contiguous() and v_cache.is_contiguous(),
          "k_cache and v_cache are uint8 [pages, kv_heads, page_size, head_dim], contiguous")
    pages, heads, page, dim = k_cache.shape
    blocks = k_scale.shape[-1]
    _need(k_scale.shape == v_scale.shape == (pages, heads, blocks) and k_scale.dtype == v_scale.dtype == torch.float32
          and k_scale.is_contiguous() and v_scale.is_contiguous() and blocks > 0 and page % blocks == 0,
          "k_scale and v_scale are float32 [pages, kv_heads, page_size // scale_block], contiguous")
    return _capi.KvCache(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, page,
                         heads, dim, page // blocks)


def _batch(block_table, cu_tokens, lengths, total):
    n = lengths.shape[0]
    i32 = torch.int32
    _need(block_table.dtype == cu_tokens.dtype == lengths.dtype == i32 and block_table.dim() == 2
          and block_table.shape[0] == n and cu_tokens.shape == (n + 1,) and lengths.dim() == 1,
          "block_table [batch, columns], cu_tokens [batch + 1] and the lengths [batch] are int32")
    cols = block_table.shape[1]
    _need((cols <= 1 or block_table.stride(1) == 1) and cu_tokens.is_contiguous() and lengths.is_contiguous(),
          "block_table's rows, cu_tokens and the lengths are contiguous")
    return _capi.KvBatch(n, cols, block_table.data_ptr(), max(block_table.stride(0), cols), cu_tokens.data_ptr(),
                         lengths.data_ptr(), total)


def kv_cache_write(k_cache, v_cache, k_scale, v_scale, k, v, block_table, cu_tokens, start):
    """Quantizes the packed new tokens ``k``, ``v`` [tokens, kv_heads, head_dim] (float32,
    float16 or bfloat16; tokens and heads may be strided) into the cache, in place.

    Sequence b's tokens follow the ``start[b]`` it already holds. A block's scale is
    max|x| / 448 over its tokens; when a new token raises it, the block's earlier codes are
    re-encoded. Two sequences of one call must not write the same page.
    """
    _same_device(k_cache, v_cache, k_scale, v_scale, k, v, block_table, cu_tokens, start)
    c = _cache(k_cache, v_cache, k_scale, v_scale)
    dt = _dtype(k, "k", _DTYPES)
    _need(k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype and k.shape[1] == c.kv_heads
          and k.shape[2] == c.head_dim and k.stride(2) == v.stride(2) == 1,
          "k and v are [tokens, kv_heads, head_dim] of one type, with contiguous rows")
    b = _batch(block_table, cu_tokens, start, k.shape[0])
    check(_capi.load().lcml_kv_cache_write(ctypes.byref(c), ctypes.byref(b), k.data_ptr(), k.stride(0), k.stride(1),
                                           v.data_ptr(), v.stride(0), v.stride(1), dt, _stream()))


def kv_cache_read(k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, start, *, total, dtype=torch.bfloat16):
    """Reads tokens back as (k, v) [total, kv_heads, head_dim] of ``dtype``: packed token
    cu_tokens[b] + i is position start[b] + i of sequence b. ``total`` is cu_tokens[batch]."""
    _same_device(k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, start)
    c = _cache(k_cache, v_cache, k_scale, v_scale)
    _need(dtype in _DTYPES, f"kv_cache_read: unsupported dtype {dtype}")
    b = _batch(block_table, cu_tokens, start, total)
    k = torch.empty((total, c.kv_heads, c.head_dim), dtype=dtype, device=k_cache.device)
    v = torch.empty_like(k)
    check(_capi.load().lcml_kv_cache_read(ctypes.byref(c), ctypes.byref(b), k.data_ptr(), v.data_ptr(),
                                          _DTYPES[dtype], _stream()))
    return k, v


def _attention_desc(q, cache, batch, max_tokens, scale, causal, window, softcap, variant):
    dt = _dtype(q, "q", (torch.float16, torch.bfloat16))
    _need(q.dim() == 3 and q.shape[2] == cache.head_dim and q.stride(2) == 1,
          "kv_attention: q is [tokens, q_heads, head_dim] with contiguous rows")
    return _capi.KvAttentionDesc(ctypes.pointer(cache), ctypes.pointer(batch), q.data_ptr(), q.stride(0), q.stride(1),
                                 None, 0, 0, None, q.shape[1], dt, q.shape[0] if max_tokens is None else max_tokens,
                                 cache.head_dim ** -0.5 if scale is None else scale, softcap, window, int(causal), None,
                                 variant)


def kv_attention_workspace_size(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, *,
                                max_tokens=None, window=0, variant=0):
    """Bytes of scratch the same call of :func:`kv_attention` needs (0: none)."""
    cache, batch = _cache(k_cache, v_cache, k_scale, v_scale), _batch(block_table, cu_tokens, kv_len, q.shape[0])
    d = _attention_desc(q, cache, batch, max_tokens, None, True, window, 0.0, variant)
    n = _capi.load().lcml_kv_attention_workspace_size(ctypes.byref(d))
    check(1 if n < 0 else 0)
    return n


def kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, *, max_tokens=None, scale=None,
                 causal=True, window=0, softcap=0.0, out=None, lse=None, workspace=None, variant=0):
    """Attention of the packed queries ``q`` [tokens, q_heads, head_dim] (float16 or bfloat16)
    over the cache; returns ``out`` of q's shape and type.

    Sequence b holds ``kv_len[b]`` tokens, its queries the last of them (written before this
    call). ``max_tokens``: an upper bound of one sequence's queries, known on the host (default:
    all of q's). ``scale``: 1 / sqrt(head_dim) by default; ``window``: how many positions up to
    its own a query sees (0: all); ``softcap``: scores become softcap * tanh(score / softcap).
    A query that sees nothing gets zeros. ``lse``: optional float32 [tokens, q_heads] output.
    """
    _same_device(k_cache, v_cache, k_scale, v_scale, q, block_table, cu_tokens, kv_len, out, lse, workspace)
    cache, batch = _cache(k_cache, v_cache, k_scale, v_scale), _batch(block_table, cu_tokens, kv_len, q.shape[0])
    d = _attention_desc(q, cache, batch, max_tokens, scale, causal, window, softcap, variant)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.stride(2) == 1,
              "kv_attention: out has q's shape and type, with contiguous rows")
    d.out, d.out_token_stride, d.out_head_stride = out.data_ptr(), out.stride(0), out.stride(1)
    if lse is not None:
        _need(lse.shape == q.shape[:2] and lse.dtype == torch.float32 and lse.is_contiguous(),
              "kv_attention: lse is float32 [tokens, q_heads]")
        d.lse = lse.data_ptr()
    lib = _capi.load()
    need = lib.lcml_kv_attention_workspace_size(ctypes.byref(d))
    if need > 0:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        _need(workspace.numel() * workspace.element_size() >= need, f"kv_attention: workspace of {need} bytes needed")
        d.workspace = workspace.data_ptr()
    check(lib.lcml_kv_attention(ctypes.byref(d), _stream()))
    return out
