"""The operators of a decoder layer around the FP8 GEMMs, over the C ABI of
``include/lcml_decoder.h``: RMS norm with the residual's addition and an e4m3
output, the paged e4m3 key/value cache (quantizing write, read back) and the
attention over it.

All of them take CUDA tensors, enqueue on torch's current stream of the
tensors' device and neither synchronise nor read lengths back: the lengths of a
ragged batch stay on the device. Codes are uint8 e4m3 as everywhere in this
package. Refused arguments raise ValueError or LcmlError; a page or length out
of range is never followed and shows in :func:`luisaml_b200.device_error`.
Inference only: in grad mode an input that requires a gradient is refused.

A cache is four tensors that the caller keeps::

    k_cache, v_cache   uint8   [pages, kv_heads, page_size, head_dim]
    k_scale, v_scale   float32 [pages, kv_heads, page_size // scale_block]

(head_dim 64, 128 or 256; scale_block a multiple of 16) and a ragged batch is
three int32 tensors: ``block_table`` [batch, columns] (position t of sequence b
lives in slot t % page_size of page block_table[b, t // page_size]),
``cu_tokens`` [batch + 1] (sequence b owns the packed tokens cu_tokens[b] ..
cu_tokens[b + 1] - 1) and a length per sequence.
"""
from __future__ import annotations

import os

import torch

from . import _capi

_capi.load()  # the binding links liblcml_fp8.so
try:
    from . import _decoder_bind as _bind
except ImportError as e:
    raise ImportError(f"{os.path.join(_capi.HERE, '_decoder_bind.so')} not built for this interpreter and torch: run "
                      f"`python -c 'import __graft_entry__ as g; g.build()'` or `make -C luisaml_b200` ({e})") from e


def rmsnorm_quantize(x, weight, residual=None, *, eps=1e-6, scale=None, out=None, scale_out=None, h_out=None):
    """RMS norm of ``x`` (+ ``residual``) with e4m3 codes out: the A operand of :func:`luisaml_b200.gemm`.

    x, residual: [rows, cols] float32, float16 or bfloat16 (rows may be strided);
    weight: [cols], x's type or float32. ``scale``: a calibrated float32 [1]; without
    it each row gets max|y| / 448. Returns (codes uint8 [rows, cols], scales, h):
    scales is float32 [rows] (or ``scale``), h is x + residual in x's type (None
    without a residual and ``h_out``; ``h_out`` may be x or residual itself).
    """
    return _bind.rmsnorm_quantize(x, weight, residual, eps, scale, out, scale_out, h_out)


def kv_cache_write(k_cache, v_cache, k_scale, v_scale, k, v, block_table, cu_tokens, start):
    """Quantizes the packed new tokens ``k``, ``v`` [tokens, kv_heads, head_dim] (float32,
    float16 or bfloat16; tokens and heads may be strided) into the cache, in place.

    Sequence b's tokens follow the ``start[b]`` it already holds. A block's scale is
    max|x| / 448 over its tokens; when a new token raises it, the block's earlier codes are
    re-encoded. Two sequences of one call must not write the same page.
    """
    _bind.kv_cache_write(k_cache, v_cache, k_scale, v_scale, k, v, block_table, cu_tokens, start)


def kv_cache_read(k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, start, *, total, dtype=torch.bfloat16):
    """Reads tokens back as (k, v) [total, kv_heads, head_dim] of ``dtype``: packed token
    cu_tokens[b] + i is position start[b] + i of sequence b. ``total`` is cu_tokens[batch]."""
    return _bind.kv_cache_read(k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, start, total, dtype)


def kv_attention_workspace_size(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, *,
                                max_tokens=None, window=0, variant=0):
    """Bytes of scratch the same call of :func:`kv_attention` needs (0: none)."""
    return _bind.kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, max_tokens, None,
                              True, window, 0.0, None, None, None, variant, True)


def kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, *, max_tokens=None, scale=None,
                 causal=True, window=0, softcap=0.0, out=None, lse=None, workspace=None, variant=0):
    """Attention of the packed queries ``q`` [tokens, q_heads, head_dim] (float16 or bfloat16)
    over the cache; returns ``out`` of q's shape and type.

    Sequence b holds ``kv_len[b]`` tokens, its queries the last of them (written before this
    call). ``max_tokens``: an upper bound of one sequence's queries, known on the host (default:
    all of q's). ``scale``: 1 / sqrt(head_dim) by default; ``window``: how many positions up to
    its own a query sees (0: all); ``softcap``: scores become softcap * tanh(score / softcap).
    A query that sees nothing gets zeros. ``lse``: optional float32 [tokens, q_heads] output.
    ``workspace``: scratch of :func:`kv_attention_workspace_size` bytes (default: allocated).
    """
    return _bind.kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, max_tokens, scale,
                              causal, window, softcap, out, lse, workspace, variant, False)
