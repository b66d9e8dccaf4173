"""The operators of a decoder layer around the FP8 GEMMs, over the C ABI of
``include/lcml_decoder.h``: RMS norm with the residual's addition and an e4m3
output, the paged e4m3 key/value cache (quantizing write, read back) and the
attention over it; and what a step needs beside them (``include/lcml_decode_step.h``):
the plan of a ragged batch from request lengths, the norm and rotation of queries
and keys, attention with sinks, the sampling of the next token.

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
import typing

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
                              True, window, 0.0, None, None, None, variant, True, 0)


def kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, *, max_tokens=None, scale=None,
                 causal=True, window=0, softcap=0.0, out=None, lse=None, workspace=None, variant=0, sinks=0):
    """Attention of the packed queries ``q`` [tokens, q_heads, head_dim] (float16 or bfloat16)
    over the cache; returns ``out`` of q's shape and type.

    Sequence b holds ``kv_len[b]`` tokens, its queries the last of them (written before this
    call). ``max_tokens``: an upper bound of one sequence's queries, known on the host (default:
    all of q's). ``scale``: 1 / sqrt(head_dim) by default; ``window``: how many positions up to
    its own a query sees (0: all), ``sinks``: how many first positions it sees besides (the pages
    between are not looked at: their table entries may be anything); ``softcap``: scores become softcap * tanh(score / softcap).
    A query that sees nothing gets zeros. ``lse``: optional float32 [tokens, q_heads] output.
    ``workspace``: scratch of :func:`kv_attention_workspace_size` bytes (default: allocated).
    """
    return _bind.kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, max_tokens, scale,
                              causal, window, softcap, out, lse, workspace, variant, False, sinks)


class KvPlan(typing.NamedTuple):
    """What :func:`kv_plan` returns: int32 tensors on the batch's device."""
    cu_tokens: torch.Tensor   # [batch + 1]
    start: torch.Tensor       # [batch]: tokens each row holds before the step (start of kv_cache_write)
    kv_len: torch.Tensor      # [batch]: and after it (kv_len of kv_attention)
    positions: torch.Tensor   # [total]: each packed token's position, -1 past the last one
    slots: torch.Tensor       # [total]: page * page_size + slot, -1 where it has none
    free_count: torch.Tensor  # [1]: pages left on the free list


def kv_plan(new_tokens, held, block_table, free_pages, free_count, *, page_size, total, ended=None, kv_len=None, free_count_out=None):
    """Plans a step of a ragged batch on the device: row b holds ``held[b]`` tokens and brings
    ``new_tokens[b]`` more (int32 [batch]).

    Takes the pages that the new tokens need from the end of the free list (``free_pages`` int32
    [capacity], of which the first ``free_count`` [1] are free) and enters them into ``block_table``,
    in place. ``ended`` (bool [batch]): rows whose request is over; their pages go back onto the
    list first and ``new_tokens`` is the row's new request's. ``total``: length of the packed maps, at
    least the batch's new tokens. ``kv_len`` and ``free_count_out``: outputs, which may be ``held`` and
    ``free_count`` themselves, so that a captured step moves on with each replay.
    Returns a :class:`KvPlan`. Its tensors that are not given share one allocation, which lives as long as any
    of them: none may be resized (it would run into the next), and a small one that is kept for long is better
    cloned. An empty free list shows in :func:`luisaml_b200.device_error` as 8,
    lengths that do not fit as 7; what has no page gets -1 and is never followed.
    """
    return tuple.__new__(KvPlan, _bind.kv_plan(new_tokens, held, block_table, free_pages, free_count, ended, page_size, total, kv_len, free_count_out))


def qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, *, eps=1e-6, interleaved=False, q_out=None, k_out=None):
    """RMS norm of every head of ``q`` and ``k`` [tokens, heads, head_dim] (float32, float16 or bfloat16;
    tokens and heads may be strided), then their rotation by ``positions`` (int32 [tokens]; a token of
    negative position is not touched).

    ``inv_freq`` (float64 or float32 [rotary / 2]): radians per position of each pair of the first rotary
    elements, (i, i + rotary / 2) or, ``interleaved``, (2 i, 2 i + 1). ``q_weight``, ``k_weight`` [head_dim], q's type or
    float32; None: no norm. head_dim is even and at most 512. Returns (q_out, k_out), new tensors by
    default; they may be ``q`` and ``k`` themselves.
    """
    return _bind.qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, q_out, k_out)


def sample(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None, out=None, logprob=None):
    """Draws a token of every row of ``logits`` [rows, vocab] (float32, float16 or bfloat16) with the numbers
    ``uniform`` (float32 [rows], in [0, 1)); returns int32 [rows].

    Parameters are tensors of one value a row: ``temperature`` (0: the largest logit), ``top_k`` int32 (0: all),
    ``top_p`` of what top_k keeps (1: all), ``min_p`` of the largest probability (0: all). The draw is among the
    tokens that all of them keep, equal logits in the order of their indices, and takes the lowest index at
    which their probabilities, summed by rising index, pass ``uniform``. Probabilities are held in 64 bits, good
    to 1e-12 of each (where up to 256 tokens stay: or to 2^-52 of the largest). Equal calls give equal tokens; the
    same row in another batch or at another alignment is summed in another order and may give another token where
    ``uniform`` meets a border to the rounding of a 64-bit sum. ``logprob``: optional float32 [rows]
    output, the log of the token's probability among the kept ones. A row of -infinity alone gives -1.
    """
    return _bind.sample(logits, uniform, temperature, top_k, top_p, min_p, out, logprob)
