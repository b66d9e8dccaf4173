"""The decode step's operators without a GPU: prototypes, and refusals before any work is enqueued."""
import ctypes
import os

import pytest

from conftest import ROOT
from test_capi_symbols import declared
from test_decoder_cpu import _attention, _batch, _cache, capi  # noqa: F401


def test_prototypes_cover_header(capi):
    names = declared(os.path.join(ROOT, "include", "lcml_decode_step.h"))
    assert len(names) == 4 and not [n for n in names if n not in capi.PROTOTYPES]


def _refused(capi, name, desc, *more):
    assert getattr(capi.load(), name)(ctypes.byref(desc), *more, None) == 1
    assert capi.load().lcml_last_error()


@pytest.mark.parametrize("bad", [dict(batch=-1), dict(batch=16385), dict(page_size=0), dict(page_size=65537), dict(table_cols=-1), dict(table_stride=3), dict(total_tokens=-1),
                                 dict(total_tokens=1 << 31), dict(free_capacity=-1), dict(block_table=None), dict(new_tokens=None), dict(held=None), dict(free_pages=None),
                                 dict(free_count=None), dict(cu_tokens=None), dict(start=None), dict(kv_len=None), dict(positions=None), dict(slots=None),
                                 dict(free_count_out=None), dict(held=(3 << 20) + 2), dict(batch=16384, table_cols=1 << 20, table_stride=1 << 20)])
def test_a_bad_plan_is_refused(capi, bad):
    f = dict(batch=2, page_size=16, table_cols=4, table_stride=4, block_table=1 << 20, new_tokens=2 << 20, held=3 << 20, free_pages=4 << 20, free_capacity=9,
             free_count=5 << 20, total_tokens=2, cu_tokens=6 << 20, start=7 << 20, kv_len=8 << 20, positions=9 << 20, slots=10 << 20, free_count_out=11 << 20)
    _refused(capi, "lcml_kv_plan", capi.KvPlanDesc(**{**f, **bad}))


def _rope(capi, **kw):
    f = dict(tokens=2, q_heads=4, k_heads=2, head_dim=64, rotary=64, dtype=capi.DTYPE_BFLOAT16, q=1 << 20, k=2 << 20, q_token_stride=256, q_head_stride=64,
             k_token_stride=128, k_head_stride=64, q_out=3 << 20, k_out=4 << 20, q_out_token_stride=256, q_out_head_stride=64, k_out_token_stride=128, k_out_head_stride=64,
             q_weight=5 << 20, k_weight=6 << 20, weight_dtype=capi.DTYPE_FLOAT, eps=1e-6, positions=7 << 20, inv_freq=8 << 20, inv_freq_dtype=11)
    return capi.QkNormRopeDesc(**{**f, **kw})


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(q_heads=-1), dict(head_dim=0), dict(head_dim=65), dict(head_dim=514), dict(rotary=63), dict(rotary=66), dict(rotary=-2),
                                 dict(dtype=17), dict(weight_dtype=10), dict(inv_freq_dtype=16), dict(eps=-1.0), dict(eps=float("nan")), dict(q=None), dict(k_out=None),
                                 dict(positions=None), dict(inv_freq=None), dict(q=(1 << 20) + 1), dict(inv_freq=(8 << 20) + 4), dict(k_head_stride=-1),
                                 dict(q_out_head_stride=0), dict(q_out_token_stride=0), dict(k_out_head_stride=32), dict(q_out_token_stride=192)])
def test_bad_rotation_arguments_are_refused(capi, bad):
    _refused(capi, "lcml_qk_norm_rope", _rope(capi, **bad))


def test_nothing_to_rotate(capi):
    assert capi.load().lcml_qk_norm_rope(ctypes.byref(_rope(capi, tokens=0, q=None)), None) == 0
    assert capi.load().lcml_qk_norm_rope(ctypes.byref(_rope(capi, q_heads=0, k_heads=0)), None) == 0


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(vocab=-1), dict(vocab=0), dict(vocab=0x7fffffff), dict(dtype=17), dict(logits=None), dict(uniform=None), dict(tokens=None),
                                 dict(ld=99), dict(logits=(1 << 20) + 2), dict(top_k=(4 << 20) + 1), dict(logprob=(8 << 20) + 3)])
def test_bad_sampling_arguments_are_refused(capi, bad):
    f = dict(rows=2, vocab=100, logits=1 << 20, ld=100, dtype=capi.DTYPE_FLOAT, uniform=2 << 20, temperature=3 << 20, top_k=4 << 20, top_p=5 << 20, min_p=6 << 20,
             tokens=7 << 20, logprob=8 << 20)
    _refused(capi, "lcml_sample", capi.SampleDesc(**{**f, **bad}))


def test_no_rows_to_sample(capi):
    assert capi.load().lcml_sample(ctypes.byref(capi.SampleDesc(rows=0, vocab=0, dtype=capi.DTYPE_FLOAT)), None) == 0


def test_bad_sinks_are_refused(capi):
    _refused(capi, "lcml_kv_attention_sinks", _attention(capi, _cache(capi), _batch(capi), window=8), -1)
    _refused(capi, "lcml_kv_attention_sinks", _attention(capi, _cache(capi), _batch(capi), window=-8), 4)
    _refused(capi, "lcml_kv_attention_sinks", _attention(capi, _cache(capi), _batch(capi), window=8, causal=0), 4)


def test_host_tensors_and_gradients_are_refused(capi):
    import torch
    import luisaml_b200 as lb
    i32 = torch.zeros(2, dtype=torch.int32)
    q, f, u = torch.zeros(2, 1, 64), torch.ones(32), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA"):
        lb.kv_plan(i32, i32, torch.zeros(2, 1, dtype=torch.int32), i32, i32[:1], page_size=16, total=2)
    for call in (lambda x: lb.qk_norm_rope(x, q, i32, f), lambda x: lb.qk_norm_rope(q, x, i32, f), lambda x: lb.qk_norm_rope(q, q, i32, f, x[0, 0]),
                 lambda x: lb.sample(x[:, 0], u), lambda x: lb.sample(q[:, 0], u, temperature=x[:, 0, 0])):
        with pytest.raises(ValueError, match="gradient"):
            call(q.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call(q.clone().requires_grad_())
