"""The decoder operators' C ABI without a GPU: prototypes, and refusals before any work is enqueued."""
import ctypes
import os

import pytest

from conftest import ROOT
from test_capi_symbols import declared


@pytest.fixture(scope="module")
def capi():
    from luisaml_b200 import _capi
    _capi.load()
    return _capi


def test_prototypes_cover_header(capi):
    names = declared(os.path.join(ROOT, "include", "lcml_decoder.h"))
    assert len(names) == 5 and not [n for n in names if n not in capi.PROTOTYPES]


def _cache(capi, **kw):
    f = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, num_pages=8, page_size=64, kv_heads=2, head_dim=128, scale_block=64)
    return capi.KvCache(**{**f, **kw})


def _batch(capi, **kw):
    f = dict(batch=2, table_cols=4, block_table=5 << 20, table_stride=4, cu_tokens=6 << 20, lengths=7 << 20, total_tokens=2)
    return capi.KvBatch(**{**f, **kw})


def _attention(capi, cache, batch, **kw):
    f = dict(q=8 << 20, q_token_stride=1024, q_head_stride=128, out=9 << 20, out_token_stride=1024, out_head_stride=128, q_heads=8,
             dtype=capi.DTYPE_BFLOAT16, max_tokens=1, softmax_scale=0.1, causal=1, workspace=10 << 20)
    d = capi.KvAttentionDesc(cache=ctypes.pointer(cache), batch=ctypes.pointer(batch), **{**f, **kw})
    d._refs = (cache, batch)
    return d


@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(scale_block=24), dict(scale_block=48), dict(kv_heads=0), dict(page_size=0), dict(k=None),
                                 dict(v=(2 << 20) + 8), dict(num_pages=-1)])
def test_a_bad_cache_is_refused(capi, bad):
    lib = capi.load()
    c, b = _cache(capi, **bad), _batch(capi)
    assert lib.lcml_kv_cache_read(ctypes.byref(c), ctypes.byref(b), 8 << 20, 9 << 20, capi.DTYPE_BFLOAT16, None) == 1
    assert lib.lcml_last_error()
    assert lib.lcml_kv_attention(ctypes.byref(_attention(capi, c, b)), None) == 1
    assert lib.lcml_kv_attention_workspace_size(ctypes.byref(_attention(capi, c, b))) == -1


@pytest.mark.parametrize("bad", [dict(q_heads=7), dict(q_heads=0), dict(dtype=99), dict(softcap=-1.0), dict(window=-1), dict(q=None), dict(out=None),
                                 dict(q_token_stride=-1), dict(variant=3), dict(q=(8 << 20) + 1), dict(softmax_scale=float("nan"))])
def test_bad_attention_arguments_are_refused(capi, bad):
    lib = capi.load()
    assert lib.lcml_kv_attention(ctypes.byref(_attention(capi, _cache(capi), _batch(capi), **bad)), None) == 1
    assert lib.lcml_last_error()


def test_empty_batches_do_nothing(capi):
    lib = capi.load()
    c, b = _cache(capi), _batch(capi, batch=0, total_tokens=0)
    assert lib.lcml_kv_cache_read(ctypes.byref(c), ctypes.byref(b), 8 << 20, 9 << 20, capi.DTYPE_BFLOAT16, None) == 0
    assert lib.lcml_kv_attention(ctypes.byref(_attention(capi, c, b)), None) == 0


@pytest.mark.parametrize("bad", [dict(x=None), dict(weight=None), dict(q=None), dict(cols=0), dict(rows=-1), dict(x_dtype=99), dict(ldx=10),
                                 dict(scale_out=None), dict(scale=5 << 20)])
def test_bad_norm_arguments_are_refused(capi, bad):
    lib = capi.load()
    f = dict(rows=2, cols=64, x=1 << 20, ldx=64, weight=2 << 20, x_dtype=capi.DTYPE_FLOAT, weight_dtype=capi.DTYPE_FLOAT, eps=1e-6,
             scale_out=3 << 20, q=4 << 20)
    d = capi.RmsnormDesc(**{**f, **bad})
    assert lib.lcml_rmsnorm_quantize(ctypes.byref(d), None) == 1
    assert lib.lcml_last_error()


def test_host_tensors_are_refused(capi):
    import torch
    import luisaml_b200 as lb
    with pytest.raises(ValueError):
        lb.rmsnorm_quantize(torch.zeros(2, 64), torch.ones(64))
