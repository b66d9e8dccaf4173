"""Refusals of the decoder-layer operators that need no GPU, beyond those of test_decoder_cpu.py."""
import ctypes
import subprocess
import sys

import pytest

from conftest import ROOT
from test_decoder_cpu import _attention, _batch, _cache, capi  # noqa: F401


@pytest.mark.parametrize("bad", [dict(out_head_stride=0), dict(out_token_stride=0), dict(out_head_stride=64), dict(out_token_stride=896),
                                 dict(out_token_stride=128, out_head_stride=128)])
def test_an_output_that_overlaps_is_refused(capi, bad):
    lib = capi.load()
    assert lib.lcml_kv_attention(ctypes.byref(_attention(capi, _cache(capi), _batch(capi), **bad)), None) == 1
    assert b"overlap" in lib.lcml_last_error()


def test_inputs_that_require_a_gradient_are_refused(capi):
    import torch
    import luisaml_b200 as lb
    u8, f, i32 = torch.zeros(2, 1, 16, 64, dtype=torch.uint8), torch.zeros(2, 1, 1), torch.zeros(1, 1, dtype=torch.int32)
    cache, batch = (u8, u8.clone(), f, f.clone()), (i32, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    x, w, k = torch.zeros(2, 64), torch.ones(64), torch.zeros(1, 1, 64)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda: lb.rmsnorm_quantize(grad(x), w), lambda: lb.rmsnorm_quantize(x, grad(w)), lambda: lb.rmsnorm_quantize(x, w, grad(x)),
             lambda: lb.kv_cache_write(*cache, grad(k), k, *batch), lambda: lb.kv_cache_write(*cache, k, grad(k), *batch),
             lambda: lb.kv_attention(grad(k.half()), *cache, *batch), lambda: lb.kv_cache_read(u8, u8, grad(f), f, *batch, total=1)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # the next check: these are host tensors
            call()


def test_star_import_without_torch():
    """the names are there, and the call says what is missing"""
    code = ("import sys; sys.modules['torch'] = None\n"
            "from luisaml_b200 import *\n"
            "assert quantize and check\n"
            "try:\n    kv_attention(None)\nexcept ImportError as e:\n    assert 'kv_attention' in str(e) and 'torch' in str(e); print('said so')")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert out.returncode == 0 and "said so" in out.stdout, out.stderr
