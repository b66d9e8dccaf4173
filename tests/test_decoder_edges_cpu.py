"""Refusals of the decoder-layer operators that need no GPU, beyond those of test_decoder_cpu.py."""
import ctypes

import pytest

from test_decoder_cpu import _attention, _batch, _cache, capi  # noqa: F401


@pytest.mark.parametrize("bad", [dict(out_head_stride=0), dict(out_token_stride=0), dict(out_head_stride=64), dict(out_token_stride=896),
                                 dict(out_token_stride=128, out_head_stride=128)])
def test_an_output_that_overlaps_is_refused(capi, bad):
    lib = capi.load()
    assert lib.lcml_kv_attention(ctypes.byref(_attention(capi, _cache(capi), _batch(capi), **bad)), None) == 1
    assert b"overlap" in lib.lcml_last_error()
