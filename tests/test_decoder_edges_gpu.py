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
