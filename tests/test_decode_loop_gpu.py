"""The example of a decoder that keeps its own batch: its captured steps draw what single steps draw, and no page is lost."""
import os
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_example(dev):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_loop
    import luisaml_b200 as lb
    same, _, _, pages = decode_loop.run(batch=5, prompt=150, steps=30, request=20, vocab=2000, layers=2, q_heads=8, kv_heads=2, ffn=512, page=16, window=40, sinks=3)
    assert same and lb.device_error() == 0
    # rows whose request ended hold what they have drawn since, the others their prompt and 30 tokens
    ends = [max(i for i in range(-1, 30) if i < 0 or (i + 5 * b) % 20 == 19) for b in range(5)]
    held = [30 - e if e >= 0 else 150 - 11 * b + 30 for b, e in enumerate(ends)]
    assert pages == sum(-(-h // 16) for h in held)
