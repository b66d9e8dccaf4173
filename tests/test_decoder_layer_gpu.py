"""The example of a decoder layer: prompts and captured steps against plain fp32 torch."""
import importlib.util
import os

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [dict(q_heads=8, kv_heads=2, head_dim=64, ffn=256, page=16), dict(q_heads=4, kv_heads=4, head_dim=128, ffn=384)])
def test_decoder_layer_example(dev, sizes):
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    prompt_error, step_error, _, _ = example.run(batch=5, prompt=150, steps=20, check=5, **sizes)
    # A path from x to the output passes three e4m3 roundings at most (norm or
    # cache, attention or FFN output, each at most 2^-4 of a value and 2^-5 in
    # the mean), so they add up to less than 3 * 2^-5 of the output.
    assert prompt_error < 3 * 2**-5 and step_error < 3 * 2**-5
