"""The example of a decoder that keeps its own batch compares the tokens of every step."""
import os
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu
SIZES = dict(batch=3, prompt=50, steps=12, request=7, vocab=1000, layers=1, q_heads=4, kv_heads=2, ffn=256, page=16, window=24, sinks=2)


@pytest.mark.parametrize("wrong", [None, 0, 5, 11])
def test_example_compares_every_step(dev, monkeypatch, wrong):
    """one of the single steps shows another token, its successor goes on with the right one"""
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_loop
    step, seen, right = decode_loop.Decoder.step, [], {}

    def planted(self, tokens, new, ended, max_tokens, draw):
        got = step(self, right.get(id(tokens), tokens), new, ended, max_tokens, draw)
        if ended is None or torch.cuda.is_current_stream_capturing():  # prompts, and the captured step
            return got
        seen.append(got)
        if len(seen) - 1 != wrong:
            return got
        other = got.clone()
        other[1] += 1
        right[id(other)] = got
        return other

    monkeypatch.setattr(decode_loop.Decoder, "step", planted)
    same, _, _, _ = decode_loop.run(**SIZES)
    assert len(seen) == SIZES["steps"] and same == (wrong is None)


def test_example_draws_by_its_numbers(dev, monkeypatch):
    """each row's tokens change from step to step: the weights are not such that a token is followed by itself"""
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_loop
    step, seen = decode_loop.Decoder.step, []

    def kept(self, tokens, new, ended, max_tokens, draw):
        got = step(self, tokens, new, ended, max_tokens, draw)
        if not torch.cuda.is_current_stream_capturing():
            seen.append(got)
        return got

    monkeypatch.setattr(decode_loop.Decoder, "step", kept)
    assert decode_loop.run(**SIZES)[0]
    drawn = torch.stack(seen[:SIZES["steps"] + 1])
    assert min(drawn[:, b].unique().numel() for b in range(SIZES["batch"])) > SIZES["steps"] // 2
