"""Edges of the decode step's operators (include/lcml_decode_step.h): temperatures
small against the spacing of the logits, and calls at the ends of the documented ranges."""
import math

import numpy as np
import pytest
import torch

from test_decode_step_gpu import _all, _check_plan, _check_sample, _error_word_stays_clear, _kept, _no_device_error, _rows  # noqa: F401

pytestmark = pytest.mark.gpu


def _expected(x, t, u, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of one row, weights below 2^-1000 taken as 0"""
    (kept,), w = _kept(x, t, top_k, top_p, min_p, (0.0,))
    w = np.where(w < 2.0 ** -1000, 0.0, w)[kept]
    c = np.cumsum(w)
    i = int((c <= u * c[-1]).sum())
    return int(kept[i]), math.log(w[i] / c[-1])


@pytest.mark.parametrize("setting", [{}, {"top_k": 2}, {"top_k": 600}, {"top_p": 0.9}, {"min_p": 0.1}])
@pytest.mark.parametrize("vocab,at", [(3001, (5, 9)), (3001, (9, 5)), (3001, (5, 2900)), (3001, (2900, 5)), (50001, (7, 8)), (50001, (40000, 7))])
@pytest.mark.parametrize("top", [20.0, 1000.0, 10000.0, 1e9])
def test_sample_logits_a_few_floats_apart(dev, top, vocab, at, setting):
    """The two largest logits lie 1 to 40 floats apart, the temperature is 1/1500 to 1/20 of a
    float's spacing there: the second one's weight is 0 or next to it, never negative."""
    import luisaml_b200 as lb
    step = float(np.spacing(np.float32(top)))
    rows = [(n, np.float32(step / f), u) for n in (1, 2, 3, 7, 23, 40) for f in (1500, 1000, 800, 650, 347, 100, 20) for u in (0.0, 0.25, 1.0 - 2.0 ** -24)]
    x = torch.zeros(len(rows), vocab)
    x[:, at[0]] = top
    x[:, at[1]] = torch.tensor([top - n * step for n, _, _ in rows])
    t, u = (torch.tensor([float(r[i]) for r in rows], device=dev) for i in (1, 2))
    tokens, logprob = torch.full((len(rows),), -7, dtype=torch.int32, device=dev), torch.full((len(rows),), 7.0, device=dev)
    per_row = {k: _all(dev, len(rows), v, torch.int32 if k == "top_k" else torch.float32) for k, v in setting.items()}
    lb.sample(x.to(dev), u, temperature=t, out=tokens, logprob=logprob, **per_row)
    for r, (n, temperature, number) in enumerate(rows):
        token, want = _expected(x[r].double().numpy(), float(temperature), number, **{k: float(np.float32(v)) if k != "top_k" else v for k, v in setting.items()})
        assert tokens[r] == token, (n, temperature, number)
        # a weight's error and the sum's, and half a step of the output
        assert abs(float(logprob[r]) - want) <= 2.0 ** -24 * abs(want) + 1e-11, (n, temperature, number)


@pytest.mark.parametrize("setting", [{}, {"top_k": 30}, {"top_p": 0.7}, {"min_p": 1e-3}])
def test_sample_many_logits_a_few_floats_apart(dev, setting):
    """40 neighbouring floats in rows of their own order"""
    import luisaml_b200 as lb
    step, rng = float(np.spacing(np.float32(1000.0))), np.random.default_rng(0)
    rows = [(np.float32(step / f), u) for f in (1500, 800, 300, 30) for u in (0.0, 0.5, 1.0 - 2.0 ** -24)]
    x = np.zeros((len(rows), 9001), dtype=np.float32)
    for row in x:
        row[rng.choice(9001, 40, replace=False)] = 1000.0 - step * np.arange(40)
    t, u = (torch.tensor([float(r[i]) for r in rows], device=dev) for i in (0, 1))
    tokens = torch.full((len(rows),), -7, dtype=torch.int32, device=dev)
    per_row = {k: _all(dev, len(rows), v, torch.int32 if k == "top_k" else torch.float32) for k, v in setting.items()}
    lb.sample(torch.from_numpy(x).to(dev), u, temperature=t, out=tokens, **per_row)
    for r, (temperature, number) in enumerate(rows):
        want = _expected(x[r].astype(np.float64), float(temperature), number, **{k: float(np.float32(v)) if k != "top_k" else v for k, v in setting.items()})
        assert tokens[r] == want[0], (temperature, number)


def test_sample_weights_to_twelve_digits(dev):
    """Two tokens and a number that lies 1.2e-12 to 5e-12 of the first one's weight beside the border
    between them: the first one's weight decides on which side, to 1e-12."""
    import luisaml_b200 as lb
    x = np.arange(np.float32(0.25).view(np.uint32), np.float32(1.0).view(np.uint32), dtype=np.uint32).view(np.float32)  # all floats of [0.25, 1)
    w = np.exp(-x.astype(np.float64))
    u = (w / (1 + w)).astype(np.float32)
    off = 1 - u.astype(np.float64) / (1 - u.astype(np.float64)) / w  # of w, above the border
    near = np.nonzero((np.abs(off) > 1.2e-12) & (np.abs(off) < 5e-12))[0]
    assert len(near) > 500
    logits = torch.zeros(len(near), 2, device=dev)
    logits[:, 0] = torch.from_numpy(-x[near]).to(dev)
    got = lb.sample(logits, torch.from_numpy(u[near]).to(dev))
    assert torch.equal(got.cpu(), torch.from_numpy((off[near] < 0).astype(np.int32)))


@pytest.mark.parametrize("dtype,least,most,step", [("f32", 39001, 45001, 500), ("bf16", 78001, 90001, 1000)])
def test_sample_rows_as_long_as_shared_memory(dev, dtype, least, most, step):
    """A row a CTA, a little shorter and a little longer than what it holds: the draws of the same rows by
    several CTAs each, which are checked. No number lies within a rounding of a 64-bit sum of a border."""
    import luisaml_b200 as lb
    for vocab in range(least, most, step):
        x, u = _rows(dev, 3, vocab, dtype)
        for setting in ({}, {"top_p": 0.9}, {"top_k": 700, "min_p": 0.001}):
            per_row = {k: _all(dev, 81, v, torch.int32 if k == "top_k" else torch.float32) for k, v in setting.items()}
            want = _check_sample(x, u, **{k: v[:3] for k, v in per_row.items()})
            got = lb.sample(x.repeat(27, 1), u.repeat(27), **per_row)  # more rows than half the SMs
            assert torch.equal(got.view(27, 3), want.expand(27, 3)), (vocab, setting)


@pytest.mark.parametrize("setting", [{}, {"temperature": 0.6, "top_p": 0.95}, {"top_k": 50}, {"top_k": 3000, "top_p": 0.8}, {"min_p": 0.02}])
@pytest.mark.parametrize("vocab", [900, 10007, 128001])
def test_sample_a_row_alone_in_a_batch_and_at_each_alignment(dev, vocab, setting):
    """sums in another order, by another number of CTAs: the same tokens but next to a border (none here is)"""
    import luisaml_b200 as lb
    x, u = _rows(dev, 4, vocab)
    per_row = {k: _all(dev, 100, v, torch.int32 if k == "top_k" else torch.float32) for k, v in setting.items()}
    few = {k: v[:4] for k, v in per_row.items()}
    want = _check_sample(x, u, **few)
    for r in range(4):
        assert lb.sample(x[r:r + 1], u[r:r + 1], **{k: v[:1] for k, v in per_row.items()}).item() == want[r]
    assert torch.equal(lb.sample(x.repeat(25, 1), u.repeat(25), **per_row).view(25, 4), want.expand(25, 4))
    for off in range(1, 4):
        wide = torch.zeros(4, vocab + 5, device=dev)
        wide[:, off:off + vocab] = x
        assert torch.equal(lb.sample(wide[:, off:off + vocab], u, **few), want), off


@pytest.mark.parametrize("use_ended", [False, True])
@pytest.mark.parametrize("batch,new,held,page,cols,spare,code", [
    (8, 700, 50, 16, 60, 8 * 60, 0),
    (8, 700, 50, 16, 60, 3, 8),  # the list runs out
    (8, 700, 50, 16, 30, 8 * 60, 7),  # rows longer than the table
    (300, 9, 20, 16, 2, 300 * 2, 0),
    (300, 9, 40, 16, 2, 300 * 2, 7),
    (300, 9, 24, 16, 3, 10, 8),
    (1, 5000, 0, 1, 5000, 5000, 0),
    (1, 5000, 0, 1, 5000, 4999, 8),
    (1, 5000, 1, 1, 5000, 5001, 7)])
def test_plan_says_what_does_not_fit(dev, batch, new, held, page, cols, spare, code, use_ended):
    """the error word is 8, 7 or clear, as the lengths say"""
    _check_plan(dev, [new] * batch, [held] * batch, [False] * batch, page, cols, spare=spare, use_ended=use_ended)
    assert _no_device_error() == code


@pytest.mark.parametrize("case", ["negative new", "negative held", "tokens left out", "list full"])
def test_plan_says_which_lengths_are_wrong(dev, case):
    new, held, ended, kw = [3, 4, 5], [20, 0, 33], [False, False, case == "list full"], {}
    if case == "negative new":
        new[1] = -1
    elif case == "negative held":
        held[1] = -5
    elif case == "tokens left out":
        kw["total"] = 11
    else:
        kw["capacity"] = 10
    _check_plan(dev, new, held, ended, 16, 4, spare=8 if case == "list full" else 12, **kw)
    assert _no_device_error() == 7
