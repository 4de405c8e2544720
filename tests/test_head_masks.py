"""Finite masks in the bias of the head: entries as low as any program writes them leave the softmax, and nothing else.

A masked entry's logit lies 1e4 and more below the others' (|x W| < 100 here), its exponential is 0 in 64 bits as in 32: the
values are those of the same call with a bias of -inf there, and so are the bounds (test_head.Exact).
"""
import math

import pytest
import torch

from test_head import BF, F32, Exact, both, check_grads, check_loss, inputs

gpu = pytest.mark.gpu
MASKS = [-1e4, -1e9, -1e10, -1e12, -1e20, -1e25, -1e30, -1e31, float(torch.finfo(torch.float32).min)]
ROWS = [1, 2, 3, 300]


def masked(t, v, where, mask, seed, d=64):
    x, w, target, b = inputs(t, d, v, seed=seed, ignored=0.1)
    b[where] = mask
    off = torch.zeros(v, dtype=torch.bool, device="cuda")
    off[where] = True
    left = (~off).nonzero().view(-1)
    target = torch.where(target >= 0, left[target.clamp_min(0).long() % len(left)].int(), target)
    return x, w, target, b, off


@gpu
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("where", [slice(0, 40), slice(256, 512), slice(1436, 1500), slice(96, 1470)])
def test_masked_entries(where, mask, t):
    """The first columns, a whole tile, the last ones, all but a few on either side."""
    x, w, target, b, off = masked(t, 1500, where, mask, seed=20)
    ex = Exact(x, w, target, b.masked_fill(off, -math.inf))
    for kind in (F32, BF):
        nll, lse, dx, dw, db = both(x, w, target, b, kind)
        check_loss(ex, nll, lse)
        check_grads(ex, kind, dx=dx, dw=dw, db=db)
        assert not dw[:, off].any() and not db[off].any()


@gpu
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("mask", [-1e10, -1e30])
def test_padding_of_a_large_vocabulary(mask, t):
    """100,000 entries, the last 64 of them padding: half of the last tile's columns hold nothing but the mask."""
    x, w, target, b, off = masked(t, 100000, slice(99936, 100000), mask, seed=21)
    ex = Exact(x, w, target, b.masked_fill(off, -math.inf))
    nll, lse, dx, dw, db = both(x, w, target, b, BF)
    check_loss(ex, nll, lse)
    check_grads(ex, BF, dx=dx, dw=dw, db=db)


@gpu
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("mask", MASKS)
def test_nothing_but_the_mask(mask, t):
    """Every entry masked: the largest logit is known to half a step of the mask (and |x W| < 100), lse to that and log V."""
    v = 700
    x, w, target, b, _ = masked(t, v, slice(0, 0), mask, seed=22)
    b.fill_(mask)
    nll, lse, dx, dw, db = both(x, w, target, b, F32)
    near = 100 + math.log(v) + 3 * 2.0 ** -24 * abs(mask)
    assert ((lse.double() - mask).abs() <= near).all()
    assert (nll[target >= 0].abs() <= 2 * near).all() and not nll[target < 0].any()
    for a in (dx, dw, db):
        assert torch.isfinite(a).all()


@gpu
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("shift", [300.0, -300.0, 5000.0, -70000.0])
def test_a_shift_of_all_logits(t, shift):
    """One number added to every bias moves lse by it and leaves nll and the gradients, but for roundings of its size."""
    x, w, target, b, _ = masked(t, 900, slice(0, 0), 0.0, seed=23)
    ex = Exact(x, w, target, b + shift)
    nll, lse, dx, dw, db = both(x, w, target, b + shift, F32)
    check_loss(ex, nll, lse)
    check_grads(ex, F32, dx=dx, dw=dw, db=db)
