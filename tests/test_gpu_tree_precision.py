"""How many bits of a probability reach hxm_tree_attention's product with V: those of two 16-bit
halves, each rounded, as in hxm_paged_attention.

A sequence has a token of score x, weight w = 2^x in [1/2, 1), of value 64, and two of score 0,
weight 1, of values -64 hi and -64 lo, the halves of w as rounding gives them, so that
    out (2 + w) / 64 = w - hi - lo
is what the halves leave of w, with no larger term that would hide it.  With s = 8 (bf16) or 11
(f16) significant bits:
* hi is off by half of a step of 2^-s at most, lo by half of one of 2^-s of that, 2^-(2 s + 2) of
  1 (a first half that is cut off instead leaves up to 2^-s and so twice that);
* w itself: the score's exponent is off by two roundings of the scale's two factors and one of
  the product, (2 + 1) 2^-24, in f16 by one more where 7 is added, 2^-22, times ln 2; exp2 by
  2^-23 of w; the weights of 1 by as much of their values, 2^-23 together;
* the output's rounding, 2^-s of what is left.
"""
import math

import numpy as np
import pytest
import torch

import hxm.ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,s", [("bf16", 8), ("f16", 11)])
@pytest.mark.parametrize("group", [1, 40, 100])       # one, two and four waves over the rows
def test_bits_of_a_probability(dev, name, s, group):
    dt = torch.float16 if name == "f16" else torch.bfloat16
    x = -(torch.arange(1, 257, dtype=torch.float64) / 257).to(dt)
    scale = float(np.float32(math.log(2.0)))
    w = (x.double() * scale).exp()
    hi = w.to(dt)
    lo = (w - hi.double()).to(dt)
    n, page, B, dim = 4, 16, len(x), 64
    kc = torch.zeros(B, 1, page, dim, dtype=dt)
    vc = torch.zeros(B, 1, page, dim, dtype=dt)
    kc[:, 0, 0, 0] = x
    vc[:, 0, 0] = 64
    vc[:, 0, 1] = (-64 * hi.double()).to(dt)[:, None]
    vc[:, 0, 2] = (-64 * lo.double()).to(dt)[:, None]
    assert torch.equal(vc[:, 0, 2, 0].double(), -64 * lo.double())
    kc[:, 0, 3, 0] = -120                             # the node itself: nothing, of value 0
    q = torch.zeros(B, 1, group, dim, dtype=dt)
    q[..., 0] = 1
    table = torch.arange(B, dtype=torch.int32, device=dev)[:, None]
    lens = torch.full((B,), n, dtype=torch.int32, device=dev)
    out = ops.tree_attention(q.to(dev), kc.to(dev), vc.to(dev), table, lens, scale=scale)
    got = out.cpu().double()[:, 0] * (2 + w)[:, None, None] / 64
    left = (w - hi.double() - lo.double())[:, None, None]
    assert left.abs().max() <= 2.0 ** -(2 * s + 2)
    noise = (3 * 2.0 ** -24 + (2.0 ** -22 if name == "f16" else 0)) * math.log(2.0) + 2 * 2.0 ** -23
    tol = 2.0 ** -(2 * s + 2) + noise + 2.0 ** -s * got.abs()
    bad = ~((got - left).abs() <= tol)
    worst = float((got - left).abs().max() * 2 ** (2 * s + 2))
    assert not bad.any(), (int(bad[:, 0, 0].sum()), worst)
