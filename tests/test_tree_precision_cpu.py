"""What the 64-bit oracle's two-part bound of tree attention tells apart, on the
CPU: probabilities in two 16-bit parts lie within it, rounded once they do not.

Rounded once, L about equal probabilities 1/L are off by some h / (4 L) each with
either sign, a row by h / (4 sqrt(L)). The bound's fp32 terms, 2^-24 (2 (D + 8)
reach + 2 L + 64) with reach some 6 for these inputs, are 1144 steps of 2^-24 at
L = 300, D = 32, or 0.14 h in fp16 against 0.014 h of the rounding: there the bound
cannot tell the two apart. In bf16 they are 0.017 h against 0.014 h times the
largest of some 300 outputs, over 2.5; at L = 40 and below they are well under."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import tree_attention_f64


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L,D", [(9, 16), (40, 64), (300, 32)])
def test_two_part_bound(L, D, dtype):
    g = torch.Generator().manual_seed(L)
    q, k, v = (torch.randn(s, generator=g).to(dtype) for s in ((2, 5, D), (L, 1, D), (L, 1, D)))
    see = torch.rand(5, L, generator=g) < 0.8
    see[:, 0] = True
    scale = 1 / math.sqrt(D)
    ref, bound = tree_attention_f64(q, k, v, see, scale, parts=2)
    once = tree_attention_f64(q, k, v, see, scale)[1]
    s = (q.double() @ k[:, 0].double().t() * scale).masked_fill(~see, -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    hi = p.to(dtype).double()
    both = hi + (p - hi).to(dtype).double()
    err = {n: ((w @ v[:, 0].double() / p.sum(-1, keepdim=True)).to(dtype).double() - ref).abs()
           for n, w in (("one", hi), ("two", both))}
    assert bool((err["two"] <= bound).all()) and bool((err["one"] <= once).all())
    if L < 300 or dtype == torch.bfloat16:
        assert not bool((err["one"] <= bound).all())
