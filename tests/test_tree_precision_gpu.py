"""The probabilities of tree attention lose nothing that shows in the output:
every element is within half a step of the output's type, the rounding of a
probability in two parts and the fp32 sums (``tree_attention_f64`` with
``parts=2``). With probabilities rounded once to 16 bits the error against 64
bits is 1.3 to 1.4 times the output's own rounding, and elements near zero are
off by many steps."""

from __future__ import annotations

import math

import pytest
import torch

from engine.decode import draft_tree
from engine.attention import tree_attention
from oracle import tree_attention_f64
from test_tree_gpu import DEV, Case

pytestmark = pytest.mark.gpu


def check(c, out, sequences=None):
    for b in range(c.B) if sequences is None else sequences:
        at = c.slots(b)
        k, v = c.k.view(-1, c.Hk, c.D)[at], c.v.view(-1, c.Hk, c.D)[at]
        ref, bound = tree_attention_f64(c.q[b].transpose(0, 1), k, v, c.see(b), 1 / math.sqrt(c.D), parts=2)
        over = (out[b].double() - ref).abs() - bound
        assert float(over.max()) <= 0, f"sequence {b}: {int((over > 0).sum())} elements over, {float(over.max()):.3e}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("N,Hq,Hk", [(8, 8, 2), (13, 8, 2), (26, 8, 2), (65, 4, 1)])  # 32, 52, 104 and 260 rows a head
def test_every_row_layout(N, Hq, Hk, D, dtype):
    c = Case([0, 30, 200], N, D, dtype, Hq=Hq, Hk=Hk, seed=N + D)
    check(c, c.run())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_split_sequences_and_a_padded_batch(dtype):
    # a bound below one key's weight of some 1/3000: a lost or doubled key shows here too
    c = Case([3000, 700, 64], 9, 64, dtype, seed=4, nodes=[9, 4, 0])
    check(c, c.run())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_peaked_scores(dtype):
    # one key takes most of a row: its probability is near 1, the others are far below
    c = Case([40, 600], 11, 64, dtype, seed=5, qscale=4.0)
    check(c, c.run())


def test_a_seen_value_that_is_not_finite_shows():
    # in a tile of history alone, in the first tile that holds nodes, and never in another column
    c = Case([100], 6, 64, torch.bfloat16, seed=6)
    clean = c.run()
    for position in (5, 97):
        c2 = Case([100], 6, 64, torch.bfloat16, seed=6)
        c2.v.view(-1, 2, 64)[c2.slots(0)[position], 1, 9] = float("inf")
        out = c2.run()
        assert not torch.isfinite(out[0, 4:, :, 9].float()).any()
        out[0, 4:, :, 9] = clean[0, 4:, :, 9]
        assert torch.equal(out, clean)
