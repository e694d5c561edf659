"""Forms of a tree_attention call that the documentation allows beside the plain
one: shared trees and depths, operands that a kernel cannot read in place, calls
on two streams at once. All equal the plain call bit for bit."""

from __future__ import annotations

import pytest
import torch

from engine.attention import tree_attention
from engine.decode import DraftTree, draft_tree
from engine.model.rope import build_rope_cache
from test_tree_gpu import DEV, Case

pytestmark = pytest.mark.gpu

N = 37


def shared_case():
    c = Case([50, 600], N, 64, torch.bfloat16, seed=7)
    c.parents = [c.parents[0]] * 2
    g = torch.Generator().manual_seed(1)
    new = [torch.randn(2 * N, c.Hk, 64, generator=g).bfloat16().to(DEV) for _ in range(2)]
    rope = tuple(t.to(DEV) for t in build_rope_cache(700, 64))
    return c, new, rope


def run(c, mask, new=None, rope=None, depths=None):
    """The output and the pools behind it."""
    q, k, v, bt, lens = c.device()
    out = tree_attention(q, k, v, bt, lens, mask, rope=rope, depths=depths, new_kv=new)
    return out, k, v


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("append", [False, True])
def test_shared_tree_and_depths(append):
    c, new, rope = shared_case()
    tree = c.tree()
    one = draft_tree(torch.tensor(c.parents[0], dtype=torch.int32, device=DEV))
    new = new if append else None
    want = run(c, tree.mask, new, rope, tree.depths)
    assert one.mask.shape == (N, 2) and one.depths.shape == (N,)
    assert same(run(c, one.mask, new, rope, one.depths), want)
    assert same(run(c, one.mask, new, rope, tree.depths), want)
    assert same(run(c, tree.mask, new, rope, one.depths), want)
    assert same(run(c, one.mask.expand(2, N, 2), new, rope, one.depths.expand(2, N)), want)
    if append:  # without a rotation
        assert same(run(c, one.mask, new), run(c, tree.mask, new))


def test_operands_that_need_a_copy():
    c, new, rope = shared_case()
    tree = c.tree()
    want = run(c, tree.mask, new, rope, tree.depths)

    def odd_rows(t):  # rows 2 bytes off their alignment
        wide = torch.zeros(t.shape[0], t.shape[1], 67, dtype=t.dtype, device=DEV)
        wide[..., 1:65] = t
        return wide[..., 1:65]

    def turned(t):  # another order of the dimensions in memory
        n = t.dim()
        return t.permute(*reversed(range(n))).contiguous().permute(*reversed(range(n)))

    def spread(t):  # rows inside a wider tensor, read in place
        wide = torch.zeros(t.shape[0], 3, *t.shape[1:], dtype=t.dtype, device=DEV)
        wide[:, 1] = t
        return wide[:, 1]

    for k_form in (odd_rows, turned, spread):
        for v_form in (odd_rows, turned, spread):
            assert same(run(c, tree.mask, (k_form(new[0]), v_form(new[1])), rope, tree.depths), want)
    assert not turned(tree.mask).is_contiguous() and not turned(tree.depths).is_contiguous()
    assert same(run(c, turned(tree.mask), new, rope, tree.depths), want)
    assert same(run(c, spread(tree.mask), new, rope, spread(tree.depths)), want)
    assert same(run(c, tree.mask, new, rope, turned(tree.depths)), want)
    assert same(run(c, turned(tree.mask[0]), new, rope, turned(tree.depths)), want)


def test_two_streams_at_once():
    # each call has its own partial states
    cases = [Case([700, 3000], 26, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    args = [(*c.device(), c.tree().mask) for c in cases]
    want = [tree_attention(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tree_attention(*args[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for outs, w in zip(got, want) for o in outs)


def test_a_tree_of_the_callers_own():
    # a DraftTree is its three tensors: any relation of the nodes, not only ancestors
    c = Case([90, 1200], 40, 64, torch.float16, seed=3)
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 40, 2), dtype=torch.int32, generator=torch.Generator().manual_seed(4))
    mask[0, 5], mask[1, 39] = 0, torch.tensor([0, -256])  # an empty row; bits past the nodes alone
    tree = DraftTree(None, mask.to(DEV), None)
    bits = (mask.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32) & 1).bool().flatten(2)[..., :40]
    out = tree_attention(*c.device(), tree.mask).cpu()
    see = [torch.cat([bits[b].any(1, keepdim=True).expand(40, c.bases[b]), bits[b]], 1) for b in range(2)]
    c.see = lambda b: see[b]
    c.check(out)
    assert not out[0, :, 5].any() and not out[1, :, 39].any()
