"""Draft trees on the GPU: calls at the edge of what the documentation allows."""

from __future__ import annotations

import pytest
import torch

from engine.attention import tree_attention
from engine.cache import kv_keep
from engine.decode import draft_tree, verify_draft, verify_greedy
from test_draft_gpu import make
from test_tree_gpu import Case

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


@pytest.mark.parametrize("shared", [False, True])  # parents of shape (0,) take the Python path
def test_trees_without_nodes_accept_nothing(shared):
    B = 5
    p = torch.zeros((0,) if shared else (B, 0), dtype=torch.int32, device=DEV)
    x = torch.zeros((B, 0), dtype=torch.int64, device=DEV)
    t, u = torch.zeros((B, 0, 30), device=DEV), torch.zeros((B, 0), device=DEV)
    for call in (lambda: verify_greedy(t, x, p), lambda: verify_draft(t, x, p, u), lambda: verify_draft(t, x, p, u, t)):
        dirty = torch.full((B,), 77, dtype=torch.int32, device=DEV)  # what the allocator hands out next
        del dirty
        assert call().counts.tolist() == [0] * B


LOW, HIGH = -2 ** 63, 2 ** 63 - 1


@pytest.mark.parametrize("marker", [LOW, -2 ** 32, -2 ** 32 + 1, -2 ** 40 + 3])
def test_int64_parents_of_any_value(marker):
    # a parent below -1 is a padding slot, whatever its lower 32 bits; one far above its child is a broken chain
    rows = [[-1, 0, marker, 1, 2, 2 ** 32 + 1], [marker, 0, 0, 1, 2, HIGH]]
    same = [[-1, 0, -2, 1, 2, 100], [-2, 0, 0, 1, 2, 100]]
    a, b = draft_tree(dev(rows, torch.int64)), draft_tree(dev(same))
    assert torch.equal(a.mask, b.mask) and torch.equal(a.depths, b.depths)
    shared = draft_tree(dev(rows[0], torch.int64))
    assert torch.equal(shared.mask, b.mask[0])
    g = torch.Generator(DEV).manual_seed(1)
    logits = torch.randn((2, 6, 20), generator=g, device=DEV)
    best = logits.argmax(-1)
    x = torch.stack([best[i].gather(0, dev(same)[i].clamp(0, 5).long()) for i in range(2)])  # every child right
    p = torch.softmax(logits, -1)
    u = torch.full((2, 6), 0.25, device=DEV)
    for verify in (lambda q: verify_greedy(logits, x, q), lambda q: verify_draft(p, x, q, u)):
        assert all(torch.equal(m, n) for m, n in zip(verify(dev(rows, torch.int64)), verify(dev(same))))
        both = [verify(dev(r[0], d)) for r, d in ((rows, torch.int64), (same, torch.int32))]  # one tree for all
        assert all(torch.equal(m, n) for m, n in zip(*both))


@pytest.mark.parametrize("far", [LOW, HIGH, 2 ** 32, -2 ** 32, 2 ** 35 + 2])
def test_keep_of_int64_values_out_of_range_moves_nothing(far):
    g = torch.Generator(DEV).manual_seed(2)
    pools = [torch.randn((4, 4, 1, 16), generator=g, device=DEV).half() for _ in range(2)]
    before = [t.clone() for t in pools]
    good = dict(bt=[[0, 1]], st=[1], pa=[[0, 2, 3]], cn=[3])
    for name, value in (("bt", [[far, far]]), ("st", [far]), ("pa", [[0, far, far]]), ("cn", [min(far, 0)])):
        a = {**good, name: value}
        for pair in ((list, [pools[0]], [pools[1]]), (tuple, (pools[0],), (pools[1],))):
            kv_keep(pair[1], pair[2], *(dev(a[n], torch.int64) for n in ("bt", "st", "pa", "cn")))
            assert all(torch.equal(t, b) for t, b in zip(pools, before)), (name, pair[0])
    kv_keep([pools[0]], [pools[1]], *(dev(good[n], torch.int64) for n in ("bt", "st", "pa", "cn")))
    assert not torch.equal(pools[0], before[0])


def test_int64_ids_and_lengths_out_of_range_are_nan():
    c = Case([20, 40, 60], 4, 64, torch.float16, seed=1)
    q, k, v, bt, lens = c.device()
    mask = c.tree().mask
    clean = tree_attention(q, k, v, bt, lens, mask)
    wide = mask.unsqueeze(0)[0].transpose(0, 1).contiguous().transpose(0, 1)  # (strides of another order: Python path)
    for m in (mask, wide):
        ids, n = bt.long(), lens.long()
        ids[0, 0] = 2 ** 32 + int(bt[0, 0])
        n[1] += 2 ** 32
        out = tree_attention(q, k, v, ids, n, m)
        assert torch.isnan(out[:2].float()).all() and torch.equal(out[2], clean[2])


@pytest.mark.parametrize("mode,V", [("greedy", 501), ("greedy", 1_500_000), ("picks", 501), ("iid", 501), ("tree", 501)])
def test_rows_that_no_walk_visits_decide_nothing(mode, V):
    # (the larger vocabulary is over 64 MiB of logits: its rows are read on the walk)
    B, N, dtype = 3, 14, torch.bfloat16 if V > 501 else torch.float32
    target, tokens, parents, u, draft = make(B, N, 501, dtype, mode, seed=7)
    parents = [p[:12] + [-2, -2] for p in parents]
    t, x, p = target.to(DEV), dev(tokens, torch.int64), dev(parents)
    if V > 501:
        wide = torch.full((B, N, V), -50.0, dtype=dtype, device=DEV)
        wide[..., :501] = t
        t = wide
    d = None if draft is None else draft.to(DEV)
    run = lambda: (verify_greedy(t, x, p) if mode == "greedy" else  # noqa: E731
                   verify_draft(t, x, p, dev(u, torch.float32), d, replacement=mode == "iid"))
    want = run()
    unseen = torch.ones((B, N), dtype=torch.bool, device=DEV)
    for b, n in enumerate(want.counts.tolist()):
        unseen[b, want.path[b, :n].long()] = False
    for bad in (float("nan"), float("inf")):
        for rows in (t, d):
            if rows is not None:
                rows[unseen] = bad
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
