"""Attention of a tree of drafted tokens over the paged cache
(``engine.attention.tree_attention``) against the 64-bit oracle, elementwise
within the rounding bound that the oracle derives with each output
(``oracle.draft_ref.tree_attention_f64``)."""

from __future__ import annotations

import math
import random

import pytest
import torch

from engine.attention import paged_attention, tree_attention, tree_workspace_bytes
from engine.cache import kv_append
from engine.decode import draft_tree
from engine.model.rope import build_rope_cache, rope_apply
from oracle import mask_words, tree_attention_f64, tree_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def random_tree(r: random.Random, n: int, N: int) -> list[int]:
    """n nodes of a random tree and N - n padding slots."""
    return ([-1] + [r.randint(max(0, i // 3 - 1), i - 1) for i in range(1, n)] if n else []) + [-2] * (N - n)


class Case:
    """A pool of scattered blocks with histories and nodes in it, on the CPU."""

    def __init__(self, bases, N, D, dtype, bs=16, Hq=8, Hk=2, seed=0, nodes=None, qscale=1.0):
        r = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        B = len(bases)
        self.B, self.N, self.D, self.Hq, self.Hk, self.bs, self.dtype = B, N, D, Hq, Hk, bs, dtype
        self.bases = list(bases)
        self.lens = [h + N for h in bases]
        need = [-(-n // bs) for n in self.lens]
        ids = list(range(sum(need) + 3))
        r.shuffle(ids)
        self.blocks, at = [], 0
        for n in need:
            self.blocks.append(ids[at:at + n])
            at += n
        self.bt = torch.zeros((B, max(need)), dtype=torch.int32)
        for b, bl in enumerate(self.blocks):
            self.bt[b, :len(bl)] = torch.tensor(bl, dtype=torch.int32)
        self.k = torch.randn(len(ids), bs, Hk, D, generator=g).to(dtype)
        self.v = torch.randn(len(ids), bs, Hk, D, generator=g).to(dtype)
        self.q = (torch.randn(B, N, Hq, D, generator=g) * qscale).to(dtype)
        self.parents = [random_tree(r, N if nodes is None else nodes[b], N) for b in range(B)]

    def slots(self, b):
        pos = torch.arange(self.lens[b])
        return torch.tensor(self.blocks[b])[pos // self.bs] * self.bs + pos % self.bs

    def see(self, b):
        seen, _ = tree_ref(self.parents[b])
        see = torch.zeros((self.N, self.lens[b]), dtype=torch.bool)
        for i, s in enumerate(seen):
            if s:
                see[i, :self.bases[b]] = True
                see[i, [self.bases[b] + a for a in s]] = True
        return see

    def device(self):
        q = self.q.to(DEV).transpose(1, 2)
        return (q, self.k.to(DEV), self.v.to(DEV), self.bt.to(DEV),
                torch.tensor(self.lens, dtype=torch.int32, device=DEV))

    def tree(self):
        return draft_tree(torch.tensor(self.parents, dtype=torch.int32, device=DEV))

    def run(self, **kw):
        out = tree_attention(*self.device(), self.tree().mask, **kw)
        torch.cuda.synchronize()
        return out.cpu()

    def check(self, out, scale=None, sequences=None):
        scale = 1 / math.sqrt(self.D) if scale is None else scale
        for b in range(self.B) if sequences is None else sequences:
            at = self.slots(b)
            k, v = self.k.view(-1, self.Hk, self.D)[at], self.v.view(-1, self.Hk, self.D)[at]
            ref, bound = tree_attention_f64(self.q[b].transpose(0, 1), k, v, self.see(b), scale)
            err = (out[b].double() - ref).abs()
            assert torch.isfinite(out[b].double()).all(), f"sequence {b}"
            worst = float((err - bound).max())
            assert worst <= 0, f"sequence {b}: error over its bound by {worst:.3e}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("N,bases", [(1, [0, 1, 31, 200]), (8, [0, 24, 25, 777]), (13, [5, 300]), (26, [6, 1000]),
                                     (65, [0, 63, 700])])
def test_tree_attention(N, bases, D, dtype):
    c = Case(bases, N, D, dtype, seed=N + D)
    c.check(c.run())


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (4, 4), (28, 4), (6, 3), (16, 1), (40, 8)])
@pytest.mark.parametrize("N", [3, 17, 40])
def test_heads(Hq, Hk, N):
    c = Case([70, 511], N, 64, torch.float16, Hq=Hq, Hk=Hk, seed=Hq + N)
    c.check(c.run())


@pytest.mark.parametrize("bs", [1, 3, 16, 100])
def test_block_sizes(bs):
    c = Case([0, 45, 1500], 9, 64, torch.bfloat16, bs=bs, seed=bs)
    c.check(c.run())


@pytest.mark.parametrize("N,Hq,Hk,D", [(255, 7, 1, 128), (256, 2, 2, 64), (300, 4, 1, 256), (1024, 1, 1, 32)])
def test_large_trees(N, Hq, Hk, D):
    c = Case([130], N, D, torch.bfloat16, Hq=Hq, Hk=Hk, seed=N)
    c.check(c.run())


def test_long_history_and_ragged_batch():
    c = Case([9000, 3, 0, 4100, 33], 7, 64, torch.float16, Hq=2, Hk=1, seed=5)
    c.check(c.run())
    c.check(c.run(max_context=max(c.lens)))


def test_many_sequences():
    r = random.Random(1)
    c = Case([r.randint(0, 90) for _ in range(150)], 5, 32, torch.float16, Hq=2, Hk=2, seed=6,
             nodes=[r.randint(0, 5) for _ in range(150)])
    c.check(c.run())


@pytest.mark.parametrize("N,Hq,Hk,D", [(3, 2, 2, 64), (33, 2, 1, 128), (65, 4, 1, 32)])
def test_many_sequences_some_of_them_cut(N, Hq, Hk, D):
    # more workgroups than half of the CUs: only the longest sequences are split
    r = random.Random(N)
    c = Case([r.randint(0, 200) for _ in range(170)] + [5000, 2100 - N, 2048 - N, 2049 - N, 0], N, D, torch.bfloat16,
             Hq=Hq, Hk=Hk, seed=N)
    c.check(c.run(max_context=max(c.lens)), sequences=[0, 1, 50, 169, 170, 171, 172, 173, 174])
    c.check(c.run(), sequences=[2, 100, 170, 172])


@pytest.mark.parametrize("N,bases", [(1, [0] * 40), (5, [0, 27, 20] * 20), (33, [0, 31, 30, 62] * 12),
                                     (100, [0, 28, 60] * 10), (200, [0, 24, 56])])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_short_sequences_share_a_cu(N, bases, D):
    # one to eight tiles with a tight max_context: few stages in the ring
    c = Case(bases, N, D, torch.float16, Hq=8, Hk=2 if N < 100 else 1, seed=N)
    c.check(c.run(max_context=max(c.lens)), sequences=range(min(4, len(bases))))


def test_lengths_over_max_context_are_nan():
    c = Case([10, 300, 40], 6, 64, torch.float16, seed=3)
    out = c.run(max_context=64)
    assert torch.isnan(out[1]).all()
    c.check(out, sequences=[0, 2])


def test_largest_tree_over_a_history():
    c = Case([777], 1024, 128, torch.float16, Hq=2, Hk=1, seed=2)
    c.check(c.run())


@pytest.mark.parametrize("base", [0, 40, 3000])
def test_padding_rows_are_zero(base):
    # trees of fewer nodes than slots, one sequence without any; a single long one splits over workgroups
    c = Case([base, base + 7, base], 20, 64, torch.float16, seed=2, nodes=[20, 3, 0])
    out = c.run()
    c.check(out)
    assert (out[1][:, 3:] == 0).all() and (out[2] == 0).all()


def test_garbage_in_masked_places():
    # NaN and infinities in padding slots, behind the context and in siblings that a node does not see
    c = Case([37, 2000], 12, 128, torch.bfloat16, seed=3, nodes=[5, 9])
    clean = c.run()
    for b, n in ((0, 5), (1, 9)):
        at = c.slots(b)[c.bases[b] + n:]
        c.k.view(-1, c.Hk, c.D)[at] = float("nan")
        c.v.view(-1, c.Hk, c.D)[at] = float("inf")
        last = c.lens[b] % c.bs
        if last:
            c.k[c.blocks[b][-1], last:] = float("nan")
            c.v[c.blocks[b][-1], last:] = float("-inf")
    out = c.run()
    assert torch.equal(out, clean)
    # a node whose V is not finite: its descendants show it in those columns, the others do not
    bad = c.slots(1)[c.bases[1] + 2]
    c.v.view(-1, c.Hk, c.D)[bad, 0, 5] = float("inf")
    c.v.view(-1, c.Hk, c.D)[bad, 1, 7] = float("nan")
    c.k.view(-1, c.Hk, c.D)[c.slots(1)[c.bases[1] + 4]] = float("nan")
    seen, _ = tree_ref(c.parents[1])
    out = c.run()
    group = c.Hq // c.Hk
    for i in range(9):
        o, want = out[1][:, i], clean[1][:, i].clone()
        if 4 in seen[i]:
            assert torch.isnan(o.float()).all()
            continue
        if 2 in seen[i]:
            assert (o[:group, 5] == float("inf")).all() and torch.isnan(o[group:, 7].float()).all()
            o[:group, 5] = want[:group, 5]
            o[group:, 7] = want[group:, 7]
        assert torch.equal(o, want), i


def test_chain_equals_paged_verify():
    # a chain sees what the causal rule of the new tokens shows
    c = Case([0, 100, 1023], 6, 64, torch.float16, seed=4)
    c.parents = [[-1, 0, 1, 2, 3, 4]] * 3
    out = c.run()
    c.check(out)
    q, k, v, bt, lens = c.device()
    ref = paged_attention(q, k, v, bt, lens, causal=True).cpu()
    assert float((out.float() - ref.float()).abs().max()) <= 2 * 2.0 ** -11 * float(ref.abs().max()) * 2


def test_shared_tree_strides_and_out():
    c = Case([50, 600], 10, 64, torch.bfloat16, seed=7)
    c.parents = [c.parents[0]] * 2
    tree = draft_tree(torch.tensor(c.parents[0], device=DEV))
    q, k, v, bt, lens = c.device()
    want = tree_attention(q, k, v, bt, lens, c.tree().mask)
    c.check(want.cpu())
    assert tree.mask.dim() == 2 and torch.equal(tree_attention(q, k, v, bt, lens, tree.mask), want)
    assert torch.equal(tree_attention(q, k, v, bt.long(), lens.long(), tree.mask.expand(2, -1, -1)), want)
    # q rows that the kernel cannot read in place, pools as views, an output in (B, N, H, D) order
    wide = torch.zeros(2, 8, 10, 67, dtype=q.dtype, device=DEV)
    wide[..., 1:65] = q
    pool = torch.zeros(*k.shape[:2], 3, *k.shape[2:], dtype=k.dtype, device=DEV)
    pool[:, :, 1], pool[:, :, 2] = k, v
    rows = torch.full((2, 10, 8, 64), float("nan"), dtype=q.dtype, device=DEV)
    got = tree_attention(wide[..., 1:65], pool[:, :, 1], pool[:, :, 2], bt, lens, tree.mask, out=rows.transpose(1, 2))
    assert torch.equal(got, want) and torch.equal(rows.transpose(1, 2), want)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(scale):
    c = Case([400], 9, 64, torch.float16, seed=8)
    c.check(c.run(scale=scale), scale=scale)


def test_peaked_scores():
    c = Case([600, 5000], 9, 64, torch.float16, seed=9, qscale=8.0)
    c.check(c.run())


def test_far_apart_blocks():
    # pool rows whose element offsets pass 2^31
    D, Hk, bs = 64, 1, 16
    blocks, stride = 4, 1 << 30
    store = torch.empty((blocks - 1) * stride + bs * D, dtype=torch.float16, device=DEV)
    c = Case([40], 8, D, torch.float16, Hq=2, Hk=Hk, seed=10)
    order = [2, 0, 3]
    view = store.as_strided((blocks, bs, Hk, D), (stride, D, D, 1))
    for logical, phys in enumerate(order):
        view[phys] = c.k[c.blocks[0][logical]].to(DEV)
    vsrc = c.v.to(DEV)
    vsmall = torch.zeros(blocks, bs, Hk, D, dtype=torch.float16, device=DEV)
    for logical, phys in enumerate(order):
        vsmall[phys] = vsrc[c.blocks[0][logical]]
    bt = torch.tensor([order], dtype=torch.int32, device=DEV)
    lens = torch.tensor(c.lens, dtype=torch.int32, device=DEV)
    out = tree_attention(c.q.to(DEV).transpose(1, 2), view, vsmall, bt, lens, c.tree().mask)
    c.check(out.cpu())


def test_invalid_sequences_are_nan_and_the_others_right():
    c = Case([100, 200, 50, 3000], 6, 64, torch.float16, seed=11, nodes=[6, 6, 2, 6])
    q, k, v, bt, lens = c.device()
    mask = c.tree().mask
    lens[0] = 5                    # fewer than the nodes
    bt[1, 3] = k.shape[0]          # outside the pool
    lens[2] = bt.shape[1] * 16 + 1  # longer than the table
    out = tree_attention(q, k, v, bt, lens, mask).cpu()
    assert torch.isnan(out[0].float()).all() and torch.isnan(out[1].float()).all()
    assert torch.isnan(out[2][:, :2].float()).all() and (out[2][:, 2:] == 0).all()
    c.check(out, sequences=[3])
    bt[3, -1] = -1
    assert torch.isnan(tree_attention(q, k, v, bt, lens, mask, max_context=4000).cpu()[3].float()).all()


@pytest.mark.parametrize("tables", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rope_and_append(D, dtype, tables):
    N = 11
    c = Case([0, 37, 900], N, D, dtype, seed=D, nodes=[11, 6, 9])
    g = torch.Generator().manual_seed(1)
    kn = torch.randn(c.B * N, c.Hk, D, generator=g).to(dtype).to(DEV)
    vn = torch.randn(c.B * N, c.Hk, D, generator=g).to(dtype).to(DEV)
    cos, sin = (t.to(DEV, tables) for t in build_rope_cache(950, D))
    tree = c.tree()
    q, k, v, bt, lens = c.device()
    # the same in steps: rotate at base + depth, write the real nodes' rows, attend
    base = torch.tensor(c.bases, device=DEV)
    pos = (base.unsqueeze(1) + tree.depths.clamp(min=0)).to(torch.int32)
    q_rot = rope_apply(q, cos, sin, positions=pos)
    k_rot = rope_apply(kn.view(c.B, N, c.Hk, D).transpose(1, 2), cos, sin, positions=pos).transpose(1, 2)
    want_k, want_v = k.clone(), v.clone()
    for b in range(c.B):
        real = (tree.depths[b] >= 0).cpu()
        at = c.slots(b)[c.bases[b]:][real].to(DEV)
        want_k.view(-1, c.Hk, D)[at] = k_rot[b][real.to(DEV)]
        want_v.view(-1, c.Hk, D)[at] = vn.view(c.B, N, c.Hk, D)[b][real.to(DEV)]
    want = tree_attention(q_rot, want_k, want_v, bt, lens, tree.mask)
    out = tree_attention(q, k, v, bt, lens, tree.mask, rope=(cos, sin), depths=tree.depths, new_kv=(kn, vn))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert torch.equal(out, want)
    # without rope
    k2, v2 = (t.to(DEV) for t in (c.k, c.v))
    plain = tree_attention(q_rot, k2, v2, bt, lens, tree.mask, new_kv=(k_rot.reshape(-1, c.Hk, D), vn))
    assert torch.equal(k2, want_k) and torch.equal(v2, want_v) and torch.equal(plain, want)


def test_positions_outside_the_tables():
    c = Case([20], 6, 64, torch.float16, seed=13)
    c.parents = [[-1, 0, 1, 2, 0, 4]]
    tree = c.tree()
    cos, sin = (t.to(DEV) for t in build_rope_cache(22, 64))  # positions 20 and 21: depths 0 and 1
    q, k, v, bt, lens = c.device()
    new = (torch.ones(6, 2, 64, dtype=q.dtype, device=DEV),) * 2
    before = k.clone()
    out = tree_attention(q, k, v, bt, lens, tree.mask, rope=(cos, sin), depths=tree.depths, new_kv=new)
    deep = torch.tensor([0, 0, 1, 1, 0, 1], dtype=torch.bool, device=DEV)
    assert torch.isnan(out[0][:, deep].float()).all() and torch.isfinite(out[0][:, ~deep].float()).all()
    at = c.slots(0)[20:].to(DEV)
    assert torch.equal(k.view(-1, 2, 64)[at[deep]], before.view(-1, 2, 64)[at[deep]])


def test_depths_of_any_value():
    # a depth below 0 counts as 0; one that takes the position past the tables, or past 31 bits, makes a NaN row
    c = Case([20], 6, 64, torch.float16, seed=15)
    c.parents = [[-1, 0, 1, 2, 0, 4]]
    tree = c.tree()
    cos, sin = (t.to(DEV) for t in build_rope_cache(22, 64))
    q, k, v, bt, lens = c.device()
    new = (torch.ones(6, 2, 64, dtype=q.dtype, device=DEV),) * 2
    before = k.clone()
    depths = torch.tensor([[-5, 1, 2 ** 31 - 1, 2 ** 31 - 21, -2 ** 31, 2]], dtype=torch.int32, device=DEV)
    out = tree_attention(q, k, v, bt, lens, tree.mask, rope=(cos, sin), depths=depths, new_kv=new)
    deep = torch.tensor([0, 0, 1, 1, 0, 1], dtype=torch.bool, device=DEV)
    assert torch.isnan(out[0][:, deep].float()).all()
    at = c.slots(0)[20:].to(DEV)
    assert torch.equal(k.view(-1, 2, 64)[at[deep]], before.view(-1, 2, 64)[at[deep]])
    same = tree_attention(q, before, v.clone(), bt, lens, tree.mask, rope=(cos, sin), new_kv=new,
                          depths=torch.tensor([[0, 1, 30, 30, 0, 30]], dtype=torch.int32, device=DEV))
    assert torch.equal(out.isnan(), same.isnan()) and torch.equal(out.nan_to_num(), same.nan_to_num())


def test_append_leaves_other_rows_and_invalid_sequences():
    c = Case([10, 30], 5, 32, torch.float16, seed=14, nodes=[3, 5])
    q, k, v, bt, lens = c.device()
    bt[1, 2] = -1  # positions 32 ..: the nodes 2, 3, 4 of sequence 1
    k0, v0 = k.clone(), v.clone()
    new = tuple(torch.randn(10, 2, 32, device=DEV).to(q.dtype) for _ in range(2))
    out = tree_attention(q, k, v, bt, lens, c.tree().mask, new_kv=new)
    assert torch.isnan(out[1].float()).all()
    for pool, old, rows in ((k, k0, new[0]), (v, v0, new[1])):
        want = old.clone()
        want.view(-1, 2, 32)[c.slots(0)[10:13].to(DEV)] = rows[:3]
        want.view(-1, 2, 32)[c.slots(1)[30:32].to(DEV)] = rows[5:7]
        assert torch.equal(pool, want)


def test_same_bits_every_time_on_a_side_stream_and_in_a_graph():
    c = Case([700, 3000, 64], 26, 64, torch.bfloat16, seed=15, nodes=[26, 20, 1])
    q, k, v, bt, lens = c.device()
    mask = c.tree().mask
    want = tree_attention(q, k, v, bt, lens, mask)
    c.check(want.cpu())
    for _ in range(3):
        assert torch.equal(tree_attention(q, k, v, bt, lens, mask), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tree_attention(q, k, v, bt, lens, mask)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two graphs with workspaces of their own, replayed with other work between
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = tree_attention(q, k, v, bt, lens, mask)
        graphs.append((graph, o))
    for _ in range(3):
        q.normal_()
        want = tree_attention(q, k, v, bt, lens, mask)
        torch.cuda.synchronize()
        for graph, o in graphs:
            o.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for _, o in graphs)


def test_empty_calls():
    c = Case([10], 4, 64, torch.float16)
    q, k, v, bt, lens = c.device()
    assert tree_attention(q[:, :, :0], k, v, bt, lens, torch.zeros((1, 0, 0), dtype=torch.int32, device=DEV)).numel() == 0
    assert tree_attention(q[:0], k, v, bt[:0], lens[:0], c.tree().mask[:0]).shape[0] == 0
    assert tree_workspace_bytes(0, 8, 2, 4, 64, 16, 8) == 0


def test_refusals():
    c = Case([10, 20], 4, 64, torch.float16)
    q, k, v, bt, lens = c.device()
    mask = c.tree().mask
    cos, sin = (t.to(DEV) for t in build_rope_cache(64, 64))
    new = (torch.zeros(8, 2, 64, dtype=q.dtype, device=DEV),) * 2
    bad = [
        (RuntimeError, lambda: tree_attention(q.cpu(), k, v, bt, lens, mask)),
        (RuntimeError, lambda: tree_attention(q, k, v, bt, lens, mask.cpu())),
        (ValueError, lambda: tree_attention(q.float(), k, v, bt, lens, mask)),
        (ValueError, lambda: tree_attention(q.bfloat16(), k, v, bt, lens, mask)),
        (ValueError, lambda: tree_attention(q[..., :48], k, v, bt, lens, mask)),
        (ValueError, lambda: tree_attention(q[:, :7], k, v, bt, lens, mask)),
        (ValueError, lambda: tree_attention(q, k, v[:-1], bt, lens, mask)),
        (ValueError, lambda: tree_attention(q, k, v, bt[:1], lens, mask)),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens[:1], mask)),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens, mask.long())),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens, mask[:, :3])),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens, mask, scale=float("nan"))),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens, mask, rope=(cos, sin))),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens, mask, rope=(cos[:, :8], sin[:, :8]),
                                            depths=torch.zeros(4, dtype=torch.int32, device=DEV))),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens, mask, rope=(cos, sin),
                                            depths=torch.zeros(4, dtype=torch.int64, device=DEV))),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens, mask, new_kv=(new[0][:7], new[1]))),
        (ValueError, lambda: tree_attention(q, k.transpose(0, 1).contiguous().transpose(0, 1)[..., ::2], v[..., ::2], bt,
                                            lens, mask, new_kv=new)),
        (ValueError, lambda: tree_attention(q, k, v, bt, lens, mask, out=torch.empty(2, 8, 4, 32, device=DEV))),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    big = torch.zeros(1, 2, 1025, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="1024"):
        tree_attention(big, k, v, torch.zeros(1, 200, dtype=torch.int32, device=DEV),
                       torch.tensor([1100], dtype=torch.int32, device=DEV),
                       torch.zeros(1, 1025, 33, dtype=torch.int32, device=DEV))
