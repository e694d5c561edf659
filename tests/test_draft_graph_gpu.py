"""A whole step of draft trees captured in one HIP graph: ``draft_tree``, every
layer's ``tree_section`` with rotary embedding and append, and ``accept_draft``.
Every replay, with other trees, tokens, rows and longer histories copied into
the captured tensors and the program's own eager work between replays, must
equal the eager calls bit for bit, the pools included."""

from __future__ import annotations

import random

import pytest
import torch

from engine.cache import KVCacheConfig, PagedKVCache
from engine.decode import accept_draft, draft_tree
from engine.model import tree_section
from engine.model.rope import build_rope_cache
from test_tree_gpu import DEV, random_tree

pytestmark = pytest.mark.gpu

B, N, HQ, HK, D, LAYERS, V, BLOCKS = 3, 9, 8, 2, 64, 2, 300, 40


class Program:
    """Static buffers of a serving loop and its step."""

    def __init__(self, sampled):
        self.sampled = sampled
        self.cache = PagedKVCache(KVCacheConfig(num_layers=LAYERS, num_kv_heads=HK, head_dim=D, num_blocks=150,
                                                block_size=16, dtype=torch.float16, device=DEV))
        self.tables = [self.cache.new_sequence() for _ in range(B)]
        self.g = torch.Generator(DEV).manual_seed(5)
        self.grow([30, 3, 0])
        self.rope = tuple(t.to(DEV) for t in build_rope_cache(16 * BLOCKS, D))
        self.q = torch.empty(LAYERS, B, HQ, N, D, dtype=torch.float16, device=DEV)
        self.k, self.v = (torch.empty(LAYERS, B, HK, N, D, dtype=torch.float16, device=DEV) for _ in range(2))
        self.parents = torch.zeros(B, N, dtype=torch.int32, device=DEV)
        self.tokens = torch.zeros(B, N, dtype=torch.int64, device=DEV)
        self.target, self.draft = (torch.empty(B, N, V, device=DEV) for _ in range(2))
        self.u = torch.empty(B, N, device=DEV)

    def grow(self, counts):
        for t, n in zip(self.tables, counts):
            if n:
                for layer in range(LAYERS):
                    rows = [torch.randn(n, HK, D, generator=self.g, device=DEV).half() for _ in range(2)]
                    self.cache.append(layer, t, *rows, start=t.length if layer == 0 else t.length - n)

    def fill(self, seed):
        r = random.Random(seed)
        trees = [random_tree(r, r.randint(2, N), N) for _ in range(B)]
        self.parents.copy_(torch.tensor(trees, dtype=torch.int32))
        for x in (self.q, self.k, self.v):
            x.normal_(generator=self.g)
        logits = torch.randn(B, N, V, generator=self.g, device=DEV) * 3
        best = logits.argmax(-1).gather(1, self.parents.clamp(min=0).long())
        other = torch.randint(0, V, (B, N), generator=self.g, device=DEV)
        self.tokens.copy_(torch.where(torch.rand(B, N, generator=self.g, device=DEV) < 0.7, best, other))
        self.u.uniform_(generator=self.g)
        if self.sampled:
            self.target.copy_(torch.softmax(logits, -1))
            self.draft.copy_(torch.softmax(logits + torch.randn(B, N, V, generator=self.g, device=DEV), -1))
        else:
            self.target.copy_(logits)

    def run(self, step):
        tree = draft_tree(self.parents)
        outs = [tree_section(self.q[i], self.k[i], self.v[i], i, self.cache, step, tree, rope=self.rope)
                for i in range(LAYERS)]
        extra = (self.u, self.draft) if self.sampled else ()
        return outs, accept_draft(self.cache, step, self.parents, self.tokens, self.target, *extra)

    def pools(self):
        return [t.clone() for t in self.cache.k + self.cache.v]

    def restore(self, pools):
        for t, old in zip(self.cache.k + self.cache.v, pools):
            t.copy_(old)

    def next_step(self, into):
        """The next step's tables and lengths in the captured step's tensors."""
        step = self.cache.prepare_step(self.tables, N, max_blocks=BLOCKS)
        for name in ("block_tables", "context_lens", "cu_new", "starts"):
            getattr(into, name).copy_(getattr(step, name))
        return step


@pytest.mark.parametrize("sampled", [False, True])
def test_step_in_a_graph(sampled):
    p = Program(sampled)
    step = p.cache.prepare_step(p.tables, N, max_blocks=BLOCKS)  # the table's width: the longest sequence there will be
    step.max_context = 16 * BLOCKS                               # and its length, as both are part of the launches
    p.fill(0)
    _, done = p.run(step)  # warm-up outside the capture
    p.cache.rollback_step(step, done.counts.tolist())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs, done = p.run(step)
    emitted = 0
    for rep in range(5):
        if rep in (2, 3):
            p.grow([100 * rep, 17, 1])
        now = p.next_step(step)
        p.fill(rep + 1)
        before = p.pools()
        want_outs, want = p.run(step)
        want_pools = p.pools()
        p.restore(before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.isfinite(o.float()).all() for o in outs)
        assert all(torch.equal(a, b) for a, b in zip([*outs, *done], [*want_outs, *want]))
        assert all(torch.equal(a, b) for a, b in zip(p.pools(), want_pools))
        counts = done.counts.tolist()
        emitted += sum(counts) - B
        p.cache.rollback_step(now, counts)
    assert emitted > 3 and max(t.length for t in p.tables) > 500


def test_a_captured_step_is_bound_to_its_longest_length():
    # without the larger max_context a replay makes rows of longer sequences NaN, and reads nothing past it
    p = Program(False)
    step = p.cache.prepare_step(p.tables, N, max_blocks=BLOCKS)
    p.fill(0)
    _, done = p.run(step)
    p.cache.rollback_step(step, done.counts.tolist())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs, done = p.run(step)
    p.grow([200, 0, 0])
    p.next_step(step)
    p.fill(1)
    live = (p.parents >= -1).unsqueeze(-1)
    graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.isnan(o[0].float()[live[0].expand(N, HQ * D)]).all() and torch.isfinite(o[1:].float()).all()
