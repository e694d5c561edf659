"""Draft trees on the GPU: masks, verification of the drafted tokens and the
move of the accepted path, against the 64-bit oracle (all results are whole
numbers or copies: equal), and a run of a whole speculative step."""

from __future__ import annotations

import random

import pytest
import torch

from engine.cache import KVCacheConfig, PagedKVCache, kv_keep
from engine.decode import accept_draft, draft_tree, verify_draft, verify_greedy
from engine.model import attention_section, tree_section
from engine.model.rope import build_rope_cache
from oracle import keep_ref, mask_words, tree_ref, verify_ref
from test_tree_gpu import random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


# --- masks --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("N", [1, 2, 31, 32, 33, 64, 65, 100, 1000, 1024])
def test_masks(N):
    r = random.Random(N)
    chain = list(range(-1, N - 1))
    star = [-1] + [0] * (N - 1)
    rows = [chain, star] + [random_tree(r, r.randint(0, N), N) for _ in range(3)]
    tree = draft_tree(dev(rows))
    for b, parents in enumerate(rows):
        seen, depths = tree_ref(parents)
        assert tree.depths[b].tolist() == depths
        assert torch.equal(tree.mask[b].cpu(), mask_words(seen))
    one = draft_tree(dev(rows[2], torch.int64))
    assert torch.equal(one.mask, tree.mask[2]) and torch.equal(one.depths, tree.depths[2])


def test_masks_of_broken_trees():
    rows = [[-1, 1, 1, 5, 0, -1], [-2, 0, -1, 2, 3, -5], [3, 0, 1, -1, 3, 4], [-1, 0, 1, 2, 3, 2 ** 31 - 1]]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    tree = draft_tree(dev(rows), status=status)
    for b, parents in enumerate(rows):
        seen, depths = tree_ref(parents)
        assert tree.depths[b].tolist() == depths
        assert torch.equal(tree.mask[b].cpu(), mask_words(seen))
    assert int(status) == 1
    status.zero_()
    draft_tree(dev([[-1, 0, -2]]), status=status)
    assert int(status) == 0


# --- verification -------------------------------------------------------------------------------------------------


def check_verify(target, tokens, parents, u=None, draft=None, mode="greedy", **kw):
    """On the GPU against the oracle; target / draft CPU tensors (B, N, V)."""
    B, N, V = target.shape
    t = target.to(DEV) if not kw.get("view") else kw["view"](target)
    d = None if draft is None else draft.to(DEV) if not kw.get("view") else kw["view"](draft)
    x = dev(tokens, kw.get("token_dtype", torch.int64))
    if mode == "greedy":
        got = verify_greedy(t, x, dev(parents))
    else:
        uu = dev(u, kw.get("u_dtype", torch.float32))
        got = verify_draft(t, x, dev(parents), uu, d, replacement=mode == "iid")
        u = uu.double().tolist()
    assert got.tokens.dtype == x.dtype and got.path.dtype == torch.int32 and got.counts.dtype == torch.int32
    for b in range(B):
        path, out = verify_ref(target[b], tokens[b], parents[b], None if mode == "greedy" else u[b],
                               None if draft is None else draft[b], mode)
        n = len(path)
        assert got.counts[b].item() == n, (b, got.path[b].tolist(), path)
        assert got.path[b].tolist() == path + [-1] * (N - n), b
        assert got.tokens[b].tolist() == out + [-1] * (N - n), b
    return got


def make(B, N, V, dtype, mode, seed, shape="random", sharp=2.0):
    r = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    parents = [list(range(-1, N - 1)) if shape == "chain" else random_tree(r, N, N) for _ in range(B)]
    t = torch.randn(B, N, V, generator=g) * sharp
    d = t + torch.randn(B, N, V, generator=g) * 0.7
    if mode == "greedy":
        target, draft, pick = t.to(dtype), None, d.argsort(-1, descending=True)
    else:
        target, draft = torch.softmax(t, -1).to(dtype), torch.softmax(d, -1).to(dtype)
        pick = d.argsort(-1, descending=True)
    tokens = []
    for b in range(B):
        row = [0]
        for i in range(1, N):
            p = max(parents[b][i], 0)
            k = parents[b][:i].count(parents[b][i])
            row.append(int(pick[b, p, min(k if r.random() < 0.8 else r.randrange(V), V - 1)]))
        tokens.append(row)
    u = [[r.random() for _ in range(N)] for _ in range(B)]
    return target, tokens, parents, u, (draft if mode in ("iid", "tree") else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mode", ["greedy", "picks", "iid", "tree"])
@pytest.mark.parametrize("B,N,V,shape", [(1, 1, 5, "random"), (3, 5, 1, "chain"), (2, 6, 2, "random"),
                                         (4, 5, 63, "chain"), (5, 26, 1000, "random"), (2, 64, 4099, "random"),
                                         (2, 9, 32001, "random"), (1, 200, 777, "random")])
def test_verify(B, N, V, shape, mode, dtype):
    target, tokens, parents, u, draft = make(B, N, V, dtype, mode, seed=N + V, shape=shape)
    check_verify(target, tokens, parents, u, draft, mode)


@pytest.mark.parametrize("mode", ["greedy", "picks", "iid", "tree"])
def test_verify_large_vocabulary_and_many_draws(mode):
    target, tokens, parents, u, draft = make(6, 12, 140001, torch.float32, mode, seed=3, sharp=3.0)
    check_verify(target, tokens, parents, u, draft, mode)


@pytest.mark.parametrize("mode", ["picks", "iid", "tree"])
def test_verify_many_small(mode):
    target, tokens, parents, u, draft = make(300, 10, 40, torch.float32, mode, seed=8, sharp=1.0)
    got = check_verify(target, tokens, parents, u, draft, mode)
    assert len(set(got.counts.tolist())) > 2  # some rejected at once, some accepted


@pytest.mark.parametrize("mode", ["greedy", "tree"])
def test_verify_types_and_strides(mode):
    target, tokens, parents, u, draft = make(3, 7, 501, torch.float16, mode, seed=4)

    def padded(x):  # rows inside a wider tensor, at an odd offset
        wide = torch.full((3, 9, 530), float("nan"), dtype=x.dtype, device=DEV)
        wide[:, 1:8, 3:504] = x.to(DEV)
        return wide[:, 1:8, 3:504]

    def turned(x):  # a vocabulary stride other than 1: copied
        return x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)

    for view in (padded, turned):
        for td in (torch.int32, torch.int64):
            for ud in (torch.float32, torch.float64):
                check_verify(target, tokens, parents, u, draft, mode, view=view, token_dtype=td, u_dtype=ud)


def test_verify_parents_shared():
    target, tokens, parents, u, draft = make(4, 9, 100, torch.float32, "tree", seed=5)
    parents = [parents[0]] * 4
    args = target.to(DEV), dev(tokens, torch.int64)
    a = verify_draft(*args, dev(parents[0]), dev(u, torch.float32), draft.to(DEV))
    b = verify_draft(*args, dev(parents), dev(u, torch.float32), draft.to(DEV))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("mode", ["greedy", "picks", "iid", "tree"])
def test_verify_padding_broken_nodes_and_foreign_tokens(mode):
    target, tokens, parents, u, draft = make(5, 12, 50, torch.float32, mode, seed=6)
    parents[0] = [-2] * 12                                      # no sequence
    parents[1] = [-1, 0, 0, -2, 3, 1, 9, 5, -1, 8, 7, 2 ** 31 - 1]  # a slot, a second root, parents behind their child
    tokens[2][1:5] = [50, -1, 2 ** 31 - 1, -2 ** 31]            # outside the vocabulary
    parents[3] = [0] + parents[3][1:]                           # node 0 with a parent: no sequence
    check_verify(target, tokens, parents, u, draft, mode)


def test_verify_edges_of_the_rule():
    V, N = 8, 5
    one_hot = torch.eye(V)
    flat = torch.full((V,), 1 / V)
    star, chain = [-1, 0, 0, 0, 0], [-1, 0, 1, 2, 3]
    top = 1 - 2.0 ** -24
    cases = [
        # p == q: never rejected but at u = 1 - 2^-24, where nothing is left of p - q and p stays
        (flat.expand(N, V), [0, 1, 2, 3, 4], chain, [0.3, 0.99, 0.5, 0.0, 0.7], flat.expand(N, V)),
        (flat.expand(N, V), [0, 1, 2, 3, 4], star, [top, 1.0, 1.0, 1.0, 1.0], flat.expand(N, V)),
        # the target never says the drafts' tokens; u = 0
        (one_hot[7].expand(N, V), [0, 1, 2, 3, 4], star, [0.0, 0.0, 0.0, 0.0, 0.0], flat.expand(N, V)),
        (one_hot[0].expand(N, V), [0, 1, 2, 3, 4], star, [top, 0.5, 0.5, 0.5, 0.5], flat.expand(N, V)),
        # the same token twice among the children, tokens the draft gives no weight
        (flat.expand(N, V), [0, 3, 3, 3, 5], star, [0.4, 0.9, 0.9, 0.9, 0.9], one_hot[3].expand(N, V)),
        (flat.expand(N, V), [0, 4, 4, 2, 5], star, [0.4, 0.0, 0.9, 0.0, 0.1], one_hot[3].expand(N, V)),
        # the draft holds all its weight on a rejected token: nothing is left of q
        (one_hot[5].expand(N, V), [0, 3, 4, 5, 6], star, [0.5, 0.5, 0.5, 0.5, 0.5], one_hot[3].expand(N, V)),
        # unnormalised rows, and a row of zeros
        ((flat * 3).expand(N, V), [0, 1, 2, 3, 4], star, [0.9, 0.99, 0.99, 0.99, 0.99], (flat * 5).expand(N, V)),
        (torch.zeros(N, V), [0, 1, 2, 3, 4], star, [0.5, 0.5, 0.5, 0.5, 0.5], flat.expand(N, V)),
    ]
    for target, tokens, parents, u, draft in cases:
        for mode in ("picks", "iid", "tree"):
            check_verify(target.clone().unsqueeze(0), [tokens], [parents], [u],
                         None if mode == "picks" else draft.clone().unsqueeze(0), mode, u_dtype=torch.float64)


def test_picks_with_almost_all_mass_removed():
    # the children hold all but a sliver of the mass
    V, N = 3000, 4
    p = torch.full((V,), 1e-9)
    p[[10, 1500, 2999]] = torch.tensor([0.7, 0.2, 0.1 - 3e-6])
    for u0 in (0.0, 0.25, 0.5, 0.999):
        check_verify(p.expand(1, N, V).clone(), [[0, 10, 1500, 2999]], [[-1, 0, 0, 0]], [[u0, 1.0, 1.0, 1.0]], None,
                     "picks", u_dtype=torch.float64)


def test_greedy_ties_infinities_and_nan():
    V, N = 300, 3
    rows = torch.zeros(6, N, V)
    rows[0, :, [7, 200]] = 2.0                 # a tie
    rows[1] = -0.0
    rows[1, :, 5] = 0.0                        # signed zeros are equal
    rows[2, :, 250] = float("inf")
    rows[3] = float("-inf")
    rows[4, :, 9], rows[4, :, 2] = float("nan"), 100.0
    rows[5] = -torch.arange(V).float() - 1
    tokens = [[0, 7, 7], [0, 0, 0], [0, 250, 1], [0, 0, 1], [0, 9, 2], [0, 0, 0]]
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        check_verify(rows.to(dtype), tokens, [[-1, 0, 1]] * 6, mode="greedy")


@pytest.mark.parametrize("V", [1, 2, 3, 4, 7, 8, 9, 15, 17, 511, 513, 1025, 8191, 8200, 33000])
def test_greedy_finds_every_place(V):
    # the largest at chosen places, on a floor of -inf, of equal values, and NaN of either sign
    places = sorted({0, 1, 3, 7, 8, V // 2, V - 9, V - 8, V - 2, V - 1} & set(range(V)))
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        rows = torch.full((4 * len(places), 2, V), float("-inf"))
        for k, at in enumerate(places):
            rows[4 * k, :, at] = -3.0
            rows[4 * k + 1] = -1.0
            rows[4 * k + 1, :, at:] = 1.5
            rows[4 * k + 2] = float("inf")
            rows[4 * k + 2, :, at] = float("nan")
            rows[4 * k + 3] = -0.0
            rows[4 * k + 3, :, :at] = -5.0
            rows[4 * k + 3, :, V - 1] = 0.0
        logits = rows.to(dtype)
        logits[2::4] = logits[2::4] * -1 if V % 2 else logits[2::4]  # (-inf around it, and NaN's sign turned)
        check_verify(logits, [[0, at] for at in places for _ in range(4)], [[-1, 0]] * len(rows))


@pytest.mark.parametrize("B,N,V,dtype", [(2, 300, 60001, torch.float16), (3, 20, 300000, torch.float32),
                                         (2, 300, 50001, torch.bfloat16)])
def test_greedy_of_many_rows(B, N, V, dtype):
    # the first two read their rows on the walk (over 64 MiB of logits), the last one reads all of them first
    r = random.Random(V)
    logits = torch.randn((B, N, V), generator=torch.Generator(DEV).manual_seed(V), device=DEV).to(dtype).cpu()
    parents = [random_tree(r, N, N) for _ in range(B)]
    best = [[int((row == row.max()).nonzero()[0]) for row in seq] for seq in logits]
    tokens = [[0] + [best[b][max(parents[b][i], 0)] if r.random() < 0.7 else r.randrange(V) for i in range(1, N)]
              for b in range(B)]
    got = check_verify(logits, tokens, parents)
    assert max(got.counts.tolist()) > 2


@pytest.mark.parametrize("mode", ["picks", "iid", "tree"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_verify_parts_of_the_vocabulary(mode, dtype):
    # parts of more than one block, a last one that is full, that is short, that is one token
    for V in (4096, 4097, 65536, 135168, 270001):
        target, tokens, parents, u, draft = make(3, 6, V, dtype, mode, seed=V, sharp=1.0)
        for u0 in (0.001, 0.5, 0.9999):
            check_verify(target, tokens, parents, [[u0] + [0.99] * 3 + row[4:] for row in u], draft, mode)


def test_sampling_is_the_targets():
    """The first emitted token over many draws is distributed as the target's
    at node 0, whatever the draft: within five standard deviations of every
    bin's binomial count."""
    B, V, k = 40000, 12, 3
    g = torch.Generator(DEV).manual_seed(1)
    p = torch.softmax(torch.randn(V, generator=g, device=DEV) * 1.5, 0)
    q = torch.softmax(torch.randn(V, generator=g, device=DEV) * 1.5, 0)
    parents = dev([[-1] + [0] * k]).expand(B, k + 1).contiguous()
    u = torch.rand((B, k + 1), generator=g, device=DEV)
    target, draft = p.expand(B, k + 1, V), q.expand(B, k + 1, V)
    for replacement in (False, True):
        kids = torch.multinomial(q.expand(B, V), k, replacement=replacement, generator=g)
        tokens = torch.cat([torch.zeros((B, 1), dtype=torch.int64, device=DEV), kids], 1)
        got = verify_draft(target, tokens, parents, u, draft, replacement=replacement)
        n = torch.bincount(got.tokens[:, 0], minlength=V).double()
        dev_n = (B * p.double() * (1 - p.double())).sqrt()
        assert float(((n - B * p.double()).abs() / dev_n).max()) < 5


def test_verify_in_a_graph_and_on_a_side_stream():
    target, tokens, parents, u, draft = make(4, 20, 3001, torch.float32, "tree", seed=9)
    t, d, x, p = target.to(DEV), draft.to(DEV), dev(tokens, torch.int64), dev(parents)
    uu = dev(u, torch.float32)
    graph = torch.cuda.CUDAGraph()
    verify_draft(t, x, p, uu, d)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = verify_draft(t, x, p, uu, d)
        tree = draft_tree(p)
        greedy = verify_greedy(t, x, p)
    for seed in range(3):
        uu.uniform_(generator=torch.Generator(DEV).manual_seed(seed))
        want = verify_draft(t, x, p, uu, d)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(tree.mask, draft_tree(p).mask)
    assert all(torch.equal(a, b) for a, b in zip(greedy, verify_greedy(t, x, p)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = verify_draft(t, x, p, uu, d)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_greedy_in_two_graphs_and_on_two_streams():
    # each call has its own workspace: graphs replayed in turn and calls on two streams at once do not meet in it
    r = random.Random(2)
    trees = [[random_tree(r, 30, 30) for _ in range(3)] for _ in range(2)]
    logits = [torch.randn((3, 30, 5000), device=DEV) for _ in range(2)]
    tokens = [torch.zeros((3, 30), dtype=torch.int64, device=DEV) for _ in range(2)]
    p = [dev(t) for t in trees]
    up = [x.clamp(min=0).long() for x in p]

    def refill(seed):
        g = torch.Generator(DEV).manual_seed(seed)
        for i in range(2):
            logits[i].normal_(generator=g)
            tokens[i].copy_(logits[i].argmax(-1).gather(1, up[i]))  # every child right: whole chains pass

    refill(0)
    verify_greedy(logits[0], tokens[0], p[0])
    torch.cuda.synchronize()
    graphs, got = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            got.append(verify_greedy(logits[i], tokens[i], p[i]))
    for seed in range(1, 4):
        refill(seed)
        want = [verify_greedy(logits[i], tokens[i], p[i]) for i in range(2)]
        torch.cuda.synchronize()
        for i in (0, 1, 0, 1):
            graphs[i].replay()
        torch.cuda.synchronize()
        side = [torch.cuda.Stream() for _ in range(2)]
        both = []
        for i in range(2):
            with torch.cuda.stream(side[i]):
                both.append([verify_greedy(logits[i], tokens[i], p[i]) for _ in range(5)])
        torch.cuda.synchronize()
        for i in range(2):
            assert max(want[i].counts.tolist()) > 3
            for other in [got[i], *both[i]]:
                assert all(torch.equal(a, b) for a, b in zip(want[i], other))


def test_verify_refusals_and_empty():
    target, tokens, parents, u, draft = make(2, 5, 30, torch.float32, "tree", seed=1)
    t, d, x, p, uu = target.to(DEV), draft.to(DEV), dev(tokens, torch.int64), dev(parents), dev(u, torch.float32)
    bad = [
        (RuntimeError, lambda: verify_draft(target, x, p, uu, d)),
        (RuntimeError, lambda: verify_draft(t, x.cpu(), p, uu, d)),
        (RuntimeError, lambda: verify_greedy(t, x, p.cpu())),
        (ValueError, lambda: verify_draft(t.double(), x, p, uu)),
        (ValueError, lambda: verify_draft(t[0], x, p, uu)),
        (ValueError, lambda: verify_draft(t, x.float(), p, uu)),
        (ValueError, lambda: verify_draft(t, x[:, :4], p, uu)),
        (ValueError, lambda: verify_draft(t, x, p[:1], uu)),
        (ValueError, lambda: verify_draft(t, x, p.float(), uu)),
        (ValueError, lambda: verify_draft(t, x, p, uu.half())),
        (ValueError, lambda: verify_draft(t, x, p, uu[:, :4])),
        (ValueError, lambda: verify_draft(t, x, p, None, d)),
        (ValueError, lambda: verify_draft(t, x, p, uu, d.half())),
        (ValueError, lambda: verify_draft(t, x, p, uu, d[..., :29])),
        (ValueError, lambda: verify_greedy(t[..., :0], x, p)),
        (ValueError, lambda: draft_tree(dev([[0.0]], torch.float32))),
        (ValueError, lambda: draft_tree(torch.zeros((1, 1025), dtype=torch.int32, device=DEV))),
        (RuntimeError, lambda: draft_tree(torch.zeros((1, 4), dtype=torch.int32))),
        (ValueError, lambda: accept_draft(None, None, p, x, t, None, d)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    assert verify_greedy(t[:0], x[:0], p[:0]).counts.shape == (0,)
    assert verify_greedy(t[:, :0], x[:, :0], p[:, :0]).path.shape == (2, 0)
    assert draft_tree(torch.zeros((0, 4), dtype=torch.int32, device=DEV)).mask.shape == (0, 4, 1)


# --- keeping the accepted path ------------------------------------------------------------------------------------


def make_pools(layers, blocks, bs, Hk, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [[torch.randn(blocks, bs, Hk, D, generator=g).to(dtype) for _ in range(layers)] for _ in range(2)]


@pytest.mark.parametrize("layers,Hk,D,bs,N", [(1, 1, 16, 16, 2), (3, 2, 64, 3, 30), (2, 8, 128, 16, 100),
                                              (70, 1, 32, 16, 12), (1, 3, 256, 1, 40), (1, 2, 64, 16, 1024)])
def test_keep(layers, Hk, D, bs, N):
    r = random.Random(N)
    dtype = torch.bfloat16 if layers % 2 else torch.float16
    starts = [0, 5, 37, 100]
    need = [-(-(s + N) // bs) for s in starts]
    ids = list(range(sum(need)))
    r.shuffle(ids)
    bt = torch.zeros(4, max(need), dtype=torch.int32)
    blocks, at = [], 0
    for b, n in enumerate(need):
        blocks.append(ids[at:at + n])
        bt[b, :n] = torch.tensor(blocks[b], dtype=torch.int32)
        at += n
    # overlapping moves among them: dense rising paths, the whole tree, nothing
    paths = [[0] + sorted(r.sample(range(1, N), min(N - 1, 9))), list(range(N)), [],
             [0] + sorted(r.sample(range(1, N), (N - 1) * 4 // 5))]
    ks, vs = make_pools(layers, len(ids), bs, Hk, D, dtype, seed=N)
    kd, vd = [t.to(DEV) for t in ks], [t.to(DEV) for t in vs]
    path = dev([p + [-1] * (N - len(p)) for p in paths])
    kv_keep(kd, vd, bt.to(DEV), dev(starts), path, dev([len(p) for p in paths]))
    for pools, got in ((ks, kd), (vs, vd)):
        for t, g in zip(pools, got):
            for b in range(4):
                keep_ref(t, blocks[b], starts[b], paths[b])
            assert torch.equal(g.cpu(), t)


def test_keep_ignores_what_is_out_of_range_and_takes_views():
    ks, vs = make_pools(2, 6, 4, 2, 32, torch.float16, seed=2)
    wide = [torch.zeros(6, 4, 2, 2, 32, dtype=torch.float16, device=DEV) for _ in range(2)]
    for l in range(2):
        wide[l][:, :, 0], wide[l][:, :, 1] = ks[l].to(DEV), vs[l].to(DEV)
    kd, vd = [w[:, :, 0] for w in wide], [w[:, :, 1] for w in wide]
    # sequence 0: node 3 (position 5) goes to position 3, nodes 9 and 4 are past N; 1: nodes past N or below j, a count
    # past N; 2: node 2 lies in block -1; 3: a negative start
    bt = dev([[0, 1, 9], [3, 4, 5], [2, -1, 2], [0, 0, 0]])
    path = dev([[0, 3, 9, 4], [0, 5, 200, 1], [0, 2, 4, 7], [0, 2, 3, 7]])
    kv_keep(tuple(kd), vd, bt, dev([2, 1, 3, -4], torch.int64), path, dev([4, 9, 4, 4]))
    for l in range(2):
        for got, src in ((kd[l].cpu(), ks[l]), (vd[l].cpu(), vs[l])):
            want = src.clone()
            want[0, 3] = src[1, 1]
            assert torch.equal(got, want)


def test_keep_refusals():
    ks, vs = make_pools(2, 4, 4, 1, 32, torch.float16, seed=1)
    kd, vd = [t.to(DEV) for t in ks], [t.to(DEV) for t in vs]
    bt, st, pa, cn = dev([[0, 1]]), dev([0]), dev([[0, 2]]), dev([2])
    bad = [
        (ValueError, lambda: kv_keep(kd, vd[:1], bt, st, pa, cn)),
        (ValueError, lambda: kv_keep(kd, [vd[0], vd[1].bfloat16()], bt, st, pa, cn)),
        (ValueError, lambda: kv_keep([t.float() for t in kd], [t.float() for t in vd], bt, st, pa, cn)),
        (ValueError, lambda: kv_keep([kd[0], kd[1][:3]], vd, bt, st, pa, cn)),
        (ValueError, lambda: kv_keep([kd[0], kd[1].transpose(0, 1)], vd, bt, st, pa, cn)),
        (ValueError, lambda: kv_keep(kd, vd, bt, st, pa[0], cn)),
        (ValueError, lambda: kv_keep(kd, vd, bt, st, pa.float(), cn)),
        (ValueError, lambda: kv_keep(kd, vd, bt, st, pa, dev([2, 2]))),
        (ValueError, lambda: kv_keep(kd, vd, bt, st, torch.zeros((1, 1025), dtype=torch.int32, device=DEV), cn)),
        (RuntimeError, lambda: kv_keep(kd, vd, bt.cpu(), st, pa, cn)),
        (RuntimeError, lambda: kv_keep(kd, vs, bt, st, pa, cn)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    kv_keep([], [], bt, st, pa, cn)
    kv_keep(kd, vd, bt[:0], st[:0], pa[:0], cn[:0])
    assert all(torch.equal(a.cpu(), b) for a, b in zip(kd + vd, ks + vs))


# --- a whole step -------------------------------------------------------------------------------------------------


class Toy:
    """A small model whose logits follow from the attention outputs: embeddings,
    two attention layers with rotary embedding, a head. ``step`` runs L tokens of
    every sequence, as a chain or a tree."""

    def __init__(self, seed=0, Hq=4, Hk=2, D=64, V=97, layers=2):
        g = torch.Generator().manual_seed(seed)
        self.Hq, self.Hk, self.D, self.V, self.layers = Hq, Hk, D, V, layers
        w = Hq * D
        mk = lambda *s: (torch.randn(*s, generator=g) / s[-1] ** 0.5).to(DEV)  # noqa: E731
        self.emb = torch.randn(V, w, generator=g).to(DEV)
        self.wq = [mk(w, w) for _ in range(layers)]
        self.wkv = [(mk(Hk * D, w), mk(Hk * D, w)) for _ in range(layers)]
        self.wo = [mk(w, w) for _ in range(layers)]
        self.head = mk(V, w) * 4
        self.rope = tuple(t.to(DEV) for t in build_rope_cache(512, D))

    def cache(self):
        return PagedKVCache(KVCacheConfig(num_layers=self.layers, num_kv_heads=self.Hk, head_dim=self.D, num_blocks=64,
                                          block_size=16, dtype=torch.float16, device=DEV))

    def step(self, cache, step, tokens, tree=None):
        B, L = tokens.shape
        x = self.emb[tokens]
        for i in range(self.layers):
            h = x / x.pow(2).mean(-1, keepdim=True).sqrt()
            q = (h @ self.wq[i].t()).half().view(B, L, self.Hq, self.D).transpose(1, 2)
            k, v = ((h @ w.t()).half().view(B, L, self.Hk, self.D).transpose(1, 2) for w in self.wkv[i])
            if tree is None:
                o = attention_section(q, k, v, i, cache, step, rope=self.rope)
            else:
                o = tree_section(q, k, v, i, cache, step, tree, rope=self.rope)
            x = x + o.float() @ self.wo[i].t()
        return x @ self.head.t()


def test_greedy_trees_decode_the_same_tokens():
    """Speculative decoding with greedy trees emits the tokens of plain greedy
    decoding; half of the drafted children are right on purpose."""
    model, B, prompt_len, want_len = Toy(), 2, 9, 14
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, model.V, (B, prompt_len), generator=g).to(DEV)
    # plain greedy decoding
    cache = model.cache()
    tables = [cache.new_sequence() for _ in range(B)]
    logits = model.step(cache, cache.prepare_step(tables, prompt_len), prompt)[:, -1]
    plain = [logits.argmax(-1)]
    margins = []
    while len(plain) < want_len + 6:
        logits = model.step(cache, cache.prepare_step(tables, 1), plain[-1].unsqueeze(1))[:, -1]
        top = logits.topk(2).values
        margins.append(float((top[:, 0] - top[:, 1]).min()))
        plain.append(logits.argmax(-1))
    plain = torch.stack(plain, 1).tolist()
    assert min(margins) > 0.02  # the two paths' 16-bit roundings cannot change an argmax
    # trees: node 0, two children of it, two of the first, one of the second child of that
    shape = [-1, 0, 0, 1, 1, 4, -2]
    r = random.Random(4)
    cache = model.cache()
    tables = [cache.new_sequence() for _ in range(B)]
    logits = model.step(cache, cache.prepare_step(tables, prompt_len), prompt)[:, -1]
    out = [[int(t)] for t in logits.argmax(-1)]
    parents = dev([shape] * B)
    accepted = 0
    while min(len(o) for o in out) < want_len:
        rows = []
        for b in range(B):
            nxt = plain[b][len(out[b]):] + [0, 0, 0]
            row = [out[b][-1]] + [r.randrange(model.V) for _ in range(6)]
            row[r.choice((1, 2))] = nxt[0]
            row[r.choice((3, 4))] = nxt[1]
            row[5] = nxt[2]
            rows.append(row)
        tokens = dev(rows, torch.int64)
        step = cache.prepare_step(tables, len(shape))
        tree = draft_tree(parents)
        logits = model.step(cache, step, tokens, tree)
        done = accept_draft(cache, step, parents, tokens, logits)
        counts = done.counts.tolist()
        cache.rollback_step(step, counts)
        for b, n in enumerate(counts):
            out[b] += done.tokens[b, :n].tolist()
            accepted += n - 1
        assert [t.length for t in tables] == [prompt_len + len(o) - 1 for o in out]
    assert accepted > 4
    for b in range(B):
        assert out[b][:want_len] == plain[b][:want_len]
    # what the cache holds is what plain decoding of the same tokens leaves there (kept rows were rotated at their depth)
    again = model.cache()
    t2 = [again.new_sequence() for _ in range(B)]
    for b in range(B):
        text = torch.cat([prompt[b], dev(out[b][:-1], torch.int64)]).unsqueeze(0)
        model.step(again, again.prepare_step([t2[b]], text.shape[1]), text)
        for layer in range(model.layers):
            for x, y in zip(cache.gather(layer, tables[b]), again.gather(layer, t2[b])):
                assert float((x.float() - y.float()).abs().max()) < 0.02 * float(y.abs().max())


def test_step_errors():
    model = Toy()
    cache = model.cache()
    table = cache.new_sequence()
    step = cache.prepare_step([table], 4)
    q = torch.zeros(1, 4, 3, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError):
        tree_section(q, q[:, :2], q[:, :2], 0, cache, step, draft_tree(dev([[-1, 0, 0]])))
    for counts in ([5], [-1], [1, 1]):
        with pytest.raises(ValueError):
            cache.rollback_step(step, counts)
    cache.rollback_step(step, [2])
    assert table.length == 2
