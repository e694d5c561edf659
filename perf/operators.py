"""The operators of speculative decoding with draft trees, as a serving program
calls them: attention of a tree of drafted tokens over the paged cache, the
verification of the drafted tokens, and the move of the accepted path's K and
V to the end of the history.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare(case, seed)`` makes what the program has in hand before the call,
``run(state)`` is one pass (the package's operators where ``own`` is true, the
same from elementary torch operations where it is false), ``work(case)`` its
unavoidable bytes and FLOPs and ``exact(case, seed)`` the outputs in 64 bits,
one sequence at a time.

A draft tree of N nodes is given by the parent of every node: node 0, the last
token the sequence has (parent -1), then drafted tokens, each after its parent;
-2 marks a padding slot of a batch. The nodes' K and V sit behind the history,
node i at position base + i, and node i sees the history and its ancestors,
itself included; its rotary position is base + its depth.

Kinds of case:

* ``attend``: ``tree_attention`` over histories and nodes already in the pool;
* ``step``: one layer of a step: ``draft_tree`` of the parents, then
  ``tree_attention`` with the rotary embedding and the append of the nodes;
* ``verify``: ``verify_draft`` of target against draft probabilities and given
  uniform numbers (``mode``: "tree" drafts without replacement, "iid" with
  replacement, "top" the draft's likeliest tokens, whose probabilities are
  not given) or ``verify_greedy`` of logits ("greedy");
* ``keep``: ``kv_keep`` of the accepted paths in every layer's pool.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
BS = 16  # tokens per KV block, the engine's default
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
NONE = 2.0 ** -40  # a residual of less mass than this counts as none


def _package():
    path = os.path.abspath("custom-inference-engine_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import engine.attention
    import engine.cache
    import engine.decode

    return engine


def listed():
    return [
        # a single user's small tree over a short history: launch and latency
        {"name": "attend_1x8", "kind": "attend", "B": 1, "N": 8, "lo": 777, "hi": 777, "Hq": 32, "Hk": 8, "D": 64,
         "dtype": "fp16", "padded": False},
        # a full batch with trees of different sizes over ragged histories
        {"name": "attend_32x16", "kind": "attend", "B": 32, "N": 16, "lo": 256, "hi": 4096, "Hq": 32, "Hk": 8,
         "D": 64, "dtype": "fp16", "padded": True},
        # large trees over long documents, the largest call
        {"name": "attend_4x64", "kind": "attend", "B": 4, "N": 64, "lo": 8192, "hi": 16384, "Hq": 32, "Hk": 8,
         "D": 128, "dtype": "bf16", "padded": False},
        # one very large tree, many query heads on few kv heads
        {"name": "attend_1x255", "kind": "attend", "B": 1, "N": 255, "lo": 4001, "hi": 4001, "Hq": 28, "Hk": 4,
         "D": 128, "dtype": "bf16", "padded": False},
        # one layer of a single user's step: pure latency
        {"name": "step_1x8", "kind": "step", "B": 1, "N": 8, "lo": 777, "hi": 777, "Hq": 32, "Hk": 8, "D": 64,
         "dtype": "fp16", "padded": False},
        # one layer of a batched step
        {"name": "step_8x26", "kind": "step", "B": 8, "N": 26, "lo": 1024, "hi": 8192, "Hq": 32, "Hk": 8, "D": 128,
         "dtype": "bf16", "padded": True},
        # the classic chain of four drafts
        {"name": "verify_chain_8x5", "kind": "verify", "mode": "iid", "tree": "chain", "B": 8, "N": 5, "V": 32000,
         "dtype": "fp32"},
        # a full batch of sampled trees over a large vocabulary
        {"name": "verify_tree_32x26", "kind": "verify", "mode": "tree", "tree": "random", "B": 32, "N": 26,
         "V": 128000, "dtype": "fp32"},
        # the draft's likeliest continuations, 16-bit probabilities, a vocabulary of odd size
        {"name": "verify_top_4x64", "kind": "verify", "mode": "top", "tree": "random", "B": 4, "N": 64, "V": 50001,
         "dtype": "bf16"},
        # greedy decoding: the target's logits
        {"name": "verify_greedy_8x26", "kind": "verify", "mode": "greedy", "tree": "random", "B": 8, "N": 26,
         "V": 128000, "dtype": "bf16"},
        # the accepted path of one sequence
        {"name": "keep_1x8", "kind": "keep", "B": 1, "N": 8, "layers": 16, "lo": 100, "hi": 100, "Hk": 8, "D": 64,
         "dtype": "fp16"},
        # and of a batch
        {"name": "keep_32x26", "kind": "keep", "B": 32, "N": 26, "layers": 32, "lo": 10, "hi": 60, "Hk": 8, "D": 128,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((32, 8), (32, 8), (16, 16), (32, 32), (28, 4), (16, 2))


def draw(rng):
    """One more case of the ranges above, no costlier than the largest."""
    while True:
        kind = rng.choice(("attend", "attend", "step", "verify", "verify", "keep"))
        c = {"kind": kind}
        if kind in ("attend", "step"):
            Hq, Hk = rng.choice(_HEADS)
            lo = _log_int(rng, 1, 8192)
            c.update(B=_log_int(rng, 1, 48), N=_log_int(rng, 1, 256), lo=lo,
                     hi=min(16384, int(lo * rng.choice((1, 2, 4, 16)))), Hq=Hq, Hk=Hk,
                     D=rng.choice((64, 64, 128, 128, 32, 256)), dtype=rng.choice(("fp16", "bf16")),
                     padded=rng.random() < 0.4)
            top = {"bytes": 400e6, "flops": 60e9}
        elif kind == "verify":
            c.update(mode=rng.choice(("tree", "iid", "top", "greedy")), tree=rng.choice(("random", "random", "chain")),
                     B=_log_int(rng, 1, 48), N=_log_int(rng, 1, 80), V=_log_int(rng, 1000, 160000),
                     dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")))
            if c["B"] * c["N"] * c["V"] > 32 * 26 * 128000:
                continue
            top = {"bytes": 40e6, "flops": 1e9}
        else:
            c.update(B=_log_int(rng, 1, 48), N=_log_int(rng, 2, 80), layers=rng.choice((1, 4, 16, 22, 32)),
                     lo=_log_int(rng, 1, 100), hi=100, Hk=rng.choice((1, 2, 4, 8)), D=rng.choice((32, 64, 128, 256)),
                     dtype=rng.choice(("fp16", "bf16")))
            if _pool_tokens(c) * c["Hk"] * c["D"] * c["layers"] > 5e8:
                continue
            top = {"bytes": 200e6, "flops": 1e9}
        w = work(c)
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            return c


# --- sizes that follow from the case alone ----------------------------------------------------------------------


def _rng(c, salt):
    return random.Random(salt * 1000003 + 8191 * c["N"] + 101 * c["B"] + c.get("lo", 0) + c.get("V", 0))


def _bases(c):
    """History length of every sequence."""
    r = _rng(c, 1)
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["B"])]


def _pool_tokens(c):
    return sum(-(-(h + c["N"]) // BS) * BS for h in _bases(c))


def _kept(c):
    """Accepted path of every sequence: node 0, then nodes that lie behind the path's new places (so that a second
    pass over the same pool moves the same rows again)."""
    r, paths = _rng(c, 2), []
    for _ in range(c["B"]):
        n = r.randint(1, max(1, min(8, (c["N"] + 1) // 2)))
        paths.append([0] + sorted(r.sample(range(n, c["N"]), n - 1)))
    return paths


def work(c):
    """Bytes read and written once, and FLOPs, of one pass."""
    B, N = c["B"], c["N"]
    if c["kind"] == "verify":
        # the distribution that the last token of every sequence comes from, and the draft's that it is the rest of
        rows = 2 if c["mode"] in ("tree", "iid") else 1
        elt = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": B * rows * c["V"] * elt + 16 * B * N, "flops": 2 * B * rows * c["V"]}
    if c["kind"] == "keep":
        moved = sum(sum(1 for j, i in enumerate(p) if i != j) for p in _kept(c))
        return {"bytes": 2 * 2 * 2 * c["layers"] * moved * c["Hk"] * c["D"] + 8 * B * N, "flops": 0}
    Hq, Hk, D = c["Hq"], c["Hk"], c["D"]
    by = fl = 0
    for h in _bases(c):
        by += 2 * 2 * Hk * D * (h + N) + 2 * 2 * Hq * D * N + 4 * (-(-(h + N) // BS)) + 4 * N * (-(-N // 32))
        fl += 4 * Hq * D * N * (h + 1)
    if c["kind"] == "step":
        by += 2 * 2 * Hk * D * N * B
    return {"bytes": by, "flops": fl}


# --- inputs -----------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _randn(g, *shape, dtype):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _trees(c, seed):
    """Parents of every sequence's nodes: a chain, or drafted level by level with a few children a node; a padded
    batch holds trees of N / 2 to N nodes."""
    r, N, out = random.Random(seed), c["N"], []
    for _ in range(c["B"]):
        n = r.randint((N + 1) // 2, N) if c.get("padded") else N
        if c.get("tree") == "chain":
            parents = list(range(-1, n - 1))
        else:
            parents = [-1]
            while len(parents) < n:
                i = len(parents)
                parents.append(r.randint(max(0, i // 4 - 1), max(0, (i - 1) // 2)))
        out.append(parents + [-2] * (N - n))
    return out


def _mask_words(parents):
    """The nodes that every node sees, itself included, as rows of 32-bit words, and the nodes' depths."""
    N = len(parents)
    W = -(-N // 32)
    seen, depths = [], []
    for i, p in enumerate(parents):
        seen.append(0 if p < -1 else (1 << i) | (seen[p] if p >= 0 else 0))
        depths.append(-1 if p < -1 else 1 + depths[p] if p >= 0 else 0)
    words = [[(s >> (32 * w)) & 0xFFFFFFFF for w in range(W)] for s in seen]
    return [[w - (1 << 32) if w >> 31 else w for w in row] for row in words], depths


def _paged(c, seed):
    """Block tables over scattered blocks and context lengths (history and nodes)."""
    lens = [h + c["N"] for h in _bases(c)]
    need = [-(-n // BS) for n in lens]
    ids = list(range(sum(need) + 4))
    random.Random(seed + 1).shuffle(ids)
    bt = torch.zeros((c["B"], max(need)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    return bt.to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV), len(ids), max(lens)


def _probabilities(c, g):
    """Target and draft logits (B, N, V) of a peaked vocabulary, the draft a rough image of the target."""
    shape = (c["B"], c["N"], c["V"])
    t = torch.randn(shape, generator=g, device=DEV)
    t.mul_(t.abs().mul_(1.7))  # a few likely tokens and a long tail
    d = torch.randn(shape, generator=g, device=DEV).mul_(0.8).add_(t)
    return t, d


def prepare(c, seed):
    g, dtype = _gen(seed), DTYPES[c["dtype"]]
    B, N = c["B"], c["N"]
    s = {"c": c}
    if c["kind"] == "verify":
        lists = _trees(c, seed)
        ranks = [[p[:i].count(p[i]) for i in range(N)] for p in lists]  # which child of its parent a node is
        s["parents"] = torch.tensor(lists, dtype=torch.int32).to(DEV)
        rank = torch.tensor(ranks, device=DEV)
        t, d = _probabilities(c, g)
        k = min(c["V"], int(rank.max()) + 1)
        u = torch.rand((B, N, c["V"]), generator=g, device=DEV).clamp_(1e-20)
        if c["mode"] in ("top", "greedy"):
            drafts = d.topk(k, dim=-1).indices
        elif c["mode"] == "tree":  # without replacement: the largest of the logits plus Gumbel noise
            drafts = (d - u.log_().neg_().log_()).topk(k, dim=-1).indices
        else:
            p = torch.softmax(d, -1).cumsum(-1)
            drafts = torch.searchsorted(p, torch.rand((B, N, k), generator=g, device=DEV) * p[..., -1:])
            drafts.clamp_(max=c["V"] - 1)
            del p
        del u
        flat = s["parents"].clamp(min=0).long() * k + rank.clamp(max=k - 1)
        s["tokens"] = drafts.reshape(B, -1).gather(1, flat)
        if c["mode"] == "greedy":
            s["target"] = t.to(dtype)
        else:
            s["target"] = torch.softmax(t, -1).to(dtype)
            if c["mode"] != "top":
                s["draft"] = torch.softmax(d, -1).to(dtype)
            s["u"] = torch.rand((B, N), generator=g, device=DEV)
        return s
    Hk, D = c["Hk"], c["D"]
    s["bt"], s["lens"], blocks, s["longest"] = _paged(c, seed)
    if c["kind"] == "keep":
        shape = (c["layers"], blocks, BS, Hk, D)
        s["k"], s["v"] = _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype)
        s["pools"] = [list(s[x].unbind(0)) for x in "kv"]  # a cache holds its layers' pools as lists
        paths = _kept(c)
        s["path"] = torch.tensor([p + [-1] * (N - len(p)) for p in paths], dtype=torch.int32).to(DEV)
        s["counts"] = torch.tensor([len(p) for p in paths], dtype=torch.int32).to(DEV)
        s["starts"] = s["lens"] - N
        return s
    lists = _trees(c, seed)
    s["k"], s["v"] = _randn(g, blocks, BS, Hk, D, dtype=dtype), _randn(g, blocks, BS, Hk, D, dtype=dtype)
    # a projection leaves (B, N, H, D); attention takes its (B, H, N, D) view
    s["q"] = _randn(g, B, N, c["Hq"], D, dtype=dtype).transpose(1, 2)
    if c["kind"] == "attend":
        s["mask"] = torch.tensor([_mask_words(p)[0] for p in lists], dtype=torch.int64).to(torch.int32).to(DEV)
    else:
        s["parents"] = torch.tensor(lists, dtype=torch.int32).to(DEV)
        s["k_new"], s["v_new"] = _randn(g, B * N, Hk, D, dtype=dtype), _randn(g, B * N, Hk, D, dtype=dtype)
        freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        angle = torch.arange(s["longest"], dtype=torch.float64).unsqueeze(1) * freq
        s["cos"], s["sin"] = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
    return s


# --- one pass ---------------------------------------------------------------------------------------------------


def run(s):
    c = s["c"]
    with torch.no_grad():
        if own:
            e = _package()
            if c["kind"] == "attend":
                return e.attention.tree_attention(s["q"], s["k"], s["v"], s["bt"], s["lens"], s["mask"],
                                                  max_context=s["longest"])
            if c["kind"] == "step":
                tree = e.decode.draft_tree(s["parents"])
                o = e.attention.tree_attention(s["q"], s["k"], s["v"], s["bt"], s["lens"], tree.mask,
                                               max_context=s["longest"], rope=(s["cos"], s["sin"]),
                                               depths=tree.depths, new_kv=(s["k_new"], s["v_new"]))
                return o, s["k"], s["v"]
            if c["kind"] == "verify":
                if c["mode"] == "greedy":
                    r = e.decode.verify_greedy(s["target"], s["tokens"], s["parents"])
                else:
                    r = e.decode.verify_draft(s["target"], s["tokens"], s["parents"], s["u"],
                                              draft_probs=s.get("draft"), replacement=c["mode"] == "iid")
                return r.tokens, r.path, r.counts
            e.cache.kv_keep(*s["pools"], s["bt"], s["starts"], s["path"], s["counts"])
            return s["k"], s["v"]
        if c["kind"] == "attend":
            return _plain_attend(s, _plain_bits(s["mask"], c["N"]))
        if c["kind"] == "step":
            return _plain_step(s)
        if c["kind"] == "verify":
            return _plain_greedy(s) if c["mode"] == "greedy" else _plain_verify(s)
        return _plain_keep(s)


def _plain_bits(mask, N):
    bits = (mask.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device=DEV)) & 1
    return bits.flatten(2)[..., :N].bool()


def _plain_slots(s, positions):
    """Pool rows (block * BS + offset) of positions (B, n)."""
    return s["bt"].long().gather(1, positions // BS) * BS + positions % BS


def _plain_attend(s, seen):
    c = s["c"]
    B, N, Hq, Hk, D = c["B"], c["N"], c["Hq"], c["Hk"], c["D"]
    L = s["longest"]
    j = torch.arange(L, device=DEV)
    rel = j.unsqueeze(0) - (s["lens"].long() - N).unsqueeze(1)  # (B, L): node index of a key
    inside = ((rel >= 0) & (rel < N)).unsqueeze(1)
    keys = seen.gather(2, rel.clamp(0, N - 1).unsqueeze(1).expand(B, N, L)) & inside
    keys |= (rel < 0).unsqueeze(1) & seen.any(-1, keepdim=True)  # a row that sees no node is none
    at = _plain_slots(s, torch.minimum(j.unsqueeze(0), s["lens"].long().unsqueeze(1) - 1))
    k = s["k"].view(-1, Hk, D)[at].float().permute(0, 2, 3, 1).contiguous()  # (B, Hk, D, L)
    v = s["v"].view(-1, Hk, D)[at].float().transpose(1, 2).contiguous()      # (B, Hk, L, D)
    q = s["q"].float().reshape(B, Hk, Hq // Hk * N, D)
    sc = (q @ k).mul_(1.0 / math.sqrt(D)).view(B, Hq, N, L)
    sc.masked_fill_(~keys.unsqueeze(1), -math.inf)
    p = sc.sub_(sc.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, Hq // Hk * N, L) @ v).view(B, Hq, N, D)
    return torch.where(total > 0, o / total, 0.0).to(DTYPES[c["dtype"]])


def _plain_rotate(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)


def _plain_step(s):
    c = s["c"]
    B, N, Hk, D = c["B"], c["N"], c["Hk"], c["D"]
    # ancestors by doubling the parent relation: link[i, p] of node i and its parent p, to itself where there is none
    parents = s["parents"].long()
    node = torch.arange(N, device=DEV)
    real = parents >= -1
    up = torch.where(parents >= 0, parents, node)
    seen = torch.eye(N, dtype=torch.bool, device=DEV).expand(B, N, N) & real.unsqueeze(-1)
    for _ in range(max(1, (N - 1).bit_length())):
        seen = seen | seen.gather(1, up.unsqueeze(-1).expand(B, N, N)) & real.unsqueeze(-1)
        up = up.gather(1, up)
    depth = seen.sum(-1) - 1
    base = s["lens"].long() - N
    pos = (base.unsqueeze(1) + depth.clamp(min=0))
    cos, sin = s["cos"][pos], s["sin"][pos]  # (B, N, D / 2)
    k = _plain_rotate(s["k_new"].view(B, N, Hk, D), cos.unsqueeze(2), sin.unsqueeze(2))
    at = _plain_slots(s, base.unsqueeze(1) + node)
    pool_k, pool_v = s["k"].view(-1, Hk, D), s["v"].view(-1, Hk, D)
    node_row = real.view(B, N, 1, 1)  # a padding slot's rows stay as they are
    pool_k[at] = torch.where(node_row, k, pool_k[at])
    pool_v[at] = torch.where(node_row, s["v_new"].view(B, N, Hk, D), pool_v[at])
    q = _plain_rotate(s["q"], cos.unsqueeze(1), sin.unsqueeze(1))
    return _plain_attend({**s, "q": q}, seen), s["k"], s["v"]


def _plain_path(s, cur, last, taken):
    """tokens, path and counts from the nodes taken (B, N, node 0 among them) and the last token."""
    N = s["c"]["N"]
    counts = taken.sum(1, dtype=torch.int32)
    node = torch.arange(N, device=DEV)
    order = torch.where(taken, node, N).sort(1).values  # taken nodes first, in order
    live = node < counts.unsqueeze(1)
    path = torch.where(live, order, -1).to(torch.int32)
    nxt = order.roll(-1, 1).clamp(max=N - 1)
    tokens = torch.where(node < (counts - 1).unsqueeze(1), s["tokens"].gather(1, nxt),
                         torch.where(live, last.unsqueeze(1), -1))
    return tokens, path, counts


def _plain_verify(s):
    c = s["c"]
    B, N, V = c["B"], c["N"], c["V"]
    row = torch.arange(B, device=DEV)
    cur = torch.zeros(B, dtype=torch.int64, device=DEV)
    taken = torch.zeros((B, N), dtype=torch.bool, device=DEV)
    taken[:, 0] = True
    p = s["target"][:, 0].double()  # what the next token of the current node is drawn from
    q = s["draft"][:, 0].double() if "draft" in s else None
    u = s["u"].double()
    parents = s["parents"].long()
    for i in range(1, N):
        child = parents[:, i] == cur
        x = s["tokens"][:, i]
        px = p[row, x]
        qx = q[row, x] if q is not None else torch.ones_like(px)
        yes = child & (u[:, i] * qx < px)
        no = (child & ~yes).unsqueeze(1)
        if q is None:
            rest = p.index_put((row, x), torch.zeros_like(px))
        else:
            rest = (p - q).clamp_(min=0)
        mass = rest.sum(1, keepdim=True)
        p = torch.where(no & (mass > NONE), rest / mass, p)
        if q is not None and c["mode"] == "tree":
            left = q.index_put((row, x), torch.zeros_like(px))
            mass = left.sum(1, keepdim=True)
            q = torch.where(no & (mass > NONE), left / mass, q)
        taken[:, i] = yes
        cur = torch.where(yes, i, cur)
        p = torch.where(yes.unsqueeze(1), s["target"][:, i].double(), p)
        if q is not None:
            q = torch.where(yes.unsqueeze(1), s["draft"][:, i].double(), q)
    total = p.cumsum(1)
    last = (total <= u[:, :1] * total[:, -1:]).sum(1)
    return _plain_path(s, cur, last, taken)


def _plain_greedy(s):
    c = s["c"]
    B, N = c["B"], c["N"]
    best = s["target"].float()
    top = best.amax(-1, keepdim=True)
    ids = torch.arange(c["V"], device=DEV)
    best = torch.where(best == top, ids, c["V"]).amin(-1)  # the lowest index among the largest
    cur = torch.zeros(B, dtype=torch.int64, device=DEV)
    taken = torch.zeros((B, N), dtype=torch.bool, device=DEV)
    taken[:, 0] = True
    parents = s["parents"].long()
    for i in range(1, N):
        yes = (parents[:, i] == cur) & (s["tokens"][:, i] == best.gather(1, cur.unsqueeze(1))[:, 0])
        taken[:, i] = yes
        cur = torch.where(yes, i, cur)
    return _plain_path(s, cur, best.gather(1, cur.unsqueeze(1))[:, 0], taken)


def _plain_keep(s):
    c = s["c"]
    j = torch.arange(c["N"], device=DEV)
    live = j < s["counts"].unsqueeze(1)
    base = s["starts"].long().unsqueeze(1)
    src = _plain_slots(s, base + torch.where(live, s["path"].long(), 0)).flatten()
    dst = _plain_slots(s, base + torch.where(live, j, 0)).flatten()
    k, v = (s[x].view(c["layers"], -1, c["Hk"], c["D"]) for x in "kv")
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    return s["k"], s["v"]


# --- the same in 64 bits, one sequence at a time ----------------------------------------------------------------


def _exact_attend(q, k, v, see):
    """q (Hq, N, D), k / v (L, Hk, D), see (N, L) bool, all keys of a row that sees none masked."""
    Hq, N, D = q.shape
    Hk = k.shape[1]
    G = Hq // Hk
    o = torch.zeros((Hq, N, D), dtype=torch.float64, device=q.device)
    rows = see.any(1)
    for h in range(Hq):
        w = q[h] @ k[:, h // G].t().contiguous() / math.sqrt(D)
        w = torch.softmax(w.masked_fill(~see, -math.inf)[rows], -1)
        o[h, rows] = w @ v[:, h // G].contiguous()
    return o


def _exact_rotate(x, cos, sin):
    """Rotated in the tables' values, then rounded to the type that the operator keeps q and the pool's K in."""
    h = x.shape[-1] // 2
    a, b = x[..., :h].double(), x[..., h:].double()
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).float().to(x.dtype)


def _exact_walk(c, tokens, parents, target, draft, u):
    """Path and last token of one sequence."""
    path, cur = [0], 0
    while True:
        p = target[cur].double()
        if c["mode"] == "greedy":
            t = int((p == p.max()).nonzero()[0])
            nxt = [i for i in range(cur + 1, len(parents)) if parents[i] == cur and tokens[i] == t][:1]
            if not nxt:
                return path, t
            cur = nxt[0]
            path.append(cur)
            continue
        q = draft[cur].double() if draft is not None else None
        taken = None
        for i in range(cur + 1, len(parents)):
            if parents[i] != cur:
                continue
            x = tokens[i]
            if float(u[i]) * (float(q[x]) if q is not None else 1.0) < float(p[x]):
                taken = i
                break
            rest = (p - q).clamp(min=0) if q is not None else p.clone()
            if q is None:
                rest[x] = 0
            if float(rest.sum()) > NONE:
                p = rest / rest.sum()
            if q is not None and c["mode"] == "tree":
                rest = q.clone()
                rest[x] = 0
                if float(rest.sum()) > NONE:
                    q = rest / rest.sum()
        if taken is None:
            total = p.cumsum(0)
            return path, int(torch.searchsorted(total, float(u[0]) * total[-1], right=True))
        cur = taken
        path.append(cur)


def exact(c, seed):
    s = prepare(c, seed)
    B, N = c["B"], c["N"]
    if c["kind"] == "keep":
        for b, path in enumerate(_kept(c)):
            h, ids = int(s["starts"][b]), s["bt"][b].tolist()
            for j, i in enumerate(path):
                for pool in (s["k"], s["v"]):
                    pool[:, ids[(h + j) // BS], (h + j) % BS] = pool[:, ids[(h + i) // BS], (h + i) % BS]
        return s["k"].double(), s["v"].double()
    if c["kind"] == "verify":
        parents, tokens = s["parents"].tolist(), s["tokens"].tolist()
        out_t, out_p, out_n = [], [], []
        for b in range(B):
            draft = s["draft"][b].cpu() if "draft" in s else None
            path, last = _exact_walk(c, tokens[b], parents[b], s["target"][b].cpu(), draft,
                                     s["u"][b].tolist() if "u" in s else None)
            out_t.append([tokens[b][i] for i in path[1:]] + [last] + [-1] * (N - len(path)))
            out_p.append(path + [-1] * (N - len(path)))
            out_n.append(len(path))
        return torch.tensor(out_t), torch.tensor(out_p, dtype=torch.int32), torch.tensor(out_n, dtype=torch.int32)
    Hk, D = c["Hk"], c["D"]
    outs, lists = [], _trees(c, seed)
    kp, vp = s["k"].view(-1, Hk, D), s["v"].view(-1, Hk, D)
    for b, h in enumerate(_bases(c)):
        pos = torch.arange(h + N, device=DEV)
        at = s["bt"][b].long()[pos // BS] * BS + pos % BS
        q = s["q"][b]
        see = torch.zeros((N, h + N), dtype=torch.bool)
        depth = []
        for i, p in enumerate(lists[b]):
            if p >= -1:
                see[i, :h] = True
                if p >= 0:
                    see[i] |= see[p]
                see[i, h + i] = True
            depth.append(0 if p < 0 else depth[p] + 1)
        if c["kind"] == "step":
            d = h + torch.tensor(depth, device=DEV)
            cos, sin = s["cos"][d].double(), s["sin"][d].double()
            q = _exact_rotate(q, cos, sin)
            n = sum(p >= -1 for p in lists[b])  # a padding slot's rows stay as they are
            new = slice(b * N, b * N + n)
            kp[at[h:h + n]] = _exact_rotate(s["k_new"][new], cos[:n].unsqueeze(1), sin[:n].unsqueeze(1))
            vp[at[h:h + n]] = s["v_new"][new]
        outs.append(_exact_attend(q.double(), kp[at].double(), vp[at].double(), see.to(DEV)))
    o = torch.stack(outs)
    return o if c["kind"] == "attend" else (o, s["k"].double(), s["v"].double())
