"""Draft trees in 64 bits on the CPU: the tree's visibility, attention over it
with a bound of the rounding a 16-bit kernel may show, the verification walk
and the move of the accepted path. Plain loops over the definitions; the walk
keeps the whole distributions and normalises them step by step."""

from __future__ import annotations

import math

import torch

NO_MASS = 2.0 ** -40


def tree_ref(parents: list[int]) -> tuple[list[set[int]], list[int]]:
    """(nodes that every node sees, depths) of one tree; padding slots see
    nothing (depth -1), nodes with a broken chain neither (depth -2)."""
    seen: list[set[int]] = []
    depths: list[int] = []
    for i, p in enumerate(parents):
        if p < -1:
            seen.append(set())
            depths.append(-1)
        elif p == -1:
            seen.append({i})
            depths.append(0)
        elif p >= i or depths[p] < 0:
            seen.append(set())
            depths.append(-2)
        else:
            seen.append(seen[p] | {i})
            depths.append(depths[p] + 1)
    return seen, depths


def mask_words(seen: list[set[int]]) -> torch.Tensor:
    """int32 (N, ceil(N / 32)) bit rows of a tree's visibility."""
    N = len(seen)
    out = torch.zeros((N, -(-N // 32)), dtype=torch.int64)
    for i, s in enumerate(seen):
        for a in s:
            out[i, a // 32] |= 1 << (a % 32)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32)


def tree_attention_f64(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, see: torch.Tensor,
                       scale: float, parts: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """One sequence: q (Hq, N, D), k / v (L, Hk, D), see (N, L) bool. Returns
    the outputs (Hq, N, D) in 64 bits (zero rows where a row sees nothing,
    masked keys left out of every sum) and, elementwise, how far a kernel may
    be off that rounds the probabilities and the output once each to q's type
    and accumulates in fp32:

    half a step of the output, half a step (or half the smallest 16-bit
    magnitude) of every probability times |v|, and for the fp32 sums of D
    products per score and L terms per row, 2^-24 per addition. ``parts`` = 2:
    a kernel that also keeps what the rounding of a probability left, rounded
    to q's type, as a second term; half a step of half a step is lost then."""
    h = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps / 2
    Hq, N, D = q.shape
    L, Hk, _ = k.shape
    out = torch.zeros((Hq, N, D), dtype=torch.float64)
    bound = torch.zeros((Hq, N, D), dtype=torch.float64)
    for hq in range(Hq):
        hk = hq // (Hq // Hk)
        for i in range(N):
            keys = see[i].nonzero().flatten()
            if not len(keys):
                continue
            kk, vv, qq = k[keys, hk].double(), v[keys, hk].double(), q[hq, i].double()
            s = kk @ qq * scale
            p = torch.softmax(s, 0)
            top = float(p.max())
            out[hq, i] = p @ vv
            a = p @ vv.abs()
            reach = float((kk.abs() @ qq.abs()).max()) * abs(scale)  # sum of |products| behind a score
            eps32 = 2.0 ** -24 * (2 * (D + 8) * reach + parts * L + 64)
            # probabilities are rounded relative to the running maximum, the largest being up to 1
            bound[hq, i] = (h * out[hq, i].abs() + h ** parts * a * (1 + h) + tiny * (1 + top * vv.abs().sum(0))
                            + eps32 * a)
    return out, bound


def verify_ref(target: torch.Tensor, tokens: list[int], parents: list[int], u: list[float] | None,
               draft: torch.Tensor | None, mode: str) -> tuple[list[int], list[int]]:
    """(path, emitted tokens) of one sequence; target / draft (N, V). mode:
    "greedy", "picks", "iid" or "tree". Empty lists for a padding node 0."""
    N, V = target.shape
    if parents[0] != -1:
        return [], []
    path, cur = [0], 0
    while True:
        p = target[cur].double()
        kids = [i for i in range(cur + 1, N) if parents[i] == cur and 0 <= tokens[i] < V]
        taken = None
        if mode == "greedy":
            nan = torch.isnan(p).nonzero()
            last = int(nan[0]) if len(nan) else int((p == p.max()).nonzero()[0])
            taken = next((i for i in kids if tokens[i] == last), None)
        else:
            q = draft[cur].double() if draft is not None else None
            for i in kids:
                x = tokens[i]
                if u[i] * (float(q[x]) if q is not None else 1.0) < float(p[x]):
                    taken = i
                    break
                rest = p.clone() if q is None else (p - q).clamp(min=0)
                if q is None:
                    rest[x] = 0.0
                mass = math.fsum(rest.tolist())
                if mass > NO_MASS:
                    p = rest / mass
                if mode == "tree":
                    rest = q.clone()
                    rest[x] = 0.0
                    mass = math.fsum(rest.tolist())
                    if mass > NO_MASS:
                        q = rest / mass
            if taken is None:
                cum = p.cumsum(0)
                over = (cum > u[0] * cum[-1]).nonzero()
                positive = (p > 0).nonzero()
                last = int(over[0]) if len(over) else int(positive[-1]) if len(positive) else -1
        if taken is None:
            return path, [tokens[i] for i in path[1:]] + [last]
        cur = taken
        path.append(cur)


def keep_ref(pool: torch.Tensor, blocks: list[int], start: int, path: list[int]) -> None:
    """Moves rows start + path[j] to start + j of one (num_blocks, block_size,
    Hk, D) pool, in order."""
    bs = pool.shape[1]
    for j, i in enumerate(path):
        s, d = start + i, start + j
        pool[blocks[d // bs], d % bs] = pool[blocks[s // bs], s % bs].clone()
