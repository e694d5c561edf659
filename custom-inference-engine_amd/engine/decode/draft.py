"""Draft trees of speculative decoding.

The reference drafts one chain of tokens and verifies it greedily
(``engine/decode/speculative.py:47-133``). Here a sequence's draft is a tree of
N nodes, given by the parent of every node: node 0 is the last token the
sequence has (parent -1; the reference's verify input starts with it too,
``speculative.py:88``), every other node is a drafted token that comes after
its parent, and a parent below -1 marks a padding slot of the batch. A chain is
the tree with parents -1, 0, 1, ...

A step: :func:`draft_tree` of the parents, once for all layers; per layer
``engine.model.tree_section`` (or ``engine.attention.tree_attention``); then
:func:`accept_draft` of the target's probabilities or logits, which verifies the
tokens (:func:`verify_draft`, :func:`verify_greedy`) and moves the accepted
path's K and V behind the history. The counts stay on the device until the
program reads them with the tokens; ``PagedKVCache.rollback_step`` then shortens
the sequences.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple

import torch

from engine import _lib

MAX_NODES = 1024
_TOKEN_BYTES = {torch.int32: 4, torch.int64: 8}
_UNIFORM_BYTES = {torch.float32: 4, torch.float64: 8}


@dataclass(frozen=True)
class DraftTree:
    """A batch of trees on the device: ``parents`` int32 (B, N), ``mask`` int32
    (B, N, ceil(N / 32)), bit a of row i set iff node a is node i or its
    ancestor, and ``depths`` int32 (B, N), -1 for padding slots. Without the
    batch dimension: one tree for all sequences."""
    parents: torch.Tensor
    mask: torch.Tensor
    depths: torch.Tensor


class Verified(NamedTuple):
    """``tokens`` (B, N), like the drafted ones: the accepted nodes' tokens and
    the last one, then -1; ``path`` int32 (B, N): node 0 and the accepted nodes,
    then -1; ``counts`` int32 (B,): how many entries of both (0 for a sequence
    whose node 0 is a padding slot, and for trees without nodes)."""
    tokens: torch.Tensor
    path: torch.Tensor
    counts: torch.Tensor


def _check_nodes(N: int) -> None:
    if N > MAX_NODES:
        raise ValueError(f"a draft tree has at most {MAX_NODES} nodes, got {N}")


def draft_tree(parents: torch.Tensor, status: torch.Tensor | None = None) -> DraftTree:
    """The masks and depths of trees given by ``parents``, int32 or int64
    (B, N), or (N,) for one tree, on the GPU. A node whose chain to the root
    meets a padding slot or a parent that does not come before its child is
    laid out as a padding slot (depth -2) and ORs 1 into ``status`` (optional
    int32 (1,) on the device)."""
    done = _lib.host().masks(parents, status)
    if done is not None:
        mask, depths, p = _lib.checked(done)
        return DraftTree(p, mask, depths)
    if not parents.is_cuda:
        raise RuntimeError("draft_tree requires CUDA tensors")
    if parents.dim() not in (1, 2) or parents.dtype not in _TOKEN_BYTES:
        raise ValueError(f"parents must be int32 or int64 (B, N) or (N,), got {parents.dtype} {tuple(parents.shape)}")
    _check_nodes(parents.shape[-1])
    if status is not None and (not status.is_cuda or status.device != parents.device or status.numel() < 1
                               or status.dtype not in (torch.int32, torch.uint32)):
        raise ValueError("status must be an int32 tensor on parents' device")
    p = _lib.index32(parents)
    N = p.shape[-1]
    B = p.shape[0] if p.dim() == 2 else 1
    mask = torch.empty((*p.shape, -(-N // 32)), dtype=torch.int32, device=p.device)
    depths = torch.empty_like(p)
    with torch.cuda.device(p.device):
        rc = _lib.load().cie_draft_masks(p.data_ptr(), mask.data_ptr(), depths.data_ptr(),
                                         status.data_ptr() if status is not None else None, B, N,
                                         _lib.stream_handle(p.device))
    _lib.check(rc)
    return DraftTree(p, mask, depths)


def _verify(name: str, target: torch.Tensor, draft_tokens: torch.Tensor, parents: torch.Tensor,
            uniforms: torch.Tensor | None, draft: torch.Tensor | None, replacement: bool) -> Verified:
    done = _lib.host().verify(target, draft_tokens, parents, uniforms, draft, replacement)
    if done is not None:
        return Verified(*_lib.checked(done))
    # everything else: refuse, copy or convert
    given = [("target", target), ("draft_tokens", draft_tokens), ("parents", parents)]
    given += [(n, t) for n, t in (("uniforms", uniforms), ("draft_probs", draft)) if t is not None]
    for n, t in given:
        if not t.is_cuda or t.device != target.device:
            raise RuntimeError(f"{name} requires CUDA tensors on one device ({n})")
    if target.dim() != 3 or target.dtype not in _lib.TABLE_DTYPE_CODES:
        raise ValueError(f"{name} expects fp32, fp16 or bf16 (B, N, V), got {target.dtype} {tuple(target.shape)}")
    B, N, V = target.shape
    _check_nodes(N)
    if V < 1:
        raise ValueError(f"{name}: the vocabulary is empty")
    if tuple(draft_tokens.shape) != (B, N) or draft_tokens.dtype not in _TOKEN_BYTES:
        raise ValueError(f"draft_tokens must be int32 or int64 ({B}, {N}), got {draft_tokens.dtype} "
                         f"{tuple(draft_tokens.shape)}")
    if tuple(parents.shape) not in ((B, N), (N,)) or parents.dtype not in _TOKEN_BYTES:
        raise ValueError(f"parents must be int32 or int64 ({B}, {N}) or ({N},), got {parents.dtype} "
                         f"{tuple(parents.shape)}")
    if uniforms is not None and (tuple(uniforms.shape) != (B, N) or uniforms.dtype not in _UNIFORM_BYTES):
        raise ValueError(f"uniforms must be fp32 or fp64 ({B}, {N}), got {uniforms.dtype} {tuple(uniforms.shape)}")
    if draft is not None and (draft.shape != target.shape or draft.dtype != target.dtype):
        raise ValueError(f"draft_probs must be {target.dtype} {tuple(target.shape)}, got {draft.dtype} "
                         f"{tuple(draft.shape)}")
    target = target if target.stride(-1) == 1 else target.contiguous()
    if draft is not None and draft.stride(-1) != 1:
        draft = draft.contiguous()
    draft_tokens = draft_tokens.contiguous()
    parents = _lib.index32(parents).expand(B, N).contiguous()
    tokens = torch.empty_like(draft_tokens)
    path = torch.empty_like(parents)
    # (the library writes nothing for trees without nodes)
    counts = (torch.empty if N else torch.zeros)((B,), dtype=torch.int32, device=target.device)
    lib = _lib.load()
    outs = (tokens.data_ptr(), path.data_ptr(), counts.data_ptr(), _lib.strides3(target))
    sizes = (B, N, V, _lib.TABLE_DTYPE_CODES[target.dtype])
    head = (draft_tokens.data_ptr(), _TOKEN_BYTES[draft_tokens.dtype], parents.data_ptr())
    with torch.cuda.device(target.device):
        stream = _lib.stream_handle(target.device)
        if uniforms is None:
            nbytes = int(lib.cie_verify_greedy_workspace_bytes(*sizes))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=target.device) if nbytes else None
            rc = lib.cie_verify_greedy(target.data_ptr(), *head, *outs, *sizes,
                                       ws.data_ptr() if ws is not None else None, nbytes, stream)
        else:
            u = uniforms.contiguous()
            rc = lib.cie_verify_draft(target.data_ptr(), draft.data_ptr() if draft is not None else None, *head,
                                      u.data_ptr(), _UNIFORM_BYTES[u.dtype], *outs,
                                      _lib.strides3(draft if draft is not None else target), *sizes,
                                      1 if replacement else 0, stream)
    _lib.check(rc)
    return Verified(tokens, path, counts)


def verify_draft(target_probs: torch.Tensor, draft_tokens: torch.Tensor, parents: torch.Tensor,
                 uniforms: torch.Tensor, draft_probs: torch.Tensor | None = None, *,
                 replacement: bool = False) -> Verified:
    """Speculative sampling over draft trees from given random numbers: the
    accepted path of every sequence and the token after it, distributed as the
    target's own samples when the drafts were sampled from ``draft_probs``.

    ``target_probs`` (B, N, V) fp32, fp16 or bf16: the target's probabilities
    after every node. ``draft_tokens`` (B, N) int32 or int64; a token outside
    the vocabulary is never accepted. ``parents`` (B, N) or (N,).
    ``uniforms`` (B, N) fp32 or fp64 in [0, 1): entry i tests node i, entry 0
    draws the last token. ``draft_probs`` (B, N, V) in target_probs' type: what
    a node's children were sampled from, without replacement (each child from
    what the ones before it left) or with (``replacement``); None when the
    children are the draft's own picks (its likeliest tokens, say).

    From node 0 on, the children of a node are tried in order: child i with
    token x is accepted iff ``u_i q(x) < p(x)``; after a rejection p becomes
    ``max(p - q, 0)`` and, without replacement, q loses x, each over its sum
    (unless that is below 2^-40). With picks q(x) is 1 and p loses x. When no
    child is accepted, the last token is the first y at which the running sum of
    p exceeds ``u_0 sum(p)``. All of it is computed in 64 bits. The rows of the
    visited nodes alone decide, but entries of all others are read too: nothing
    else may write them meanwhile. Nothing waits for the GPU."""
    if uniforms is None:
        raise ValueError("verify_draft needs uniforms; verify_greedy takes none")
    return _verify("verify_draft", target_probs, draft_tokens, parents, uniforms, draft_probs, bool(replacement))


def verify_greedy(target_logits: torch.Tensor, draft_tokens: torch.Tensor, parents: torch.Tensor) -> Verified:
    """Greedy verification: a child is accepted iff its token is the target's
    argmax at its parent (``target_logits`` (B, N, V) fp32, fp16 or bf16; the
    lowest index of equal logits, a NaN counts as the largest); the last token
    is the argmax at the last accepted node. The result equals plain greedy
    decoding token for token (the reference's loop over a chain,
    ``engine/decode/speculative.py:88-133``)."""
    return _verify("verify_greedy", target_logits, draft_tokens, parents, None, None, False)


def accept_draft(cache, step, parents: torch.Tensor, draft_tokens: torch.Tensor, target: torch.Tensor,
                 uniforms: torch.Tensor | None = None, draft_probs: torch.Tensor | None = None, *,
                 replacement: bool = False) -> Verified:
    """The end of a tree step (``step = cache.prepare_step(tables, N)``, all
    layers run): verifies the drafts, greedily by logits when ``uniforms`` is
    None, and moves the accepted paths' K and V behind the histories in every
    layer (``PagedKVCache.keep_step``). Two or three launches, nothing waits; once the
    program has read the counts, ``cache.rollback_step(step, counts)`` shortens
    the sequences to what they keep."""
    if uniforms is None:
        if draft_probs is not None:
            raise ValueError("draft_probs need uniforms")
        done = verify_greedy(target, draft_tokens, parents)
    else:
        done = verify_draft(target, draft_tokens, parents, uniforms, draft_probs, replacement=replacement)
    cache.keep_step(step, done.path, done.counts)
    return done
