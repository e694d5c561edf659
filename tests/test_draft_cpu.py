"""Draft trees on the CPU: what the C ABI refuses before it touches the GPU, the
oracle against hand-worked trees, and the host side of a step."""

from __future__ import annotations

import ctypes
import dataclasses
import math
import random

import pytest
import torch
from oracle.draft_ref import keep_ref, mask_words, tree_attention_f64, tree_ref, verify_ref

from engine import _lib
from engine.attention import tree_attention
from engine.cache import KVCacheConfig, PagedKVCache, StepBatch, kv_keep
from engine.decode import accept_draft, draft_tree, verify_draft, verify_greedy

FAKE = 1 << 20  # aligned, never dereferenced: validation fails first


def _st(*s):
    return (ctypes.c_int64 * len(s))(*s)


# --- refusals of the C ABI --------------------------------------------------------------------------------------


def _tree(**over):
    a = dict(q=FAKE, kn=None, vn=None, kc=FAKE, vc=FAKE, bt=FAKE, lens=FAKE, mask=FAKE, depths=None, o=FAKE, ws=FAKE,
             wsb=1 << 40, qs=_st(8192, 1024, 64, 1), kns=_st(128, 64, 1), vns=_st(128, 64, 1), ks=_st(2048, 128, 64, 1),
             vs=_st(2048, 128, 64, 1), os_=_st(8192, 1024, 64, 1), ms=16, ds=16, B=2, Hq=8, Hk=2, N=16, D=64,
             num_blocks=100, bs=16, width=50, mc=0, scale=0.125, dtype=0, cos=None, sin=None, rows=0, rdt=0)
    a.update(over)
    return _lib.load().cie_tree_attn(
        a["q"], a["kn"], a["vn"], a["kc"], a["vc"], a["bt"], a["lens"], a["mask"], a["depths"], a["o"], a["ws"],
        a["wsb"], a["qs"], a["kns"], a["vns"], a["ks"], a["vs"], a["os_"], a["ms"], a["ds"], a["B"], a["Hq"], a["Hk"],
        a["N"], a["D"], a["num_blocks"], a["bs"], a["width"], a["mc"], a["scale"], a["dtype"], a["cos"], a["sin"],
        a["rows"], a["rdt"], None)


@pytest.mark.parametrize("over,code", [
    (dict(D=48), "CIE_EHEADDIM"), (dict(dtype=2), "CIE_EDTYPE"), (dict(Hq=7), "CIE_EINVAL"), (dict(B=-1), "CIE_EINVAL"),
    (dict(N=-1), "CIE_EINVAL"), (dict(N=1025), "CIE_EINVAL"), (dict(bs=0), "CIE_EINVAL"),
    (dict(num_blocks=-1), "CIE_EINVAL"), (dict(width=-1), "CIE_EINVAL"), (dict(width=1 << 28, bs=16), "CIE_EINVAL"), (dict(width=(1 << 31) - 1, bs=1), "CIE_EINVAL"),
    (dict(scale=math.nan), "CIE_EINVAL"), (dict(scale=math.inf), "CIE_EINVAL"), (dict(q=None), "CIE_EINVAL"),
    (dict(q=FAKE + 2), "CIE_EINVAL"), (dict(o=None), "CIE_EINVAL"), (dict(kc=FAKE + 8), "CIE_EINVAL"),
    (dict(vc=None), "CIE_EINVAL"), (dict(bt=None), "CIE_EINVAL"), (dict(lens=None), "CIE_EINVAL"),
    (dict(mask=None), "CIE_EINVAL"), (dict(qs=_st(8192, 1024, 63, 1)), "CIE_EINVAL"),
    (dict(ks=_st(2048, 128, 64, 2)), "CIE_EINVAL"), (dict(vs=_st(2048, -128, 64, 1)), "CIE_EINVAL"),
    (dict(ks=_st(2048, 128, 1 << 31, 1)), "CIE_EINVAL"), (dict(ms=-1), "CIE_EINVAL"), (dict(ds=-1), "CIE_EINVAL"),
    (dict(cos=FAKE, sin=FAKE, rows=64, rdt=0), "CIE_EINVAL"),                    # without depths
    (dict(cos=FAKE, sin=None, rows=64, rdt=0, depths=FAKE), "CIE_EINVAL"),
    (dict(cos=FAKE, sin=FAKE, rows=64, rdt=3, depths=FAKE), "CIE_EDTYPE"),
    (dict(kn=FAKE), "CIE_EINVAL"), (dict(kn=FAKE, vn=FAKE, kns=_st(127, 64, 1)), "CIE_EINVAL"),
    (dict(kn=FAKE, vn=FAKE, vns=None), "CIE_EINVAL"), (dict(ws=None), "CIE_EWORKSPACE"), (dict(wsb=64), "CIE_EWORKSPACE"),
    (dict(ws=FAKE + 8), "CIE_EINVAL"), (dict(B=70000, width=4), "CIE_EINVAL"),
    (dict(B=60000, Hq=1024, Hk=1024, N=1, width=400), "CIE_EINVAL"),             # more threads than a grid has
])
def test_tree_attention_refuses(over, code):
    assert _tree(**over) == getattr(_lib, code)
    assert _lib.last_error()


def test_tree_attention_of_nothing():
    assert _tree(B=0) == 0 and _tree(N=0) == 0


def test_tree_workspace():
    f = _lib.load().cie_tree_workspace_bytes
    assert f(1, 8, 2, 16, 64, 0, 16, 2) == 0          # 32 tokens at most: never split
    small, large = f(1, 8, 2, 16, 64, 0, 16, 100), f(1, 8, 2, 64, 64, 0, 16, 100)
    assert 0 < small < large and small % 256 == 0
    for bad in ((0, 8, 2, 16, 64, 0, 16, 100), (1, 8, 3, 16, 64, 0, 16, 100), (1, 8, 2, 1025, 64, 0, 16, 100),
                (1, 8, 2, 16, 48, 0, 16, 100), (1, 8, 2, 16, 64, 0, 0, 100), (1, 8, 2, 16, 64, 0, 16, -1)):
        assert f(*bad) == 0


@pytest.mark.parametrize("over", [dict(parents=None), dict(mask=None), dict(depths=None), dict(B=-1), dict(N=-1),
                                  dict(N=1025), dict(B=1 << 22)])
def test_draft_masks_refuse(over):
    a = dict(parents=FAKE, mask=FAKE, depths=FAKE, B=2, N=5)
    a.update(over)
    assert _lib.load().cie_draft_masks(a["parents"], a["mask"], a["depths"], None, a["B"], a["N"], None) == _lib.CIE_EINVAL


def _verify(greedy, **over):
    a = dict(t=FAKE, d=FAKE, x=FAKE, xb=8, p=FAKE, u=FAKE, ub=4, tok=FAKE, path=FAKE, cnt=FAKE, ts=_st(500, 100, 1),
             ds=_st(500, 100, 1), B=2, N=5, V=100, dtype=2, ws=FAKE, wsb=1 << 30)
    a.update(over)
    lib = _lib.load()
    if greedy:
        return lib.cie_verify_greedy(a["t"], a["x"], a["xb"], a["p"], a["tok"], a["path"], a["cnt"], a["ts"], a["B"],
                                     a["N"], a["V"], a["dtype"], a["ws"], a["wsb"], None)
    return lib.cie_verify_draft(a["t"], a["d"], a["x"], a["xb"], a["p"], a["u"], a["ub"], a["tok"], a["path"], a["cnt"],
                                a["ts"], a["ds"], a["B"], a["N"], a["V"], a["dtype"], 0, None)


@pytest.mark.parametrize("greedy", [True, False])
@pytest.mark.parametrize("over,code", [
    (dict(dtype=3), "CIE_EDTYPE"), (dict(dtype=-1), "CIE_EDTYPE"), (dict(B=-1), "CIE_EINVAL"), (dict(N=-1), "CIE_EINVAL"),
    (dict(V=-1), "CIE_EINVAL"), (dict(V=0), "CIE_EINVAL"), (dict(N=1025), "CIE_EINVAL"), (dict(B=1 << 22), "CIE_EINVAL"),
    (dict(V=(1 << 30) + 1), "CIE_EINVAL"), (dict(xb=2), "CIE_EINVAL"), (dict(t=None), "CIE_EINVAL"),
    (dict(t=FAKE + 2), "CIE_EINVAL"), (dict(x=None), "CIE_EINVAL"), (dict(p=None), "CIE_EINVAL"),
    (dict(tok=None), "CIE_EINVAL"), (dict(path=None), "CIE_EINVAL"), (dict(cnt=None), "CIE_EINVAL"),
    (dict(ts=None), "CIE_EINVAL"), (dict(ts=_st(-1, 100, 1)), "CIE_EINVAL"),
])
def test_verification_refuses(greedy, over, code):
    assert _verify(greedy, **over) == getattr(_lib, code)


@pytest.mark.parametrize("over", [dict(u=None), dict(ub=2), dict(ds=None), dict(ds=_st(500, -1, 1)), dict(d=FAKE + 1)])
def test_sampled_verification_refuses(over):
    assert _verify(False, **over) == _lib.CIE_EINVAL


def test_greedy_workspace():
    f = _lib.load().cie_verify_greedy_workspace_bytes
    assert f(2, 5, 100, 2) > 0 and f(2, 5, 100, 2) == f(2, 5, 100, 0)
    assert f(1, 1024, 1 << 17, 1) == 0                # 256 MiB of logits: read on the walk
    assert f(1 << 20, 1024, 1, 0) == 0                # more rows than one launch takes
    for bad in ((0, 5, 100, 2), (2, 0, 100, 2), (2, 1025, 100, 2), (2, 5, 0, 2), (2, 5, 100, 3), (2, 5, (1 << 30) + 1, 0)):
        assert f(*bad) == 0
    assert _verify(True, ws=None) == _lib.CIE_EWORKSPACE
    assert _verify(True, wsb=f(2, 5, 100, 2) - 1) == _lib.CIE_EWORKSPACE
    assert _verify(True, ws=FAKE + 8) == _lib.CIE_EINVAL
    assert _verify(True, B=0) == 0 and _verify(False, N=0) == 0


@pytest.mark.parametrize("over", [
    dict(layers=-1), dict(B=-1), dict(N=-1), dict(N=1025), dict(B=65536), dict(heads=0), dict(hb=8), dict(hb=24),
    dict(hb=8192), dict(bs=0), dict(nb=-1), dict(width=-1), dict(width=1 << 28), dict(bt=None), dict(st=None),
    dict(path=None), dict(cnt=None), dict(ps=-1), dict(ks=_st(8, 128, 64)), dict(vs=_st(2048, -128, 64)), dict(ks=None),
    dict(k=None), dict(k=[FAKE, FAKE + 8]), dict(v=[FAKE, None])])
def test_keep_refuses(over):
    a = dict(k=[FAKE, FAKE], v=[FAKE, FAKE], layers=2, ks=_st(2048, 128, 64), vs=_st(2048, 128, 64), bt=FAKE, st=FAKE,
             path=FAKE, ps=5, cnt=FAKE, B=2, N=5, heads=2, hb=64, nb=10, bs=16, width=4)
    a.update(over)
    k, v = (None if a[n] is None else (ctypes.c_void_p * len(a[n]))(*a[n]) for n in ("k", "v"))
    assert _lib.load().cie_kv_keep(k, v, a["layers"], a["ks"], a["vs"], a["bt"], a["st"], a["path"], a["ps"], a["cnt"],
                                   a["B"], a["N"], a["heads"], a["hb"], a["nb"], a["bs"], a["width"], None) \
        == _lib.CIE_EINVAL


def test_python_boundary_requires_gpu_tensors():
    h = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    pool = torch.zeros(2, 16, 2, 64, dtype=torch.float16)
    i = torch.zeros(1, 3, dtype=torch.int32)
    p = torch.zeros(1, 3, 10)
    for call in (lambda: tree_attention(h, pool, pool, i, i[:, 0], i.unsqueeze(-1)), lambda: draft_tree(i),
                 lambda: verify_greedy(p, i, i), lambda: verify_draft(p, i, i, p[..., 0]),
                 lambda: kv_keep([pool], [pool], i, i[:, 0], i, i[:, 0])):
        with pytest.raises(RuntimeError):
            call()


# --- a step's host side -----------------------------------------------------------------------------------------------


def test_keep_step_takes_the_trees_own_step_and_rollback_frees_blocks():
    cache = PagedKVCache(KVCacheConfig(num_layers=1, num_kv_heads=1, head_dim=16, num_blocks=40, block_size=4,
                                       dtype=torch.float32, device="cpu"))
    tables = [cache.new_sequence() for _ in range(3)]
    for t in tables:
        t.blocks, t.length = [cache._alloc_block() for _ in range(4)], 14
    i = torch.tensor([14] * 3, dtype=torch.int32)
    step = StepBatch(torch.tensor([t.blocks for t in tables], dtype=torch.int32), i, torch.arange(0, 28, 9), i - 9, 9, 14,
                     tuple(tables), (5,) * 3, (14,) * 3, None, (9,) * 3)
    path = torch.zeros((3, 8), dtype=torch.int32)
    for wrong in (path, path[0], torch.zeros((3, 10), dtype=torch.int32)):
        with pytest.raises(ValueError):
            cache.keep_step(step, wrong, path[:, 0])
    early = dataclasses.replace(step, starts_host=(0, 5, 5))  # nodes that are not the newest tokens
    with pytest.raises(ValueError):
        cache.keep_step(early, torch.zeros((3, 9), dtype=torch.int32), path[:, 0])
    for wrong in ([1, 2], [1, 2, 10], [1, -1, 2]):
        with pytest.raises(ValueError):
            cache.rollback_step(step, wrong)
    free = len(cache._free)
    cache.rollback_step(step, [0, 4, 9])
    assert [t.length for t in tables] == [5, 9, 14]
    assert [len(t.blocks) for t in tables] == [2, 3, 4] and len(cache._free) == free + 3
    with pytest.raises(ValueError):
        accept_draft(cache, step, None, None, None, None, torch.zeros(1))


# --- the oracle, by hand ------------------------------------------------------------------------------------------------


def test_oracle_trees():
    seen, depths = tree_ref([-1, 0, 0, 1, 3, -2, 5, 7])
    assert depths == [0, 1, 1, 2, 3, -1, -2, -2]
    assert [sorted(x) for x in seen] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [], [], []]
    assert mask_words([{0, 31, 32}, set()] + [{a} for a in range(31)])[:2].tolist() == [[-(1 << 31) + 1, 1], [0, 0]]


def test_oracle_attention_by_hand():
    # one head, two visible keys of equal score, one that is not seen holding NaN; a row that sees nothing
    q = torch.ones(1, 2, 16, dtype=torch.float16)
    k, v = torch.ones(3, 1, 16, dtype=torch.float16), torch.full((3, 1, 16), float("nan"), dtype=torch.float16)
    v[0], v[1] = 1.0, 4.0
    out, bound = tree_attention_f64(q, k, v, torch.tensor([[True, True, False], [False] * 3]), 0.25)
    assert torch.equal(out[0, 0], torch.full((16,), 2.5, dtype=torch.float64)) and not out[0, 1].any()
    # half a step of the output and of the probabilities times |v|: 2 * 2^-11 * 2.5, and a little for fp32
    assert float(bound[0, 0].max()) < 2.6e-3 and not bound[0, 1].any()


def test_oracle_verification_is_the_targets_distribution():
    """The first emitted token over many draws, within five standard deviations
    of every bin's binomial count."""
    r, n = random.Random(7), 4000
    p, q = [0.5, 0.15, 0.05, 0.3], [0.1, 0.5, 0.25, 0.15]
    rows, drows = torch.tensor([p] * 3), torch.tensor([q] * 3)
    for mode in ("iid", "tree"):
        got = [0] * 4
        for _ in range(n):
            a = r.choices(range(4), q)[0]
            b = r.choices(range(4), [0 if mode == "tree" and y == a else q[y] for y in range(4)])[0]
            _, out = verify_ref(rows, [0, a, b], [-1, 0, 0], [r.random() for _ in range(3)], drows, mode)
            got[out[0]] += 1
        assert max(abs(g - n * x) / math.sqrt(n * x * (1 - x)) for g, x in zip(got, p)) < 5, (mode, got)


def test_oracle_sees_planted_mistakes():
    """Another mode, a wrong parent and the wrong draft distribution each move the
    oracle's answer, so a kernel with that mistake cannot agree with it."""
    r = random.Random(1)
    target = torch.softmax(torch.randn(6, 12, generator=torch.Generator().manual_seed(1)) * 2, -1)
    draft = torch.softmax(torch.randn(6, 12, generator=torch.Generator().manual_seed(2)) * 2, -1)
    parents = [-1, 0, 0, 1, 1, 2]
    seen = set()
    for _ in range(600):
        tokens = [r.choices(range(12), draft[max(p, 0)].tolist())[0] for p in parents]
        u = [r.random() for _ in range(6)]
        right = verify_ref(target, tokens, parents, u, draft, "tree")
        for name, other in (("mode", verify_ref(target, tokens, parents, u, draft, "iid")),
                            ("parent", verify_ref(target, tokens, [-1, 0, 0, 2, 1, 2], u, draft, "tree")),
                            ("draft", verify_ref(target, tokens, parents, u, target, "tree"))):
            if other != right:
                seen.add(name)
    assert seen == {"mode", "parent", "draft"}


def test_oracle_moves():
    pool = torch.arange(12.0).view(3, 4, 1, 1)
    keep_ref(pool, [2, 0, 1], 2, [0, 2, 3, 6])  # positions 0 .. 11 are rows 8 .. 11, 0 .. 7
    assert pool.flatten().tolist() == [1, 4, 2, 3, 4, 5, 6, 7, 8, 9, 10, 0]
