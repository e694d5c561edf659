"""Draft trees on the GPU: calls at the edge of what the documentation allows."""

from __future__ import annotations

import pytest
import torch

from engine.decode import verify_draft, verify_greedy

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
