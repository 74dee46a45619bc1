"""Drafted tokens: what their operators refuse, and the oracle's own properties, without a GPU."""

import random

import pytest
import torch

from plain import drafts_plain as plain
from sleuth_b200.kernels import ops


def test_tensors_off_the_device_are_refused():
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.draft_tree(z, z, z[:1], z[:1], z.view(4, 1), z, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_tree(torch.zeros(4, 2, 16), torch.zeros(1, 2, 64, 16), torch.zeros(1, 2, 64, 16), torch.zeros(4, 32), z, z, z, z.view(4, 1), z,
                           z[:1].view(1, 1), 4, 2, 2, 16, 0, 0.25)
    with pytest.raises(ValueError, match="CUDA"):
        ops.verify_drafts(torch.zeros(4, 9), 9, z, z, z, z[:1], torch.zeros(4), 1.0, z.view(1, 4), z, z, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.cache_compact(torch.zeros(1, 1, 64, 8), z.view(1, 4), z, z.view(1, 4), z)


def test_the_packed_calls_have_the_sizes_that_the_kernels_read():
    assert ops._TREE_CALL.size == 13 * 8 + 3 * 8 + 10 * 4 + 4 + 4
    assert ops._VERIFY_CALL.size == 13 * 8 + 4 * 8 + 8 + 4 * 4


def test_refusals_stay_in_one_family():
    """What the kernel rests on: after k refusals p is max(p - c_k q, 0) over its sum F_k, with c_{k+1} = c_k + F_k."""
    g = torch.Generator().manual_seed(1)
    for _ in range(20):
        p, q = (torch.softmax(2 * torch.randn(50, generator=g, dtype=torch.float64), 0) for _ in range(2))
        direct, c, f = p.clone(), 0.0, 1.0
        for _ in range(6):
            direct = torch.clamp(direct - q, min=0)
            direct = direct / direct.sum()
            c += f
            family = torch.clamp(p - c * q, min=0)
            f = float(family.sum())
            assert torch.allclose(direct, family / f, rtol=0, atol=1e-12)


def test_the_oracle_follows_the_target():
    """The oracle's own verification leaves the target's distribution as it is (exact sum over drafts, a grid over the random numbers)."""
    target, draft = torch.tensor([1.0, 0.0, -1.0]), torch.softmax(torch.tensor([0.0, 1.5, 0.5]), 0)
    p, grid, got = torch.softmax(target.double(), 0), 400, torch.zeros(3, dtype=torch.float64)
    logits, probs = target.repeat(2, 1), draft.repeat(2, 1)
    for x in range(3):
        for a in range(grid):
            for b in range(0, grid, 20):
                path, token = plain.verify(logits, [0, x], [-1, 0], [(b + 0.5) / grid * 1.0, (a + 0.5) / grid], 1.0, 3, probs)
                got[x if len(path) > 1 else token] += float(draft[x]) / (grid * grid / 20)
    assert bool(((got - p).abs() < 20 / grid).all())


def test_ways_end_at_parents_that_are_no_earlier_nodes():
    seen, depth = plain.ways([-1, 5, 0, 2, 3, 9], 0)
    assert depth == [0, 0, 1, 2, 3, 0] and seen[4] == [4, 3, 2, 0] and seen[1] == [1]
    rng = random.Random(0)
    tree = [-1] + [rng.randrange(i) for i in range(1, 40)]
    assert all(len(w) == min(d + 1, 3) for w, d in zip(*plain.ways(tree, 3)))
