"""The operators of a cache of bounded size at the ends of their arguments' ranges."""

import math

import pytest
import torch

from plain import kept_plain as plain
from test_kept_gpu import DEV, Step

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1
KINDS = [(torch.float32, 6, 3, 24), (torch.float32, 8, 2, 64), (torch.bfloat16, 4, 2, 64), (torch.bfloat16, 16, 8, 128), (torch.bfloat16, 6, 2, 128)]
KIND_IDS = [f"{str(d)[6:]}-{h}-{k}-{e}" for d, h, k, e in KINDS]


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("window,first", [(MOST, 4), (MOST - 150, 0), (MOST, MOST), (5, MOST), (40, MOST - 62), (MOST - 1, MOST - 63)])
@pytest.mark.parametrize("count", [1, 3, 200])
def test_largest_windows_and_first_rows(dtype, heads, kv_heads, dim, window, first, count):
    """A program says "no limit" with the largest number there is."""
    Step(dtype, heads, kv_heads, dim, [0, 70, 131], [count, 1, count], window, first, seed=11).check(weights=True, lse=True, promise=count != 3)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts", [[1, 1], [3, 2], [150, 70]])
def test_largest_promise_of_new_tokens(dtype, heads, kv_heads, dim, counts):
    """``max_count`` and ``max_keys`` are upper limits: the largest numbers there are say nothing, and cost no result."""
    from sleuth_b200.kernels import ops
    step = Step(dtype, heads, kv_heads, dim, [90, 3], counts, 60, 5, seed=12)
    t = step.tensors()
    out = torch.empty((step.T, heads * dim), dtype=dtype, device=DEV)
    w = step.weights.to(DEV)
    floats = ops.attention_kept_scratch_floats(step.T, 2, MOST, heads, kv_heads, dim, 64 * step.stride, dtype, weights=True)
    ops.attention_kept(t["q"], t["k"], t["v"], out, t["seq_start"], t["past"], t["counts"], t["table"], MOST, heads, kv_heads, dim, 60, 5, step.scale,
                       scratch=torch.empty(max(1, floats), device=DEV), max_keys=MOST, weights=w)
    want, _, _, want_w = plain.attention(step.q, step.k, step.v, step.seq_start, step.past, step.counts, step.table, heads, kv_heads, 60, 5, step.scale, step.weights)
    # (the same bounds as in the tests of the sizes in between)
    _, _, size, _ = plain.attention(step.q, step.k, step.v, step.seq_start, step.past, step.counts, step.table, heads, kv_heads, 60, 5, step.scale)
    rel = 2.0 ** -7 if dtype == torch.bfloat16 else 5e-5
    assert bool(((out.cpu().view(want.shape).double() - want).abs() <= rel * size + 1e-12).all())
    for s, (p, c) in enumerate(zip(step.past, step.counts)):
        assert bool(((w[s, :, :p + c].cpu().double() - want_w[s, :, :p + c]).abs() <= 5e-5 * want_w[s, :, :p + c].abs() + 1e-7).all())
