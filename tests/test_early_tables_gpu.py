"""Prompt attention begins while the kernel in front still runs: tables that this one writes count as they are afterwards."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("path", ["one page a step", "two pages a step", "kept"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (16, 8, 128)])
def test_past_from_the_kernel_in_front(path, heads, kv_heads, dim):
    from sleuth_b200.kernels import ops
    bf, g = torch.bfloat16, torch.Generator().manual_seed(6)
    past, counts, starts, stride = [0, 70, 333, 500], [200, 131, 64, 0], [0, 200, 331, 395, 395], 10
    n, T = len(past), sum(counts)
    q = torch.randn((T, heads, dim), generator=g).to(bf).to(DEV)
    k, v = (torch.randn((n * stride, kv_heads, 64, dim), generator=g).to(bf).to(DEV) for _ in range(2))
    table = torch.randperm(n * stride, generator=g).to(torch.int32).view(n, stride).to(DEV)
    starts, counts_d, out = i32(starts), i32(counts), torch.empty((T, heads * dim), dtype=bf, device=DEV)
    floats = ops.attention_kept_scratch_floats(T, n, max(counts), heads, kv_heads, dim, stride * 64, bf)
    scratch = torch.zeros(max(1, floats), device=DEV)

    def attention(past_d):
        args = (q, k, v, out, starts, past_d, counts_d, table, max(counts), heads, kv_heads, dim, 100)
        if path == "kept":
            ops.attention_kept(*args, 5, dim ** -0.5, scratch=scratch)
        else:
            ops.attention_tc(*args, dim ** -0.5, wide=path == "two pages a step")

    attention(i32(past))
    wanted = out.clone()
    # positions of trees of one node each are the numbers of rows before the step
    parents, places, ones, before, bits, positions = i32([-1] * n), i32(list(range(n))), i32([1] * n), i32(past), torch.zeros((n, 1), dtype=torch.int32, device=DEV), i32([0] * n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            ops.draft_tree(parents, places, before, ones, bits, positions, 1)
            attention(positions)
    for again in range(20):
        positions.fill_(again % 5)
        out.fill_(7.0)
        graph.replay()
        ops.gemm_tc_check(DEV)
        assert torch.equal(out, wanted), again
