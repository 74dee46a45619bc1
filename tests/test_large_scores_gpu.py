"""Scores far beyond those of trained models: where a query sees one key its weight is 1, however large the score, and two keys of equal scores share alike."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# products q . k: just above (below) what 16 bits hold, where a maximum rounded up to 16 bits lies furthest above all scores
SCORES = [(512.0, 256.0, 1.0), (512.0, -256.0, -1020.0), (2048.0, 128.0, 56.0), (2.0 ** 14, 2.0 ** 12, 255 * 2.0 ** 11), (2.0 ** 14, -2.0 ** 12, -255 * 2.0 ** 11)]


@pytest.mark.parametrize("q0,k0,k1", SCORES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (4, 1, 128), (16, 8, 128)])
@pytest.mark.parametrize("path", ["one page a step", "two pages a step", "chosen", "mma", "kept"])
def test_one_and_two_keys(path, heads, kv_heads, dim, q0, k0, k1):
    from sleuth_b200.kernels import ops
    bf, g = torch.bfloat16, torch.Generator().manual_seed(5)
    past, counts = [0, 70, 333], [200, 131, 64]
    n, T, stride = 3, sum(counts), 8
    q = torch.zeros((T, heads, dim), dtype=bf)
    q[..., 0], q[..., 1] = q0, 1.0
    k = torch.zeros((n * stride, kv_heads, 64, dim), dtype=bf)
    k[..., 0], k[..., 1] = k0, k1
    v = torch.randn((n * stride, kv_heads, 64, dim), generator=g).to(bf)
    table = torch.randperm(n * stride, generator=g).to(torch.int32).view(n, stride)
    starts = [0, 200, 331, 395]
    args = [x.to(DEV) for x in (q, k, v)]
    for window in (1, 2):
        out = torch.full((T, heads * dim), 7.0, dtype=bf, device=DEV)
        tables = (i32(starts), i32(past), i32(counts), table.to(DEV), max(counts), heads, kv_heads, dim, window)
        scale = dim ** -0.5
        if path == "mma":
            ops.attention_prefill(*args, out, *tables, scale)
        elif path == "kept":
            floats = ops.attention_kept_scratch_floats(T, n, max(counts), heads, kv_heads, dim, stride * 64, bf)
            ops.attention_kept(*args, out, *tables, 0, scale, scratch=torch.zeros(max(1, floats), device=DEV))
        else:
            ops.attention_tc(*args, out, *tables, scale, wide={"one page a step": False, "two pages a step": True, "chosen": None}[path])
        ops.gemm_tc_check(DEV)
        got = out.cpu().double().view(T, heads, dim)
        for s in range(n):
            rows = torch.arange(past[s] + counts[s])
            values = v[table[s, rows // 64].long(), :, rows % 64].double()      # [rows, kv_heads, dim]
            if window == 2:
                values[1:] = (values[1:] + values[:-1]) / 2
            want = values[past[s]:].repeat_interleave(heads // kv_heads, 1)
            # bfloat16 weights and results: half a step (2^-8) each
            err = (got[starts[s]:starts[s + 1]] - want).abs()
            assert bool((err <= ((1 + 2.0 ** -8) ** 2 - 1 + 2.0 ** -16) * want.abs() + 1e-30).all()), (window, s, float(err.max()))
