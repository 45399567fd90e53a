"""Calls of the NVFP4 operators that were answered wrongly once, or could be."""
import pytest
import torch

from test_gpu_fp4 import DEV
from test_gpu_fp4_moe import case, oracle, run

gpu = pytest.mark.gpu


# ---- rows of a few tokens one behind the other ----------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("T,k,dtype", [(2, 4, torch.bfloat16), (3, 4, torch.float32), (4, 4, torch.bfloat16), (4, 8, torch.float32)])
def test_few_tokens_without_a_norm_keep_their_own_scales(T, k, dtype):
    """Rows of very different sizes: a maximum of the row behind taken for a row's own would be far off.  Every row as if it were alone,
    bit for bit and every time."""
    c = case(T, 16, k, 256, 2048, seed=40 + T, dtype=dtype)
    x = c[0]
    x *= torch.tensor([2.0 ** (9 * (t % 2) - 3 * t) for t in range(T)], device=DEV)[:, None]
    want, tol = oracle(*c[:3], *(w[1] for w in c[3:]))
    tol = tol + (k + 1) * 2.0 ** -24 * want.abs()
    alone = torch.empty(T, 2048, device=DEV)
    for t in range(T):
        run(x[t:t + 1], c[1][t:t + 1], c[2][t:t + 1], *c[3:], out_f32=alone[t:t + 1])
    assert bool(((alone.double().cpu() - want).abs() <= tol).all())
    out, work = torch.empty(T, 2048, device=DEV), None
    for _ in range(40):
        work = run(*c, work=work, out_f32=out)
        assert torch.equal(out, alone)
