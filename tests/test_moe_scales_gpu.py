"""The expert layer where a block's scale is infinite."""
import pytest
import torch

from _moe import INF, expert_weights, routing_of
from h3_tp2_amd import ops

pytestmark = pytest.mark.gpu
E4M3, BF16, FP16 = torch.float8_e4m3fn, torch.bfloat16, torch.float16


# T, E, k, H, F: a token, few; 16 rows; 32 rows; two groups of waves
@pytest.mark.parametrize("T,E,k,H,F", [(1, 4, 2, 272, 272), (6, 4, 1, 272, 272), (20, 4, 2, 272, 272), (90, 3, 2, 272, 656), (40, 3, 1, 1552, 1680)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_an_infinite_scale_of_the_last_block(cuda, T, E, k, H, F, dtype):
    """Positive codes and tokens: a block's infinite scale makes its expert's results +inf, in the last block of K (behind which the
    units of a kernel are rounded up) as in the first."""
    g = torch.Generator(device=cuda).manual_seed(T)
    w1, s1, w2, s2 = (*expert_weights(g, E, 2 * F, H, cuda), *expert_weights(g, E, H, F, cuda))
    w1, w2 = ((w.float().abs() + 1.0).to(E4M3) for w in (w1, w2))
    x = (torch.rand(T, H, generator=g, device=cuda) + 0.25).to(dtype)
    experts = (torch.arange(T * k, dtype=torch.int32) % E).view(T, k)
    r = routing_of(ops, experts, torch.rand(T, k, generator=g, device=cuda) + 0.5, E)
    s1, s2 = s1 * 0.1, s2 * 0.1
    y = ops.moe_blocks(x, w1, s1, w2, s2, r)
    assert bool(torch.isfinite(y).all())
    hit = (r.experts == 0).any(dim=1)
    assert bool(hit.any())
    for which in ("s1", "s2"):
        for block in (0, -1):
            a, b = s1.clone(), s2.clone()
            (a if which == "s1" else b)[0, :, block] = INF
            z = ops.moe_blocks(x, w1, a, w2, b, r)
            assert torch.equal(z[~hit], y[~hit]), (which, block)
            assert bool((z[hit] == INF).all()), (which, block)
