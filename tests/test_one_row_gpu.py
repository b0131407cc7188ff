"""A residual of a single row, whose stride says nothing."""
import pytest
import torch

from _blocks import codes, scales
from _moe import expert_weights
from h3_tp2_amd import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_a_residual_of_one_row_in_any_stride(cuda, monkeypatch):
    """The stride of a single row is never used: natively and from Python alike."""
    g = torch.Generator(device=cuda).manual_seed(3)
    E, H, F, N, K = 4, 272, 144, 272, 144
    w1, s1, w2, s2 = (*expert_weights(g, E, 2 * F, H, cuda), *expert_weights(g, E, H, F, cuda))
    x = torch.randn(1, H, generator=g, device=cuda).to(BF16)
    r = ops.moe_route(torch.randn(1, E, generator=g, device=cuda), 2)
    a, w, sa, sw = codes(g, 1, K), codes(g, N, K), scales(g, 1, 2), scales(g, 3, 2)
    wide = torch.randn(3, H + 2, generator=g, device=cuda).to(BF16)
    res = wide[:1, :H]
    assert res.stride(0) == H + 2

    def calls(residual):
        return (ops.moe_blocks(x, w1, s1, w2, s2, r, residual=residual), ops.gemm_blocks_act(a, w, sa, sw, BF16, None, "silu", residual))
    want = calls(res.contiguous())
    for host in (ops._host, None):
        monkeypatch.setattr(ops, "_host", host)
        assert all(torch.equal(p, q) for p, q in zip(calls(res), want))
