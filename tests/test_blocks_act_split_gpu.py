"""The product with an epilogue where its tiles fill whole rounds on the CUs, or leave a few: no row outside the output."""
import pytest
import torch

from _blocks import codes, plan, scales
from h3_tp2_amd import ops
from test_blocks_act_split import first_rows

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
GUARD = 264                     # rows behind the output: more than a row tile


# whole rounds with a ragged last row tile, with a full one, and up to half a round left over
@pytest.mark.parametrize("M,N,K", [(4000, 4096, 144), (4090, 4096, 144), (4096, 4096, 144), (8000, 6144, 128), (8000, 14336, 128), (2000, 8192, 272),
                                   (1000, 16384, 128), (6144, 4096, 144), (6145, 4096, 144), (6100, 4096, 144), (6200, 5376, 144)])
def test_rows_behind_the_output_stay(cuda, M, N, K):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert 0 < first_rows(M, N, cus) <= M and (cus != 256 or plan(M, N)[:2] == (256, 256))
    g = torch.Generator(device=cuda).manual_seed(M + N)
    a, w = codes(g, M, K), codes(g, N, K)
    sa, sw = scales(g, M, -(-K // 128)), scales(g, -(-N // 128), -(-K // 128))
    bias = torch.randn(N, generator=g, device=cuda).to(BF16)
    product = ops.gemm_blocks(a, w, sa, sw, BF16, bias)
    buf = torch.full((M + GUARD, N), 7.0, device=cuda, dtype=BF16)
    ops.gemm_blocks_act(a, w, sa, sw, BF16, bias, out=buf[:M])
    torch.cuda.synchronize()
    assert torch.equal(buf[:M], product) and bool((buf[M:] == 7.0).all())
    # onto a residual that is the output; past it, the residual's buffer has other values too
    ref = ops.gemm_blocks_act(a, w, sa, sw, BF16, bias, "relu")
    res = torch.randn(M, N, generator=g, device=cuda).to(BF16)
    buf[:M] = res
    ops.gemm_blocks_act(a, w, sa, sw, BF16, bias, "relu", buf[:M], out=buf[:M])
    torch.cuda.synchronize()
    assert bool((buf[M:] == 7.0).all())
    # ref is off the fp32 relu by half a step, 2^-8 of ref; the output off its sum with the residual by 2^-8 of that sum
    want = ref.double() + res.double()
    tol = 2.0 ** -8 * (1 + 2.0 ** -7) * (ref.double().abs() + want.abs())
    assert bool(((buf[:M].double() - want).abs() <= tol).all())
