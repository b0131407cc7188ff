"""The router's weights at the ends of their range: logits whose sigmoid fp32 cannot hold, scores that a sum of 512 terms brings off."""
import pytest
import torch

from _moe import INF, route64
from h3_tp2_amd import ops
from test_moe_gpu import same_route

pytestmark = pytest.mark.gpu
BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("E,k", [(20, 4), (300, 4), (64, 12), (8, 8)])
@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
def test_sigmoid_of_far_logits(cuda, E, k, dtype):
    """Rows around -60 to -1000, among them those where fp32 has subnormals (-87 to -104), nothing (below), and where float64 ends
    (-709.78): the quotients are ordinary numbers up to there, with a bias of zeros and without one.  An argument x - max below 32
    in size is rounded by 2^-20 at most, on top of same_route's."""
    g = torch.Generator(device=cuda).manual_seed(E)
    base = torch.tensor([0.0, -60.0, -86.0, -88.0, -90.0, -97.0, -104.0, -150.0, -300.0, -500.0, -700.0, -708.0, -712.0, -1000.0], device=cuda)
    x = (base.repeat_interleave(5)[:, None] + 2.0 * torch.randn(5 * base.numel(), E, generator=g, device=cuda)).to(dtype)
    x[::5, ::2] = -INF
    for renorm in (True, False):
        for bias in (None, torch.zeros(E, device=cuda)):
            kw = dict(scoring="sigmoid", renormalize=renorm, scale=2.5, bias=bias)
            same_route(ops.moe_route(x, k, **kw), route64(x, k, **kw), x)


def test_sigmoid_where_float64_ends(cuda):
    """exp(-x) is infinite in float64 from -709.78271484375 on, the next fp32 number it is not: a score of zero, and a weight of it."""
    end = -709.78271484375
    before = torch.tensor(end).nextafter(torch.tensor(0.0)).item()
    x = torch.tensor([[end, before, -720.0], [end, -720.0, end], [before, end, 3.0], [before, before, -INF]], device=cuda)
    for bias in (None, torch.zeros(3, device=cuda)):
        r = ops.moe_route(x, 2, "sigmoid", bias=bias)
        same_route(r, route64(x, 2, "sigmoid", bias=bias), x)
        assert r.weights.tolist() == [[1.0, 0.0], [0.0, 0.0], [1.0, 0.0], [0.5, 0.5]]


@pytest.mark.parametrize("at", [0, 5, 130, 511])
@pytest.mark.parametrize("below", [16.65, 8.0])
def test_route_with_bias_near_ties_of_512(cuda, at, below):
    """One logit that outweighs 511 others, whose terms the fp32 sum rounds away, and a bias that makes scores equal but for its own
    rounding: of some ten experts, of a third, and of all."""
    g = torch.Generator(device=cuda).manual_seed(at)
    E = 512
    x = 0.01 * torch.randn(5, E, generator=g, device=cuda) - below
    x[:, at] = 0.0
    score = torch.softmax(x.double(), 1)
    near = torch.arange(E, device=cuda)
    for row in range(5):
        bias = (0.75 - score[row]).float()
        for keep in (near % 57 == at % 57, near % 3 == at % 3, near >= 0):
            for k in (4, 8, 16):
                kw = dict(scoring="softmax", bias=torch.where(keep, bias, bias - 1.0))
                same_route(ops.moe_route(x, k, **kw), route64(x, k, **kw), x)
