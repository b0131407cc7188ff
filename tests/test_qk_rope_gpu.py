"""RMSNorm of queries and keys with the position rotation against float64 (GPU)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
EPS = 1e-6


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def table(P, R, device="cuda"):
    ang = torch.arange(P, device=device)[:, None].double() * torch.exp(-torch.arange(R // 2, device=device).double() * 9.0 / max(1, R // 2))
    return torch.cat((ang.cos(), ang.sin()), 1).float()


def ref64(x, w, tab, interleaved, eps=EPS):
    """(the definition, the sum of the magnitudes of its terms) in float64."""
    n = x.double() / torch.sqrt(x.double().square().mean(2, keepdim=True) + eps) * w.double()
    h = tab.shape[1] // 2
    c, s = tab[:, None, :h].double(), tab[:, None, h:].double()
    y, mag = n.clone(), n.abs()
    if interleaved:
        ia, ib = slice(0, 2 * h, 2), slice(1, 2 * h, 2)
    else:
        ia, ib = slice(0, h), slice(h, 2 * h)
    a, b = n[..., ia], n[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


def check(y, y64, mag):
    """One rounding to the type; in fp32 before it: the sum of squares of up to 256 terms in at most 8 + 5 roundings, the mean,
    the square root, the reciprocal, two products and the rotation's fma and product, under 32 roundings of 2^-24."""
    f = torch.finfo(y.dtype)
    tol = y64.abs() * (f.eps / 2) + mag * 2.0 ** -19 + f.smallest_normal * f.eps
    bad = ~((y.double() - y64).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,H,Hk,D,R,inter", [
    (1, 1, 1, 64, 64, False), (1, 32, 8, 128, 128, False), (2, 5, 1, 128, 96, False), (7, 3, 2, 256, 192, False),
    (8, 56, 56, 128, 96, False), (33, 9, 3, 64, 32, False), (5, 16, 4, 128, 128, True), (6, 4, 4, 64, 34, True),
    (3, 7, 7, 256, 256, True), (4, 8, 2, 128, 0, False), (130, 6, 2, 64, 48, False), (1025, 2, 1, 128, 64, True)])
@pytest.mark.parametrize("tdt", [torch.float32, BF16])
def test_qk_norm_rope(cuda, T, H, Hk, D, R, inter, dtype, tdt):
    from h3_tp2_amd import ops
    g = gen(T + H + D)
    qkv = (torch.randn(T, (H + 2 * Hk) * D, generator=g, device=cuda) * torch.exp(torch.randn(T, 1, generator=g, device=cuda))).to(dtype)
    q, k = qkv[:, :H * D].view(T, H, D), qkv[:, H * D:(H + Hk) * D].view(T, Hk, D)
    wq, wk = (1 + 0.2 * torch.randn(2, D, generator=g, device=cuda)).to(dtype)
    tab = table(T, R).to(tdt)
    before = qkv.clone()
    oq, ok = ops.qk_norm_rope(q, k, wq, wk, tab, EPS, interleaved=inter)
    assert torch.equal(qkv, before)
    for o, x, w in ((oq, q, wq), (ok, k, wk)):
        check(o, *ref64(x, w, tab, inter))
    # positions: int32 and int64, strided, the same one twice
    P = 50
    tab = table(P, R).to(tdt)
    pos = torch.randint(0, P, (T,), generator=g, device=cuda)
    pos[-1] = pos[0]
    if R:
        oq, ok = ops.qk_norm_rope(q, k, wq, wk, tab, EPS, positions=pos, interleaved=inter)
        check(oq, *ref64(q, wq, tab[pos], inter))
        check(ok, *ref64(k, wk, tab[pos], inter))
        p32 = torch.stack((pos, pos * 0 - 1), 1).int()[:, 0]
        o2 = ops.qk_norm_rope(q, k, wq, wk, tab, EPS, positions=p32, interleaved=inter)
        assert torch.equal(o2[0], oq) and torch.equal(o2[1], ok)
    # in place, on the product itself: the v columns stay
    ops.qk_norm_rope(q, k, wq, wk, tab, EPS, positions=pos, interleaved=inter, out=(q, k))
    if R:
        assert torch.equal(q, oq) and torch.equal(k, ok)
    assert torch.equal(qkv[:, (H + Hk) * D:], before[:, (H + Hk) * D:])


@pytest.mark.parametrize("inter", [False, True])
def test_positions_outside_the_table(cuda, inter):
    from h3_tp2_amd import ops
    g = gen(1)
    q, k = torch.randn(5, 3, 128, generator=g, device=cuda).to(BF16), torch.randn(5, 1, 128, generator=g, device=cuda).to(BF16)
    w = torch.ones(128, device=cuda, dtype=BF16)
    tab = table(10, 96)
    pos = torch.tensor([0, -1, 9, 10, 2 ** 40], device=cuda)
    oq, ok = ops.qk_norm_rope(q, k, w, w, tab, EPS, positions=pos, interleaved=inter)
    for o, x in ((oq, q), (ok, k)):
        assert o[[1, 3, 4]].isnan().all()
        check(o[[0, 2]], *ref64(x[[0, 2]], w, tab[[0, 9]], inter))


def test_directed_heads(cuda):
    """A zero head (eps alone), a tiny one, and one with inf or NaN, which stays in its head."""
    from h3_tp2_amd import ops
    x = torch.randn(1, 6, 128, generator=gen(2), device=cuda)
    x[0, 0] = 0
    x[0, 1] *= 1e-20
    x[0, 2, 5] = float("inf")
    x[0, 3, 7] = float("nan")
    q = x.to(BF16)
    w = torch.ones(128, device=cuda, dtype=BF16)
    tab = table(1, 96)
    oq, ok = ops.qk_norm_rope(q, q.clone(), w, w, tab, EPS)
    assert torch.equal(oq.view(torch.int16), ok.view(torch.int16))
    assert (oq[0, 0] == 0).all() and oq[0, 3].isnan().all() and oq[0, 2, 5].isnan()
    keep = [0, 1, 4, 5]
    check(oq[:, keep], *ref64(q[:, keep], w, tab, False))


def test_empty(cuda):
    from h3_tp2_amd import ops
    z = lambda *s: torch.zeros(s, device=cuda, dtype=BF16)             # noqa: E731
    oq, ok = ops.qk_norm_rope(z(0, 4, 128), z(0, 2, 128), z(128), z(128), table(0, 128), EPS)
    assert oq.shape == (0, 4, 128) and ok.shape == (0, 2, 128)
    oq, ok = ops.qk_norm_rope(z(3, 4, 128), z(3, 0, 128), z(128), z(128), table(3, 128), EPS)
    assert oq.shape == (3, 4, 128) and ok.shape == (3, 0, 128)


def test_captured(cuda):
    from h3_tp2_amd import ops
    g = gen(3)
    q, k = torch.randn(9, 8, 128, generator=g, device=cuda).to(BF16), torch.randn(9, 2, 128, generator=g, device=cuda).to(BF16)
    w = torch.ones(128, device=cuda, dtype=BF16)
    tab, pos = table(64, 128), torch.zeros(9, dtype=torch.int64, device=cuda)
    out = (torch.empty_like(q), torch.empty_like(k))
    ops.qk_norm_rope(q, k, w, w, tab, EPS, positions=pos, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.qk_norm_rope(q, k, w, w, tab, EPS, positions=pos, out=out)
    for i in range(3):
        pos.copy_(torch.arange(9, device=cuda) + i)
        graph.replay()
        torch.cuda.synchronize()
        r = ops.qk_norm_rope(q, k, w, w, tab, EPS, positions=pos)
        assert torch.equal(out[0], r[0]) and torch.equal(out[1], r[1])


def test_subnormal_mean_square(cuda):
    """A mean square below the normal fp32 range (2^-130, exact) without eps: the norm is still 1."""
    from h3_tp2_amd import ops
    sign = torch.where(torch.rand(9, 4, 128, generator=gen(5), device=cuda) < 0.5, -1.0, 1.0)
    q = (sign * 2.0 ** -65).to(BF16)
    w = (1 + 0.1 * torch.randn(128, generator=gen(6), device=cuda)).to(BF16)
    tab = table(9, 96)
    oq, ok = ops.qk_norm_rope(q, q.clone(), w, w, tab, 0.0)
    y64, mag = ref64(q, w, tab, False, eps=0.0)
    check(oq, y64, mag)
    assert torch.equal(oq, ok)


def test_only_keys(cuda):
    """No query heads at all: k alone, at head counts around a wave's pass."""
    from h3_tp2_amd import ops
    w, tab = torch.randn(64, generator=gen(8), device=cuda).to(BF16), table(70, 64)
    for Hk in (1, 8, 9, 17):
        k = torch.randn(70, Hk, 64, generator=gen(Hk), device=cuda).to(BF16)
        oq, ok = ops.qk_norm_rope(k[:, :0], k, w, w, tab, EPS, interleaved=True)
        assert oq.shape == (70, 0, 64)
        check(ok, *ref64(k, w, tab, True))
