"""The block-scaled product with bias, activation and residual in its epilogue against float64."""
import pytest
import torch

from _blocks import codes, plan, product64, scales
from h3_tp2_amd import ops

pytestmark = pytest.mark.gpu
E4M3, BF16, FP16 = torch.float8_e4m3fn, torch.bfloat16, torch.float16
ACTS = (None, "silu", "gelu", "gelu_tanh", "relu")
# every form of the dense rule on 256 CUs, with edges in rows, channels and K; the last two in whole rounds and a rest
SHAPES = [(1, 400, 272), (16, 1040, 400), (30, 13008, 144), (40, 1296, 528), (100, 5376, 256), (200, 5376, 272), (256, 8208, 144), (500, 5376, 400),
          (1000, 5376, 272), (2100, 5376, 144), (4100, 5376, 128), (6200, 5376, 272)]


def act64(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * torch.special.erfc(-v / 2.0 ** 0.5)
    if act == "gelu_tanh":
        return v * torch.sigmoid(2.0 * (2.0 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    return v.clamp_min(0.0) if act == "relu" else v


def check(y, v64, mag, act, res, dtype):
    """One rounding to the output's type; the product's bound (2^-12 of the sum of magnitudes, what an MFMA leaves out) through an
    activation whose slope is at most 1.13; the activation's own 2^-16 (exponential, reciprocal and polynomial, at most 2^-17)."""
    f = act64(v64, act)
    y64 = f if res is None else f + res.double()
    own = mag * (1.13 * 2.0 ** -12) + f.abs() * 2.0 ** -16
    tol = (y64.abs() + own) * (torch.finfo(dtype).eps / 2) + own + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = ~((y.double() - y64).abs() <= tol)
    assert not bad.any(), (act, int(bad.sum()), bad.nonzero()[:3].tolist())


def test_the_shapes_take_every_form():
    forms = {plan(M, N)[2] for M, N, _ in SHAPES}
    assert forms == {plan(int(2 ** (i / 4)), n)[2] for i in range(64) for n in (400, 1296, 5376, 8208, 13008, 21504)}


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_epilogues(cuda, M, N, K, dtype):
    g = torch.Generator(device=cuda).manual_seed(M + N)
    a, w = codes(g, M, K), codes(g, N, K)
    sa, sw = scales(g, M, -(-K // 128)) * 0.05, scales(g, -(-N // 128), -(-K // 128)) * 0.05
    bias = torch.randn(N, generator=g, device=cuda).to(dtype)
    res = (torch.randn(M, N, generator=g, device=cuda) * 3.0).to(dtype)
    v, mag = product64(a, w, sa, sw)
    for i, act in enumerate(ACTS):
        for b, r in ((bias, None), (None, res)) if i else ((bias, res), (None, None)):
            y = ops.gemm_blocks_act(a, w, sa, sw, dtype, b, act, r)
            check(y, v if b is None else v + b.double(), mag, act, r, dtype)
    assert torch.equal(ops.gemm_blocks_act(a, w, sa, sw, dtype, bias), ops.gemm_blocks(a, w, sa, sw, dtype, bias))
    assert torch.equal(ops.gemm_blocks_act(a, w, sa, sw, dtype), ops.gemm_blocks(a, w, sa, sw, dtype))
    out = res.clone()
    want = ops.gemm_blocks_act(a, w, sa, sw, dtype, bias, "gelu", res)
    assert ops.gemm_blocks_act(a, w, sa, sw, dtype, bias, "gelu", out, out=out) is out and torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", ACTS[1:])
def test_activation_values(cuda, dtype, act):
    """Every finite value of the type through the bias of a product that is zero: the activation to 2^-16 and one rounding (results
    below 2^-126, where fp32 itself is subnormal, to 2^-140); infinities and NaN as the formulas give them."""
    bits = torch.arange(65536, device=cuda, dtype=torch.int32).to(torch.int16).view(dtype)
    a, w = torch.zeros(1, 16, device=cuda).to(E4M3), torch.zeros(65536, 16, device=cuda).to(E4M3)
    y = ops.gemm_blocks_act(a, w, torch.ones(1, 1, device=cuda), torch.ones(512, 1, device=cuda), dtype, bits, act)[0]
    v = bits.double()
    ref = act64(v, act)
    ref = torch.where((v == v) & v.isfinite() & ~ref.isfinite(), torch.where(v > 0, v, 0.0), ref)        # the cube's overflow
    fin = bits.isfinite()
    info = torch.finfo(dtype)
    tol = ref.abs() * (info.eps / 2 * (1 + 2.0 ** -10) + 2.0 ** -16) + info.smallest_normal * info.eps / 2 * 1.01 + 2.0 ** -140
    bad = ~((y.double() - ref).abs() <= tol) & fin
    assert not bad.any(), (int(bad.sum()), v[bad][:5].tolist(), y[bad][:5].tolist(), ref[bad][:5].tolist())
    assert bool(torch.isnan(y[torch.isnan(bits)]).all())
    pos, neg = y[bits == float("inf")], y[bits == -float("inf")]
    assert bool((pos == float("inf")).all())
    assert bool((neg == 0).all()) if act == "relu" else bool((torch.isnan(neg) | (neg == 0)).all())


def test_strides(cuda):
    g = torch.Generator(device=cuda).manual_seed(8)
    for M, N, K in ((5, 272, 144), (300, 1040, 272), (2100, 5376, 144), (6200, 5376, 144)):
        a, w = codes(g, M, K), codes(g, N, K)
        sa, sw = scales(g, M, -(-K // 128)), scales(g, -(-N // 128), -(-K // 128))
        wide = torch.randn(M, 2 * N + 16, generator=g, device=cuda).to(BF16)
        out = torch.full((M + 1, N + 24), 7.0, device=cuda, dtype=BF16)
        res = wide[:, 8:8 + N]
        want = ops.gemm_blocks_act(a, w, sa, sw, BF16, None, "silu", res.contiguous())
        y = ops.gemm_blocks_act(a, w, sa, sw, BF16, None, "silu", res, out=out[:M, 16:16 + N])
        assert torch.equal(y, want)
        assert bool((out[M] == 7.0).all()) and bool((out[:, :16] == 7.0).all()) and bool((out[:, 16 + N:] == 7.0).all())
        one = res[:1].expand(M, N)
        assert torch.equal(ops.gemm_blocks_act(a, w, sa, sw, BF16, None, "relu", one), ops.gemm_blocks_act(a, w, sa, sw, BF16, None, "relu", one.contiguous()))


def test_offsets_past_32_bits(cuda):
    g = torch.Generator(device=cuda).manual_seed(10)
    M, N, K = 2200, 5376, 128
    a, w = codes(g, M, K), codes(g, N, K)
    sa, sw = scales(g, M, 1), scales(g, N // 128, 1)
    res = torch.empty(M, 1 << 20, dtype=BF16, device=cuda)[:, :N]
    res.copy_(torch.randn(M, N, generator=g, device=cuda))
    for m in (M, 300):
        want = ops.gemm_blocks_act(a[:m], w, sa[:m], sw, BF16, None, "silu", res[:m].contiguous())
        out = torch.empty(m, 1 << 20, dtype=BF16, device=cuda)[:, :N]
        assert torch.equal(ops.gemm_blocks_act(a[:m], w, sa[:m], sw, BF16, None, "silu", res[:m], out=out), want)


def test_captured_on_streams_and_natively(cuda, monkeypatch):
    g = torch.Generator(device=cuda).manual_seed(9)
    shapes = [(1, 1040, 272), (60, 1040, 400), (300, 5376, 256), (2100, 5376, 144), (6200, 5376, 144)]
    calls = []
    for M, N, K in shapes:
        a, w = codes(g, M, K), codes(g, N, K)
        sa, sw = scales(g, M, -(-K // 128)), scales(g, -(-N // 128), -(-K // 128))
        bias, res = torch.randn(N, generator=g, device=cuda).to(BF16), torch.randn(M, N, generator=g, device=cuda).to(BF16)
        calls.append(lambda a=a, w=w, sa=sa, sw=sw, bias=bias, res=res: ops.gemm_blocks_act(a, w, sa, sw, BF16, bias, "gelu_tanh", res))
    alone = [c() for c in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = [c() for c in calls]
    for _ in range(3):
        for y in ys:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, ys))
        calls[0]()
    streams = [torch.cuda.Stream() for _ in calls]
    out = [None] * len(calls)
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i] = calls[i]()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, out))
    monkeypatch.setattr(ops, "_host", None)
    assert all(torch.equal(a, c()) for a, c in zip(alone, calls))
