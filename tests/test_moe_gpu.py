"""The router and the layer of experts for a few tokens against their definitions in float64."""
import pytest
import torch

from _moe import INF, check, expert_weights, moe64, route64, routing_of
from h3_tp2_amd import ops

pytestmark = pytest.mark.gpu
BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


def same_route(r, ref, logits):
    """Whole numbers equal; a weight takes an exponential (2 ulp; its argument's rounding up to |x - max| 2^-24), a sum in fp32
    (at most 16 roundings on the way of an element) and three more roundings: |x| below 64 here, 128 * 2^-24 in all."""
    w, experts, offsets, order, place = ref
    assert torch.equal(r.experts.cpu(), experts)
    assert torch.equal(r.offsets.cpu(), offsets)
    assert torch.equal(r.order.cpu(), order)
    assert torch.equal(r.place.cpu(), place)
    assert r.weights.dtype == F32
    err = (r.weights.cpu().double() - w).abs()
    assert bool(((err <= w.abs() * 2.0 ** -17 + 1e-38) | (w != w) & (r.weights.cpu() != r.weights.cpu())).all()), float((err / w.abs().clamp_min(1e-30)).max())


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 32, 4), (3, 8, 8), (17, 60, 6), (64, 256, 8), (128, 64, 2), (129, 65, 3), (300, 512, 16),
                                   (1000, 100, 7), (257, 129, 16)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_route_softmax(cuda, T, E, k, dtype):
    g = torch.Generator(device=cuda).manual_seed(T * 31 + E)
    x = (torch.randn(T, E, generator=g, device=cuda) * 3.0).to(dtype)
    for renorm in (False, True):
        same_route(ops.moe_route(x, k, renormalize=renorm), route64(x, k, renormalize=renorm), x)


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (50, 256, 8), (200, 33, 5), (131, 300, 4)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [FP16, F32])
def test_route_with_bias(cuda, T, E, k, scoring, dtype):
    g = torch.Generator(device=cuda).manual_seed(T + E)
    x = (torch.randn(T, E, generator=g, device=cuda) * 2.0).to(dtype)
    bias = torch.randn(E, generator=g, device=cuda) * 0.1
    for renorm in (False, True):
        kw = dict(scoring=scoring, renormalize=renorm, scale=2.5, bias=bias)
        same_route(ops.moe_route(x, k, **kw), route64(x, k, **kw), x)
    same_route(ops.moe_route(x, k, scoring), route64(x, k, scoring), x)


@pytest.mark.parametrize("E", [5, 64, 200])
@pytest.mark.parametrize("bias", [False, True])
def test_route_ties_masks_and_nan(cuda, E, bias):
    """Equal logits, zeros of both signs, masked experts and whole masked rows, NaN, infinities, the type's lowest value."""
    g = torch.Generator(device=cuda).manual_seed(E)
    x = torch.randint(-2, 3, (150, E), generator=g, device=cuda).float()
    x[0] = 0.0
    x[1] = torch.tensor([0.0, -0.0], device=cuda).repeat(E)[:E]
    x[2] = -INF
    x[3, :] = -INF
    x[3, E // 2] = 1.0
    x[4, 1] = float("nan")
    x[5] = float("nan")
    x[6, ::2] = -INF
    x[7] = torch.finfo(F32).min
    x[8, 3] = -INF
    x[140:] = -INF
    b = torch.zeros(E, device=cuda) if bias else None
    for scoring in ("softmax", "sigmoid"):
        for renorm in (False, True):
            same_route(ops.moe_route(x, 4, scoring, renorm, bias=b), route64(x, 4, scoring, renorm, bias=b), x)
    r = ops.moe_route(x, 4, bias=b)
    assert bool((r.experts[2] == -1).all()) and bool((r.weights[2] == 0).all())
    assert r.experts[3].tolist() == [E // 2, -1, -1, -1] and r.weights[3].tolist() == [1.0, 0.0, 0.0, 0.0]
    assert bool(torch.isnan(r.weights[4]).all()) and 1 not in r.experts[4].tolist()
    if not bias:
        y = x[:10].clone()
        y[9, 2] = INF                                     # exp(inf - inf): no weights, but the expert is known
        r = ops.moe_route(y, 2)
        assert r.experts[9, 0] == 2 and bool(torch.isnan(r.weights[9]).any())


@pytest.mark.parametrize("E", [12, 16, 17, 40, 300])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_with_bias_near_ties(cuda, E, scoring):
    """Scores that the bias makes equal but for its own rounding: 64 bits tell them apart, whether up to 16 experts are that near
    or more."""
    g = torch.Generator(device=cuda).manual_seed(E)
    x = torch.randn(1, E, generator=g, device=cuda)
    score = torch.softmax(x.double(), 1) if scoring == "softmax" else torch.sigmoid(x.double())
    bias = (0.75 - score[0]).float()
    near = torch.arange(E, device=cuda) % 3 == 0
    for b in (bias, torch.where(near, bias, bias - 1.0)):
        kw = dict(scoring=scoring, bias=b)
        same_route(ops.moe_route(x, 4, **kw), route64(x, 4, **kw), x)
        two = torch.cat([x, x + 0.5, x])
        same_route(ops.moe_route(two, 4, **kw), route64(two, 4, **kw), two)


@pytest.mark.parametrize("E", [9, 100])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_with_bias_infinities(cuda, E, scoring):
    g = torch.Generator(device=cuda).manual_seed(E)
    x = torch.randn(12, E, generator=g, device=cuda)
    x[3, 4] = INF
    x[4, 2] = float("nan")
    x[5] *= 1e30
    x[6] = 1e38
    bias = 0.2 * torch.randn(E, generator=g, device=cuda)
    for at, v in ((0, INF), (1, -INF), (5, float("nan")), (7, 1e38)):
        b = bias.clone()
        b[at] = v
        b[at + 1] = v
        for b in (b, torch.full_like(b, v)):
            kw = dict(scoring=scoring, bias=b)
            same_route(ops.moe_route(x, 3, **kw), route64(x, 3, **kw), x)


def test_route_largest(cuda):
    """512 experts, 16 choices, both kinds of bias vectors and rows: those of 16 bytes and others."""
    g = torch.Generator(device=cuda).manual_seed(11)
    wide = torch.randn(150, 513, generator=g, device=cuda)
    wb = 0.1 * torch.randn(513, generator=g, device=cuda)
    for x, b in ((wide[:, :512].contiguous(), wb[:512].clone()), (wide[:, 1:], wb[1:]), (wide[:, :511].to(BF16), wb[:511])):
        for T in (120, 150):
            for scoring in ("softmax", "sigmoid"):
                for bias in (None, b):
                    kw = dict(scoring=scoring, renormalize=False, bias=bias)
                    same_route(ops.moe_route(x[:T], 16, **kw), route64(x[:T], 16, **kw), x)


def test_route_in_two_launches_captured(cuda):
    """Its counts live in a workspace that every replay fills anew."""
    x = torch.empty(3000, 40, device=cuda)
    x.normal_()
    ops.moe_route(x, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = ops.moe_route(x, 4), ops.moe_route(x[:700], 3, "sigmoid")
    for seed in range(4):
        x.normal_(generator=torch.Generator(device=cuda).manual_seed(seed))
        if seed == 2:
            x[:, :35] = -INF
        ea, eb = ops.moe_route(x, 4), ops.moe_route(x[:700], 3, "sigmoid")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip((*a, *b), (*ea, *eb)))


def test_route_strides_and_no_tokens(cuda):
    g = torch.Generator(device=cuda).manual_seed(5)
    wide = torch.randn(40, 77, generator=g, device=cuda).to(BF16)
    x = wide[:, 3:63]
    same_route(ops.moe_route(x, 3), route64(x, 3), x)
    same_route(ops.moe_route(wide[:1].expand(9, 77), 5), route64(wide[:1].expand(9, 77), 5), x)
    r = ops.moe_route(wide[:0], 4)
    assert r.offsets.tolist() == [0] * 78 and r.weights.shape == (0, 4) and r.order.numel() == 0


@pytest.mark.parametrize("T", [20000, 70000])
def test_route_many_tokens(cuda, T):
    """More than one workgroup, and more than one batch in each: the order is a stable sort."""
    g = torch.Generator(device=cuda).manual_seed(T)
    E, k = 48, 6
    x = torch.randn(T, E, generator=g, device=cuda) + torch.randn(E, generator=g, device=cuda)
    x[::7] = -INF
    r = ops.moe_route(x, k)
    top = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k].int()
    top[::7] = -1
    assert torch.equal(r.experts, top)
    flat = torch.where(top < 0, E, top).view(-1).long()
    order = torch.sort(flat, stable=True)[1]
    assert torch.equal(r.order.long(), order)
    assert torch.equal(r.order.long()[r.place.view(-1).long()], torch.arange(T * k, device=cuda))
    assert torch.equal(r.offsets[1:].long(), torch.bincount(flat, minlength=E + 1)[:E].cumsum(0)) and r.offsets[0] == 0


# ---- the layer ----

def layer(g, E, H, F, cuda):
    return (*expert_weights(g, E, 2 * F, H, cuda), *expert_weights(g, E, H, F, cuda))


@pytest.mark.parametrize("T,E,k,H,F", [(1, 1, 1, 16, 16), (1, 8, 2, 256, 128), (2, 4, 4, 400, 272), (5, 6, 2, 1200, 1040), (16, 16, 4, 512, 384),
                                       (17, 3, 2, 144, 80), (32, 12, 3, 1040, 528), (33, 5, 1, 256, 640), (64, 8, 8, 272, 256), (65, 4, 2, 528, 144),
                                       (100, 70, 6, 160, 208), (128, 5, 3, 384, 400)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_layer(cuda, T, E, k, H, F, dtype):
    g = torch.Generator(device=cuda).manual_seed(T * 7 + H)
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    x = torch.randn(T, H, generator=g, device=cuda).to(dtype)
    r = ops.moe_route(torch.randn(T, E, generator=g, device=cuda), k)
    res = torch.randn(T, H, generator=g, device=cuda).to(dtype)
    for residual in (None, res):
        y = ops.moe_blocks(x, w1, s1, w2, s2, r, residual=residual)
        assert y.shape == x.shape and y.dtype == dtype
        check(y, *moe64(x, w1, s1, w2, s2, r.weights, r.experts, residual), dtype)
    assert torch.equal(ops.moe_blocks(x, w1, s1, w2, s2, r, residual=res), y)
    out = res.clone()
    assert ops.moe_blocks(x, w1, s1, w2, s2, r, residual=out, out=out) is out and torch.equal(out, y)


def test_layer_masks_and_uneven_experts(cuda):
    """All tokens on one expert, tokens without an expert, an expert twice for a token, experts without tokens."""
    g = torch.Generator(device=cuda).manual_seed(1)
    E, H, F = 9, 272, 144
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    for T in (1, 7, 20, 40, 100):
        x = torch.randn(T, H, generator=g, device=cuda).to(BF16)
        weights = torch.rand(T, 3, generator=g, device=cuda)
        one = torch.full((T, 3), -1, dtype=torch.int32)
        one[:, 0] = 4
        twice = torch.randint(0, E, (T, 3), dtype=torch.int32, generator=torch.Generator().manual_seed(T))
        twice[:, 2] = twice[:, 0]
        none = torch.full((T, 3), -1, dtype=torch.int32)
        some = twice.clone()
        some[::3] = -1
        for experts in (one, twice, none, some):
            r = routing_of(ops, experts, weights, E)
            y = ops.moe_blocks(x, w1, s1, w2, s2, r)
            check(y, *moe64(x, w1, s1, w2, s2, weights, r.experts), BF16)
        assert bool((ops.moe_blocks(x, w1, s1, w2, s2, routing_of(ops, none, weights, E)) == 0).all())


@pytest.mark.parametrize("T,E,k,H,F", [(128, 512, 16, 256, 128), (128, 102, 16, 672, 144), (128, 101, 16, 656, 144), (128, 32, 16, 2064, 272),
                                       (128, 16, 16, 144, 16), (8, 3, 1, 272, 144), (1, 12, 8, 272, 144), (2, 7, 4, 272, 144), (2, 9, 8, 272, 144),
                                       (1, 20, 16, 400, 272), (2, 20, 9, 272, 144), (8, 2, 1, 4096, 2064), (9, 2, 1, 1424, 1552),
                                       (40, 3, 2, 1552, 2000), (20, 2, 2, 4096, 528)])
def test_layer_at_its_limits(cuda, T, E, k, H, F):
    """Most tokens, choices and experts; around the rules; a few pairs with equal choices and without one."""
    g = torch.Generator(device=cuda).manual_seed(E)
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    x = torch.randn(T, H, generator=g, device=cuda).to(BF16)
    r = ops.moe_route(torch.randn(T, E, generator=g, device=cuda) + torch.randn(E, generator=g, device=cuda), k)
    check(ops.moe_blocks(x, w1, s1, w2, s2, r), *moe64(x, w1, s1, w2, s2, r.weights, r.experts), BF16)
    q = torch.Generator().manual_seed(E)
    experts = torch.randint(-1, min(E, 3), (T, k), dtype=torch.int32, generator=q)
    r = routing_of(ops, experts, torch.randn(T, k, generator=g, device=cuda), E)
    check(ops.moe_blocks(x, w1, s1, w2, s2, r), *moe64(x, w1, s1, w2, s2, r.weights, r.experts), BF16)


def test_offsets_past_32_bits(cuda):
    """Rows of logits, experts' weights and outputs more than 4 GiB apart."""
    g = torch.Generator(device=cuda).manual_seed(12)
    far = torch.empty(600, 1 << 21, device=cuda)[:, :40]
    far.copy_(torch.randn(600, 40, generator=g, device=cuda))
    same_route(ops.moe_route(far, 4), route64(far, 4), far)
    E, H, F = 3, 272, 144
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    apart = torch.empty(E, (9 << 28) // 16, 16, dtype=torch.uint8, device=cuda)

    def spaced(w, at):
        v = apart[:, at:at + w.shape[1] * w.shape[2] // 16].view(E, w.shape[1], w.shape[2]).view(w.dtype)
        v.view(torch.uint8).copy_(w.view(torch.uint8))
        return v
    v1, v2 = spaced(w1, 0), spaced(w2, 1 << 20)
    assert v1.stride(0) * 2 > 1 << 32
    for T, k in ((1, 3), (40, 2)):
        x = torch.randn(T, H, generator=g, device=cuda).to(BF16)
        r = ops.moe_route(torch.randn(T, E, generator=g, device=cuda), k)
        out = torch.empty(T, 1 << 26, dtype=BF16, device=cuda)[:, :H]
        y = ops.moe_blocks(x, w1, s1, w2, s2, r, residual=x)
        assert torch.equal(ops.moe_blocks(x, v1, s1, v2, s2, r, residual=x, out=out), y)


def test_layer_without_tokens(cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    w = layer(g, 3, 144, 80, cuda)
    x = torch.empty(0, 144, device=cuda, dtype=BF16)
    r = ops.moe_route(torch.empty(0, 3, device=cuda), 2)
    for host in (ops._host, None):
        with pytest.MonkeyPatch.context() as m:
            m.setattr(ops, "_host", host)
            assert ops.moe_blocks(x, *w, r).shape == (0, 144) and ops.moe_blocks(x, *w, r, residual=x).shape == (0, 144)


def test_layer_strides(cuda):
    g = torch.Generator(device=cuda).manual_seed(2)
    T, E, k, H, F = 6, 5, 2, 160, 144
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    x = torch.randn(T, H, generator=g, device=cuda).to(BF16)
    res = torch.randn(T, H, generator=g, device=cuda).to(BF16)
    r = ops.moe_route(torch.randn(T, E, generator=g, device=cuda), k)
    y = ops.moe_blocks(x, w1, s1, w2, s2, r, residual=res)

    def padded(w, n, k):
        p = torch.zeros(E, w.shape[1] + n, w.shape[2] + k, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
        p[:, :w.shape[1], :w.shape[2]] = w
        return p[:, :w.shape[1], :w.shape[2]]
    wide = torch.empty(T, 3 * H, dtype=BF16, device=cuda)
    wide[:, H:2 * H] = x
    out = torch.full((T + 1, 2 * H), 7.0, dtype=BF16, device=cuda)
    swapped = [s.transpose(1, 2).contiguous().transpose(1, 2) for s in (s1, s2)]
    z = ops.moe_blocks(wide[:, H:2 * H], padded(w1, 3, 32), swapped[0], padded(w2, 1, 16), swapped[1], r, residual=res, out=out[:T, 16:16 + H])
    assert torch.equal(z, y)
    assert bool((out[T] == 7.0).all()) and bool((out[:, :16] == 7.0).all()) and bool((out[:, 16 + H:] == 7.0).all())
    # one residual row for all, one set of scales for all experts
    y = ops.moe_blocks(x, w1, s1[:1].expand(s1.shape), w2, s2[:1].expand(s2.shape), r, residual=res[:1].expand(T, H))
    check(y, *moe64(x, w1, s1[:1].expand(s1.shape), w2, s2[:1].expand(s2.shape), r.weights, r.experts, res[:1].expand(T, H)), BF16)


@pytest.mark.parametrize("T", [4, 30, 90])
def test_nan_and_infinities_stay_with_their_tokens(cuda, T):
    """A broken expert, a NaN token, infinite scales: other tokens' results are those without them, bit for bit."""
    g = torch.Generator(device=cuda).manual_seed(T)
    E, H, F = 6, 272, 144
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    x = torch.randn(T, H, generator=g, device=cuda).to(BF16)
    r = ops.moe_route(torch.randn(T, E, generator=g, device=cuda), 2)
    y = ops.moe_blocks(x, w1, s1, w2, s2, r)
    hit = (r.experts == 3).any(dim=1)
    assert bool(hit.any()) and not bool(hit.all())
    nan = torch.tensor([0x7f], dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    for broken in ("w1", "w2", "s1", "s2"):
        a = dict(w1=w1.clone(), s1=s1.clone(), w2=w2.clone(), s2=s2.clone())
        if broken[0] == "w":
            a[broken].view(torch.uint8)[3] = nan.view(torch.uint8)
        else:
            a[broken][3] = INF
        z = ops.moe_blocks(x, a["w1"], a["s1"], a["w2"], a["s2"], r)
        assert torch.equal(z[~hit], y[~hit]), broken
        assert not bool(torch.isfinite(z[hit]).any()), broken
    x2 = x.clone()
    x2[1] = float("nan")
    z = ops.moe_blocks(x2, w1, s1, w2, s2, r)
    keep = torch.arange(T, device=cuda) != 1
    assert torch.equal(z[keep], y[keep]) and bool(torch.isnan(z[1]).all())


def test_gates_of_every_size(cuda):
    """silu over the whole range of gates, by one-hot weights: large and tiny values, zeros, gates whose exponential overflows."""
    H, F = 16, 32
    w1 = torch.zeros(1, 2 * F, H, device=cuda)
    w1[0, :F, 0] = 1.0                                    # gate = x_0, up = x_1
    w1[0, F:, 1] = 1.0
    w2 = torch.zeros(1, H, F, device=cuda)
    w2[0, :, 5] = 1.0                                     # y = h_5
    ones = lambda w: torch.ones(1, -(-w.shape[1] // 128), -(-w.shape[2] // 128), device=cuda)  # noqa: E731
    gates = torch.tensor([0.0, -0.0, 1.0, -1.0, 3e-38, -3e-30, 20.0, -20.0, -80.0, -87.0, -88.5, -100.0, -1e4, 1e4, 3e38, -3e38], device=cuda)
    x = torch.zeros(16, H, device=cuda, dtype=BF16)
    x[:, 0], x[:, 1] = gates.to(BF16), 1.5
    r = routing_of(ops, torch.zeros(16, 1, dtype=torch.int32), torch.ones(16, 1, device=cuda), 1)
    y = ops.moe_blocks(x, w1.to(torch.float8_e4m3fn), ones(w1), w2.to(torch.float8_e4m3fn), ones(w2), r)
    g = x[:, 0].double()
    ref = g * torch.sigmoid(g) * 1.5
    ref = torch.where(g < -88.7, 0.0, ref)                # from there on exp(-g) is infinite in fp32
    # 3e38 * 1.5 is infinite in fp32 (and times the zeros of w2 a NaN)
    over = ref.abs() > torch.finfo(F32).max
    assert int(over.sum()) == 1 and not bool(torch.isfinite(y[over]).any())
    # h in bf16 pairs loses what lies below bf16's subnormals of the second number: 2^-134
    ok = (y[:, 0].double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -16) + 2.0 ** -133
    assert bool((ok | over).all())


def test_captured_and_on_streams(cuda):
    """Router and layer in a graph, replayed with new inputs, and on four streams at once."""
    g = torch.Generator(device=cuda).manual_seed(3)
    E, H, F, k = 8, 512, 256, 2
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    T = 24
    x = torch.empty(T, H, dtype=BF16, device=cuda)
    logits = torch.empty(T, E, device=cuda)

    def fill(seed):
        q = torch.Generator(device=cuda).manual_seed(seed)
        x.copy_(torch.randn(T, H, generator=q, device=cuda))
        logits.copy_(torch.randn(T, E, generator=q, device=cuda))
        logits[seed % T] = -INF
    run = lambda: ops.moe_blocks(x, w1, s1, w2, s2, ops.moe_route(logits, k), residual=x)  # noqa: E731
    fill(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    for seed in range(1, 5):
        fill(seed)
        eager = run()
        torch.cuda.synchronize()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        r = ops.moe_route(logits, k)
        check(y, *moe64(x, w1, s1, w2, s2, r.weights, r.experts, x), BF16)
    xs = [torch.randn(n, H, generator=g, device=cuda).to(BF16) for n in (1, 9, 40, 100)]
    ls = [torch.randn(n, E, generator=g, device=cuda) for n in (1, 9, 40, 100)]
    alone = [ops.moe_blocks(a, w1, s1, w2, s2, ops.moe_route(b, k)) for a, b in zip(xs, ls)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    out = [None] * 4
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i] = ops.moe_blocks(xs[i], w1, s1, w2, s2, ops.moe_route(ls[i], k))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, out))


def test_native_and_python_calls_agree(cuda, monkeypatch):
    g = torch.Generator(device=cuda).manual_seed(4)
    E, H, F = 6, 256, 144
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    x = torch.randn(5, H, generator=g, device=cuda).to(FP16)
    logits = torch.randn(200, E, generator=g, device=cuda)
    bias = torch.randn(E, generator=g, device=cuda)
    assert ops._host is not None and ops._host.moe_route(logits, 2, "softmax", True, 1.0, None) is not None
    r = ops.moe_route(logits[:5], 2)
    assert ops._host.moe_blocks(x, w1, s1, w2, s2, r, None, None) is not None

    def calls():
        return (*ops.moe_route(logits, 2, "sigmoid", False, 0.5, bias), *ops.moe_route(logits, 3), ops.moe_blocks(x, w1, s1, w2, s2, r),
                ops.moe_blocks(x, w1, s1, w2, s2, r, residual=x, out=torch.empty_like(x)))
    native = calls()
    monkeypatch.setattr(ops, "_host", None)
    assert all(torch.equal(a, b) for a, b in zip(native, calls()))


def test_with_the_products_around_it(cuda):
    """A block as it is used: the shared linear's product onto the residual stream, router, few tokens' layer; and the same tokens by
    the products for many, whose quants of the activations are all that sets them apart."""
    g = torch.Generator(device=cuda).manual_seed(6)
    T, E, k, H, F = 40, 8, 2, 512, 384
    w1, s1, w2, s2 = layer(g, E, H, F, cuda)
    x = torch.randn(T, H, generator=g, device=cuda).to(BF16)
    ws, ss = ops.quant_blocks(torch.randn(H, H, generator=g, device=cuda) * 0.04, rows=128)
    q, sq = ops.quant_blocks(x)
    h = ops.gemm_blocks_act(q, ws, sq, ss, BF16, activation="gelu", residual=x)
    r = ops.moe_route(torch.randn(T, E, generator=g, device=cuda), k)
    y = ops.moe_blocks(h, w1, s1, w2, s2, r, residual=h)
    check(y, *moe64(h, w1, s1, w2, s2, r.weights, r.experts, h), BF16)
    q, sq = ops.quant_blocks(h)
    rows = (r.order // k).long()
    qs, sqs = q.view(torch.uint8)[rows].view(torch.float8_e4m3fn), sq[rows]
    a, sa = ops.silu_mul_quant_blocks(ops.grouped_gemm_blocks(qs, w1, sqs, s1, r.offsets))
    z = ops.grouped_gemm_blocks(a, w2, sa, s2, r.offsets)
    many = h.double() + (z[r.place.long()].double() * r.weights.double()[:, :, None]).sum(dim=1)
    # two quants to e4m3 (2^-4 relative each at most, independent from value to value) and two roundings to bf16
    assert float((many - y.double()).norm() / (y.double() - h.double()).norm()) < 2 * 2.0 ** -4
