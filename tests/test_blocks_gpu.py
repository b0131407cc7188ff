"""The block-scaled quant, SwiGLU + quant and products (dense, by expert) against float64 (GPU)."""
import pytest
import torch

from _blocks import B, E4M3, cdiv, check_product, codes, plan, product64, quant32, scales, spread

pytestmark = pytest.mark.gpu
BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def same_bits(q, r):
    """Equal codes; a NaN code is 0x7f or 0xff."""
    q, r = q.view(torch.uint8), r.view(torch.uint8)
    nan = (q & 0x7f) == 0x7f
    assert torch.equal(nan, (r & 0x7f) == 0x7f)
    assert torch.equal(q[~nan], r[~nan])


# ---- quant ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("M,K", [(1, 16), (1, 5376), (3, 128), (33, 144), (127, 512), (129, 528), (300, 2064), (1000, 7168)])
def test_quant_blocks(cuda, M, K, rows, dtype):
    from h3_tp2_amd import ops
    g = gen(M + K)
    x = (torch.randn(M, K, generator=g, device=cuda) * torch.exp(2 * torch.randn(M, 1, generator=g, device=cuda))).to(dtype)
    x[0] = 0                                                          # blocks of zeros in the 1 x 128 form
    q, s = ops.quant_blocks(x, rows=rows)
    qr, sr = quant32(x.float(), rows)
    assert q.shape == (M, K) and s.shape == (cdiv(M, rows), cdiv(K, B)) and s.dtype == F32
    assert torch.equal(s, sr)
    same_bits(q, qr)
    # the definition in float64: half a step of the code, and three fp32 roundings in front of it
    v = x.double() / spread(sr.double(), M, K, rows)
    tol = torch.clamp_min(v.abs() * 2.0 ** -4, 2.0 ** -10) * (1 + 2.0 ** -20)
    assert ((q.double() - v.clamp(-448, 448)).abs() <= tol + v.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("rows", [1, 128])
def test_quant_blocks_directed_values(cuda, rows):
    """Zeros, subnormals, huge values, inf and NaN stay in their blocks."""
    from h3_tp2_amd import ops
    x = torch.randn(260, 400, generator=gen(3), device=cuda)
    x[5, 3] = float("nan")
    x[140, 130] = float("inf")
    x[7, 300:] = 1e-40
    x[8, 256:384] = 3e38
    x[256:] = 0
    for dt in (F32, BF16):
        q, s = ops.quant_blocks(x.to(dt), rows=rows)
        qr, sr = quant32(x.to(dt).float(), rows)
        assert torch.equal(torch.isnan(s), torch.isnan(sr)) and torch.equal(s[~sr.isnan()], sr[~sr.isnan()])
        same_bits(q, qr)


def test_quant_blocks_strides_and_outputs(cuda):
    """A column slice of a wider tensor in, caller's codes and scales in other strides out, nothing else written."""
    from h3_tp2_amd import ops
    wide = torch.randn(70, 1200, generator=gen(4), device=cuda).to(BF16)
    x = wide[:, 64:64 + 656]
    qbuf = torch.full((70, 800), 0x55, dtype=torch.uint8, device=cuda)
    sbuf = torch.full((72, 8), -7.0, device=cuda)
    q, s = ops.quant_blocks(x, q=qbuf.view(E4M3)[:, :656], scale=sbuf[1:71, 1:7])
    qr, sr = quant32(x.float())
    assert torch.equal(s, sr) and torch.equal(sbuf[1:71, 1:7], sr)
    same_bits(q.contiguous(), qr)
    assert (qbuf[:, 656:] == 0x55).all() and (sbuf[:, 0] == -7).all() and (sbuf[:, 7] == -7).all() and (sbuf[0] == -7).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M,F", [(1, 16), (2, 128), (31, 144), (64, 2048), (65, 2064), (200, 5376)])
def test_silu_mul_quant_blocks(cuda, M, F, dtype):
    from h3_tp2_amd import ops
    x = torch.randn(M, 2 * F, generator=gen(M + F), device=cuda).mul_(3).clamp_(-16, 16).to(dtype)
    q, s = ops.silu_mul_quant_blocks(x)
    g, u = x.double().chunk(2, dim=1)
    h = g * torch.sigmoid(g) * u
    hp = torch.nn.functional.pad(h, (0, -F % B)).view(M, -1, B)
    s64 = torch.clamp_min(hp.abs().amax(2) / 448.0, 1.0 / (448.0 * 512.0))
    # |g| <= 16: the exponential's argument is 1.5 |g| ulp off at most, exp2 and rcp 2 ulp, three more roundings: 2^-19
    assert ((s.double() - s64).abs() <= s64 * 2.0 ** -19).all()
    v = h / spread(s.double(), M, F, 1)
    tol = torch.clamp_min(v.abs() * 2.0 ** -4, 2.0 ** -10) * (1 + 2.0 ** -15) + v.abs() * 2.0 ** -18
    assert ((q.double() - v.clamp(-448, 448)).abs() <= tol).all()


def test_silu_mul_quant_blocks_edges(cuda):
    """Gates that saturate, inf and NaN: what the fp32 formula gives, block by block."""
    from h3_tp2_amd import ops
    F = 640
    x = torch.randn(4, 2 * F, generator=gen(9), device=cuda).to(BF16)
    x[0, :128] = -200.0                                                # exp overflows: -0
    x[0, 128:256] = 200.0                                              # h = g u
    x[1, 300] = float("nan")
    x[2, F + 10] = float("inf")
    x[3, 5] = float("-inf")                                            # -inf / inf
    q, s = ops.silu_mul_quant_blocks(x)
    g, u = x.float().chunk(2, dim=1)
    h = g / (1 + torch.exp(-g)) * u
    qr, sr = quant32(h)
    assert torch.equal(torch.isnan(s), torch.isnan(sr)) and torch.equal(torch.isinf(s), torch.isinf(sr))
    ok = torch.isfinite(sr)
    assert torch.allclose(s[ok], sr[ok], rtol=2.0 ** -18, atol=0)
    assert torch.equal(q.float().isnan(), qr.float().isnan())
    assert (q[0, :128].float() == 0).all()


@pytest.mark.parametrize("dtype,gates", [(BF16, (-86.5, -87.0, -87.5, -88.0, -88.5)), (FP16, (-87.3125, -87.375, -88.0, -88.6875))])
def test_silu_mul_quant_blocks_gates_before_the_overflow(cuda, dtype, gates):
    """Gates whose exponential is past 2^126, so that 1 / (1 + exp(-g)) is subnormal, and still finite: the formula's value,
    which large up projections bring back into the codes' range, and its infinity.  One value to a block, so that every code is
    -448 and the scale shows the value.  Behind the argument, whose rounding is made good: exp2 and rcp 2^-23 each, six
    roundings of 2^-24: 2^-20.  From the overflow on it is -0, as the division by inf gives."""
    from h3_tp2_amd import ops
    ups = (1e28, 1e30, 1e34, 1e36, 3e38, -1e36) if dtype == BF16 else (1.0, 6e4, -6e4)
    cells = [(g, u) for g in gates for u in (*ups, float("inf"))]
    F = B * len(cells)
    x = torch.tensor([[c[i] for i in (0, 1) for c in cells for _ in range(B)]], dtype=F32, device=cuda).to(dtype)
    q, s = ops.silu_mul_quant_blocks(x)
    g, u = x.double().chunk(2, dim=1)
    h = (g / (1 + torch.exp(-g)) * u)[0, ::B]
    fin = torch.isfinite(h)
    assert torch.isinf(s[0, ~fin]).all() and (~fin).sum() == len(gates)
    s64 = torch.clamp_min(h[fin].abs() / 448.0, 1.0 / (448.0 * 512.0))
    assert ((s[0, fin].double() - s64).abs() <= s64 * 2.0 ** -20).all()
    big = fin & (h.abs() > 1.0 / 512.0)
    assert dtype == FP16 or big.sum() >= 2 * len(gates)
    codes8 = q.float().view(len(cells), B)
    assert torch.equal(codes8[big], (448.0 * torch.sign(h[big]).float())[:, None].expand(-1, B))
    over = torch.tensor([[-89.0] * B + [1e36] * B], device=cuda).to(BF16)
    q, s = ops.silu_mul_quant_blocks(over)
    assert (q.view(torch.uint8) == 0x80).all() and (s == 1.0 / (448.0 * 512.0)).all()


# ---- dense product --------------------------------------------------------------------------------------------------

SHAPES = [(1, 16, 16), (1, 5376, 21504), (2, 128, 128), (5, 144, 272), (16, 2064, 144), (17, 528, 720), (33, 1200, 2064),
          (64, 5376, 512), (65, 1536, 1536), (129, 4096, 400), (200, 7168, 5376), (257, 272, 528), (1000, 1536, 4608)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gemm_blocks_random(cuda, M, K, N):
    from h3_tp2_amd import ops
    g = gen(M + N)
    a, w = codes(g, M, K), codes(g, N, K)
    sa, sw = scales(g, M, cdiv(K, B)), scales(g, cdiv(N, B), cdiv(K, B))
    dt = FP16 if N == 5376 else BF16
    bias = (torch.randn(N, generator=g, device=cuda) * 0.5).to(dt) if M % 2 else None
    y = ops.gemm_blocks(a, w, sa, sw, dt, bias)
    y64, mag = product64(a, w, sa, sw, bias)
    check_product(y, y64, mag, dt)
    # the scales in the quant's order (tokens contiguous) give the same bits
    y2 = ops.gemm_blocks(a, w, sa.t().contiguous().t(), sw.t().contiguous().t(), dt, bias)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("M,K,N", SHAPES + [(600, 512, 1024), (3000, 256, 528)])
def test_gemm_blocks_exact(cuda, M, K, N):
    """Integer codes and power-of-two scales: every sum is exact, so the output is the exact value rounded once."""
    from h3_tp2_amd import ops
    g = gen(M + K)
    a, w = codes(g, M, K, integers=True), codes(g, N, K, integers=True)
    sa, sw = scales(g, M, cdiv(K, B), pow2=True), scales(g, cdiv(N, B), cdiv(K, B), pow2=True)
    y64, _ = product64(a, w, sa, sw)
    assert torch.equal(ops.gemm_blocks(a, w, sa, sw), y64.to(BF16))


@pytest.mark.parametrize("M", [1, 7, 40, 130, 700])
def test_gemm_blocks_strides(cuda, M):
    """Operands as slices of wider buffers whose other bytes are NaN codes, and an output slice: nothing past K is read into
    the sum, nothing outside the slice is written."""
    from h3_tp2_amd import ops
    K, N = 592, 400
    g = gen(M)
    abuf = torch.full((M, 704), 0x7f, dtype=torch.uint8, device=cuda).view(E4M3)
    wbuf = torch.full((N + 32, 736), 0x7f, dtype=torch.uint8, device=cuda).view(E4M3)
    a, w = abuf[:, 32:32 + K], wbuf[:N, 64:64 + K]
    a.view(torch.uint8).copy_(codes(g, M, K).view(torch.uint8))
    w.view(torch.uint8).copy_(codes(g, N, K).view(torch.uint8))
    sa = torch.full((M, 9), float("nan"), device=cuda)
    sa[:, 2:7] = scales(g, M, 5)
    sw = torch.full((5, 8), float("nan"), device=cuda)
    sw[:4, 1:6] = scales(g, 4, 5)
    out = torch.full((M + 2, N + 48), -3.0, device=cuda, dtype=BF16)
    y = ops.gemm_blocks(a, w, sa[:, 2:7], sw[:4, 1:6], out=out[1:M + 1, 16:16 + N])
    y64, mag = product64(a, w, sa[:, 2:7], sw[:4, 1:6])
    check_product(y, y64, mag, BF16)
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[1:M + 1, 16:16 + N] = False
    assert (out[keep] == -3).all()


def test_gemm_blocks_nan_stays_in_its_row(cuda):
    from h3_tp2_amd import ops
    g = gen(1)
    a, w = codes(g, 40, 512), codes(g, 256, 512)
    sa, sw = scales(g, 40, 4), scales(g, 2, 4)
    good = ops.gemm_blocks(a, w, sa, sw)
    a.view(torch.uint8)[7, 300] = 0x7f
    sa[9, 2] = float("inf")
    y = ops.gemm_blocks(a, w, sa, sw)
    assert y[7].isnan().all() and not y[9].isfinite().any()
    rest = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(y[rest], good[rest])


def test_gemm_blocks_empty(cuda):
    from h3_tp2_amd import ops
    z = lambda *s: torch.zeros(s, device=cuda)                         # noqa: E731
    y = ops.gemm_blocks(z(0, 256).to(E4M3), z(64, 256).to(E4M3), z(0, 2), z(1, 2))
    assert y.shape == (0, 64)
    y = ops.gemm_blocks(z(4, 256).to(E4M3), z(0, 256).to(E4M3), z(4, 2), z(0, 2))
    assert y.shape == (4, 0)
    with pytest.raises(Exception, match="K must be positive"):
        ops.gemm_blocks(z(4, 0).to(E4M3), z(64, 0).to(E4M3), z(4, 0), z(1, 0))


# every form that a call can run in: (M, N) with the place in the library's list that its rule gives on 256 CUs
FORMS = [(7, 400, 0), (24, 4096, 0), (30, 13008, 1), (60, 16000, 3), (300, 2576, 3), (300, 5376, 5), (500, 6160, 6),
         (300, 21520, 7), (2050, 5376, 8)]


@pytest.mark.parametrize("M,N,form", FORMS)
@pytest.mark.parametrize("K", [16, 128, 272, 640])
def test_gemm_blocks_forms(cuda, M, N, form, K):
    """Each form at ragged rows and channels and at 1, 3 and 5 k-blocks: the exact values, and the bits of row-by-row calls."""
    from h3_tp2_amd import ops
    assert plan(M, N)[2] == form
    g = gen(M + K)
    a, w = codes(g, M, K, integers=True), codes(g, N, K, integers=True)
    sa, sw = scales(g, M, cdiv(K, B), pow2=True), scales(g, cdiv(N, B), cdiv(K, B), pow2=True)
    out = torch.full((M + 2, N + 16), -3.0, device=cuda, dtype=BF16)
    y = ops.gemm_blocks(a, w, sa, sw, out=out[1:M + 1, :N])
    assert torch.equal(y, product64(a, w, sa, sw)[0].to(BF16))
    assert (out[0] == -3).all() and (out[M + 1] == -3).all() and (out[:, N:] == -3).all()
    a, w, sa, sw = codes(g, M, K), codes(g, N, K), scales(g, M, cdiv(K, B)), scales(g, cdiv(N, B), cdiv(K, B))
    y = ops.gemm_blocks(a, w, sa, sw)
    y64, mag = product64(a, w, sa, sw)
    check_product(y, y64, mag, BF16)
    for m in (0, M // 2, M - 1):
        assert torch.equal(y[m:m + 1], ops.gemm_blocks(a[m:m + 1], w, sa[m:m + 1], sw)), m


def exact_operands(g, M, N, K, E=None):
    """Integer codes, scales of 2^-2 .. 2^1: products are multiples of 2^-4 and a block's sum at most 2^13, so that every fp32 sum over
    K <= 640 is exact, with an integer bias too."""
    a, w = codes(g, M, K, integers=True), codes(g, (E or 1) * N, K, integers=True)
    pow2 = lambda *s: torch.exp2(torch.randint(-2, 2, s, generator=g, device="cuda").float())            # noqa: E731
    sa, sw = pow2(M, cdiv(K, B)), pow2(E or 1, cdiv(N, B), cdiv(K, B))
    return (a, w, sa, sw[0]) if E is None else (a, w.view(E, N, K), sa, sw)


@pytest.mark.parametrize("M,N,form", FORMS)
@pytest.mark.parametrize("dtype,biased", [(BF16, True), (FP16, False), (FP16, True)])
def test_gemm_blocks_epilogues(cuda, M, N, form, dtype, biased):
    """Each form's epilogue with a bias and in fp16, at ragged rows and channels: the exact value, rounded once; nothing outside the
    output is written."""
    from h3_tp2_amd import ops
    assert plan(M, N)[2] == form
    K = 272
    g = gen(M + N)
    a, w, sa, sw = exact_operands(g, M, N, K)
    bias = torch.randint(-300, 301, (N,), generator=g, device=cuda).float().to(dtype) if biased else None
    out = torch.full((M + 2, N + 16), -3.0, device=cuda, dtype=dtype)
    y = ops.gemm_blocks(a, w, sa, sw, dtype, bias, out=out[1:M + 1, :N])
    y64, _ = product64(a, w, sa, sw, bias)
    assert torch.equal(y, y64.to(dtype))
    assert (out[0] == -3).all() and (out[M + 1] == -3).all() and (out[:, N:] == -3).all()


@pytest.mark.parametrize("M", [200, 199])
def test_gemm_blocks_out_projection(cuda, M):
    """The out projection of a short sequence in fp16 with a bias, random operands."""
    from h3_tp2_amd import ops
    g = gen(M)
    K, N = 7168, 5376
    a, w, sa, sw = codes(g, M, K), codes(g, N, K), scales(g, M, K // B), scales(g, N // B, K // B)
    sa, bias = sa * 0.1, (torch.randn(N, generator=g, device=cuda) * 0.5).to(FP16)
    y = ops.gemm_blocks(a, w, sa, sw, FP16, bias)
    y64, mag = product64(a, w, sa, sw, bias)
    assert y64.abs().max() < 65504
    check_product(y, y64, mag, FP16)


def test_gemm_blocks_streaming_weight(cuda):
    """More than 64 MiB of weights: the loads with the non-temporal hint, against the same rows of a slice without it."""
    from h3_tp2_amd import ops
    g = gen(8)
    M, K, N = 9, 6160, 12288
    a, w, sa, sw = codes(g, M, K), codes(g, N, K), scales(g, M, 49), scales(g, 96, 49)
    y = ops.gemm_blocks(a, w, sa, sw)
    assert torch.equal(y[:, :2048], ops.gemm_blocks(a, w[:2048], sa, sw[:16]))
    assert torch.equal(y[:, -256:], ops.gemm_blocks(a, w[-256:], sa, sw[-2:]))
    y64, mag = product64(a, w, sa, sw)
    check_product(y, y64, mag, BF16)


@pytest.mark.parametrize("dtype,biased", [(BF16, True), (FP16, False), (FP16, True)])
def test_gemm_blocks_streaming_weight_epilogues(cuda, dtype, biased):
    """The streaming loads with a bias and in fp16: the exact value, rounded once."""
    from h3_tp2_amd import ops
    g = gen(18)
    M, K, N = 11, 272, 249856
    assert plan(M, N)[2] == 0 and N * K > 64 << 20
    a, w, sa, sw = exact_operands(g, M, N, K)
    bias = torch.randint(-300, 301, (N,), generator=g, device=cuda).float().to(dtype) if biased else None
    y = ops.gemm_blocks(a, w, sa, sw, dtype, bias)
    for n in range(0, N, 32768):
        part = slice(n, min(N, n + 32768))
        ref, _ = product64(a, w[part], sa, sw[n // B:cdiv(part.stop, B)], None if bias is None else bias[part])
        assert torch.equal(y[:, part], ref.to(dtype)), n


def test_gemm_blocks_extreme_scales(cuda):
    """Scales of 0, inf and NaN in the last of an odd number of blocks, and products that round to a negative zero: every form
    gives the bits of the single row."""
    from h3_tp2_amd import ops
    g = gen(9)
    K, N = 384, 2576
    w, sw = codes(g, N, K), scales(g, 21, 3)
    sw[3, 2], sw[5, 2], sw[7, 2], sw[9] = 0.0, float("inf"), float("nan"), 1e-44
    a, sa = codes(g, 300, K), scales(g, 300, 3)
    sa[11] = 1e-30
    y = ops.gemm_blocks(a, w, sa, sw)
    for m in (0, 11, 299):
        one = ops.gemm_blocks(a[m:m + 1], w, sa[m:m + 1], sw)
        assert torch.equal(y[m:m + 1].view(torch.int16)[~one.isnan()], one.view(torch.int16)[~one.isnan()])
        assert torch.equal(y[m:m + 1].isnan(), one.isnan())
    assert y[0, 7 * 128].isnan() and not y[0, 5 * 128].isfinite()


# ---- by expert ------------------------------------------------------------------------------------------------------

def grouped64(a, w, sa, sw, off):
    M, N = a.shape[0], w.shape[1]
    y, mag = torch.zeros(M, N, dtype=torch.float64, device="cuda"), torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        if hi > lo:
            y[lo:hi], mag[lo:hi] = product64(a[lo:hi], w[e], sa[lo:hi], sw[e])
    return y, mag


GROUPS = [
    ("one expert", [0, 37], 37),
    ("single rows", [0, 1, 2, 3], 3),
    ("empty first, middle, last", [0, 0, 5, 5, 40, 40], 40),
    ("nothing", [0, 0, 0, 0], 30),
    ("rows before and behind", [4, 20, 20, 33], 50),
    ("tile edges", [0, 16, 32, 96, 160, 288], 288),
    ("ragged", [0, 3, 130, 131, 500, 777, 1000], 1100),
    ("many experts", [min(97, i // 2) for i in range(201)], 97),
    ("large", [0, 900, 1000, 2600], 2600),
]


@pytest.mark.parametrize("name,off,M", GROUPS, ids=[c[0] for c in GROUPS])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("K,N", [(272, 400), (1536, 512)])
def test_grouped(cuda, name, off, M, idx, K, N):
    """Rows outside every expert hold NaN codes and scales, and stay as they were in the output."""
    from h3_tp2_amd import ops
    g = gen(M + K)
    E = len(off) - 1
    a, sa = codes(g, M, K), scales(g, M, cdiv(K, B))
    w, sw = codes(g, E * N, K).view(E, N, K), scales(g, E, cdiv(N, B), cdiv(K, B))
    mine = torch.zeros(M, dtype=torch.bool, device=cuda)
    mine[off[0]:off[-1]] = True
    a.view(torch.uint8)[~mine] = 0x7f
    sa[~mine] = float("nan")
    dt = FP16 if name == "ragged" else BF16
    out = torch.full((M, N), -3.0, device=cuda, dtype=dt)
    y = ops.grouped_gemm_blocks(a, w, sa, sw, torch.tensor(off, device=cuda, dtype=idx), dt, out=out)
    assert y.data_ptr() == out.data_ptr()
    y64, mag = grouped64(a, w, sa, sw, off)
    check_product(y[mine], y64[mine], mag[mine], dt)
    assert (y[~mine] == -3).all()
    # every expert's rows are the dense product's, bit for bit
    for e, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        if hi > lo and e < 12:
            assert torch.equal(y[lo:hi], ops.gemm_blocks(a[lo:hi], w[e], sa[lo:hi], sw[e], dt)), e


# (rows, experts, channels, form): each form of the rule by rows per expert; more experts than the LDS table of the large tiles
GROUPED_FORMS = [(9, 4, 400, 0), (40, 7, 272, 2), (100, 5, 400, 4), (700, 5, 400, 7), (60000, 3, 2064, 8), (9000, 300, 144, 7)]


@pytest.mark.parametrize("M,E,N,form", GROUPED_FORMS)
@pytest.mark.parametrize("K", [144, 512])
def test_grouped_forms(cuda, M, E, N, form, K):
    from h3_tp2_amd import ops
    assert plan(M, N, E, True)[2] == form
    g = gen(M + K)
    a, w = codes(g, M, K, integers=True), codes(g, E * N, K, integers=True).view(E, N, K)
    sa, sw = scales(g, M, cdiv(K, B), pow2=True), scales(g, E, cdiv(N, B), cdiv(K, B), pow2=True)
    cuts = torch.randint(0, M + 1, (E + 1,), generator=g, device=cuda).sort()[0]
    cuts[E // 2] = cuts[E // 2 + 1]                                    # one without rows
    out = torch.full((M, N), -3.0, device=cuda, dtype=BF16)
    ops.grouped_gemm_blocks(a, w, sa, sw, cuts.to(torch.int32), out=out)
    off = cuts.tolist()
    for e in range(E):
        lo, hi = off[e], off[e + 1]
        if hi > lo:
            assert torch.equal(out[lo:hi], product64(a[lo:hi], w[e], sa[lo:hi], sw[e])[0].to(BF16)), e
    assert (out[:off[0]] == -3).all() and (out[off[-1]:] == -3).all()


@pytest.mark.parametrize("M,E,N,form", GROUPED_FORMS)
def test_grouped_forms_fp16(cuda, M, E, N, form):
    """Each form's fp16 output: the exact value, rounded once."""
    from h3_tp2_amd import ops
    assert plan(M, N, E, True)[2] == form
    g = gen(M + E)
    a, w, sa, sw = exact_operands(g, M, N, 272, E)
    off = [0] + torch.randint(0, M + 1, (E - 1,), generator=g, device=cuda).sort()[0].tolist() + [M]
    y = ops.grouped_gemm_blocks(a, w, sa, sw, torch.tensor(off, device=cuda), FP16)
    for e, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        if hi > lo:
            assert torch.equal(y[lo:hi], product64(a[lo:hi], w[e], sa[lo:hi], sw[e])[0].to(FP16)), e


@pytest.mark.parametrize("M,form", [(1000, 7), (4000, 8)])
def test_grouped_streaming_weights(cuda, M, form):
    """More than 64 MiB of weights, a row tile per mean expert: the large tiles' loads with the hint give the dense bits, with an
    expert of several row tiles, one of one row and one without rows among them."""
    from h3_tp2_amd import ops
    E, N, K = 18, 2064, 2048
    assert plan(M, N, E, True)[2] == form and E * N * K > 64 << 20
    g = gen(M)
    a, w = codes(g, M, K), codes(g, E * N, K).view(E, N, K)
    sa, sw = scales(g, M, K // B), scales(g, E, cdiv(N, B), K // B)
    off = [0, M // 3, M // 3 + 1, M // 3 + 1] + [M // 3 + 1 + (M - M // 3 - 1) * i // (E - 3) for i in range(1, E - 2)]
    assert len(off) == E + 1 and off[-1] == M
    y = ops.grouped_gemm_blocks(a, w, sa, sw, torch.tensor(off, dtype=torch.int32, device=cuda))
    for e, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        if hi > lo:
            assert torch.equal(y[lo:hi], ops.gemm_blocks(a[lo:hi], w[e], sa[lo:hi], sw[e])), e


@pytest.mark.parametrize("M,form", [(60, 0), (180, 2), (300, 4), (1000, 7), (4000, 8)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_grouped_streaming_weights_forms(cuda, M, form, dtype):
    """More than 64 MiB of weights in every form that takes the hint, in both output types: the dense bits, with an expert of a
    third of the rows, one of one row and one without rows."""
    from h3_tp2_amd import ops
    E, N, K = 18, 2064, 2048
    assert plan(M, N, E, True)[2] == form and E * N * K > 64 << 20
    g = gen(M + 1)
    a, w = codes(g, M, K), codes(g, E * N, K).view(E, N, K)
    sa, sw = scales(g, M, K // B), scales(g, E, cdiv(N, B), K // B)
    off = [0, M // 3, M // 3 + 1, M // 3 + 1] + [M // 3 + 1 + (M - M // 3 - 1) * i // (E - 3) for i in range(1, E - 2)]
    assert len(off) == E + 1 and off[-1] == M
    y = ops.grouped_gemm_blocks(a, w, sa, sw, torch.tensor(off, device=cuda), dtype)
    for e, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        if hi > lo:
            assert torch.equal(y[lo:hi], ops.gemm_blocks(a[lo:hi], w[e], sa[lo:hi], sw[e], dtype)), e
    y64, mag = grouped64(a, w, sa, sw, off)
    check_product(y, y64, mag, dtype)


def test_grouped_decreasing_offsets_stay_inside(cuda):
    """Offsets that decrease are a caller's mistake: an expert whose end is before its start has no rows, and nothing outside
    the union of the others is written."""
    from h3_tp2_amd import ops
    g = gen(3)
    a, sa, w, sw = codes(g, 40, 256), scales(g, 40, 2), codes(g, 3 * 64, 256).view(3, 64, 256), scales(g, 3, 1, 2)
    out = torch.full((40, 64), -3.0, device=cuda, dtype=BF16)
    ops.grouped_gemm_blocks(a, w, sa, sw, torch.tensor([5, 20, 12, 15], device=cuda), out=out)
    assert torch.equal(out[5:12], ops.gemm_blocks(a[5:12], w[0], sa[5:12], sw[0]))
    assert (out[:5] == -3).all() and (out[20:] == -3).all()


def test_grouped_offsets_outside_are_ends(cuda):
    from h3_tp2_amd import ops
    g = gen(2)
    a, sa, w, sw = codes(g, 20, 256), scales(g, 20, 2), codes(g, 128, 256).view(2, 64, 256), scales(g, 2, 1, 2)
    off = torch.tensor([-5, 8, 4000], device=cuda, dtype=torch.int64)
    y = ops.grouped_gemm_blocks(a, w, sa, sw, off)
    assert torch.equal(y, ops.grouped_gemm_blocks(a, w, sa, sw, off.clamp(0, 20)))


def test_grouped_expert_strides(cuda):
    """The experts' weights and scales as slices of a larger stack."""
    from h3_tp2_amd import ops
    g = gen(5)
    E, N, K = 3, 144, 272
    wb = codes(g, E * 2 * (N + 16), K + 16).view(E, 2, N + 16, K + 16)
    sb = scales(g, E, 2, 3, 4)
    w, sw = wb[:, 1, :N, :K], sb[:, 1, :2, :3]
    a, sa = codes(g, 50, K), scales(g, 50, 3)
    off = torch.tensor([0, 20, 21, 50], device=cuda)
    y = ops.grouped_gemm_blocks(a, w, sa, sw, off)
    y64, mag = grouped64(a, w, sa, sw, off.tolist())
    check_product(y, y64, mag, BF16)


# ---- together, as they are used -------------------------------------------------------------------------------------

def _experts(cuda, x, off, w1, s1, w2, s2, out=None):
    from h3_tp2_amd import ops
    q, s = ops.quant_blocks(x)
    gu = ops.grouped_gemm_blocks(q, w1, s, s1, off)
    hq, hs = ops.silu_mul_quant_blocks(gu)
    return ops.grouped_gemm_blocks(hq, w2, hs, s2, off, out=out)


def _expert_mlp(cuda, seed, M=300, E=5, K=512, F=272):
    from h3_tp2_amd import ops
    g = gen(seed)
    x = torch.randn(M, K, generator=g, device=cuda).to(BF16)
    w1 = [ops.quant_blocks(torch.randn(2 * F, K, generator=g, device=cuda) * 0.05, rows=128) for _ in range(E)]
    w2 = [ops.quant_blocks(torch.randn(K, F, generator=g, device=cuda) * 0.05, rows=128) for _ in range(E)]
    st = lambda ws, i: torch.stack([w[i] for w in ws])                 # noqa: E731
    stack8 = lambda ws: torch.stack([w[0].view(torch.uint8) for w in ws]).view(E4M3)   # noqa: E731
    return x, stack8(w1), st(w1, 1), stack8(w2), st(w2, 1)


def test_expert_mlp(cuda):
    """Quant, gate | up by expert, SwiGLU + quant, down by expert, against float64 without the two activation quants.  A code
    is at most 2^-4 of its value off, so each quant moves a sum by at most 2^-4 of its rms over random signs: 2^-3 for both
    (bf16 roundings and the SwiGLU's slope of about 1 within it)."""
    x, w1, s1, w2, s2 = _expert_mlp(cuda, 0)
    off = [0, 100, 100, 117, 260, 290]
    y = _experts(cuda, x, torch.tensor(off, device=cuda), w1, s1, w2, s2)
    for e, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        if hi == lo:
            continue
        W1 = w1[e].double() * spread(s1[e].double(), *w1[e].shape, B)
        W2 = w2[e].double() * spread(s2[e].double(), *w2[e].shape, B)
        gu = x[lo:hi].double() @ W1.t()
        gg, u = gu.chunk(2, dim=1)
        r = (gg * torch.sigmoid(gg) * u) @ W2.t()
        err = (y[lo:hi].double() - r).norm() / r.norm()
        assert err < 2 * 2.0 ** -4, float(err)


def test_expert_mlp_captured(cuda):
    """The run in a graph: the offsets and the tokens change between replays, eager work runs in between, rows behind the
    last expert stay as they were."""
    x, w1, s1, w2, s2 = _expert_mlp(cuda, 1)
    off = torch.tensor([0, 50, 60, 60, 200, 300], device=cuda, dtype=torch.int32)
    out = torch.zeros_like(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _experts(cuda, x, off, w1, s1, w2, s2, out)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _experts(cuda, x, off, w1, s1, w2, s2, out)
    for i, o in enumerate(([0, 50, 60, 60, 200, 300], [0, 0, 0, 0, 0, 1], [3, 90, 91, 92, 93, 250], [0, 300, 300, 300, 300, 300])):
        x.copy_(torch.randn(x.shape, generator=gen(20 + i), device=cuda))
        off.copy_(torch.tensor(o))
        out.fill_(-3)
        graph.replay()
        torch.cuda.synchronize()
        ref = torch.full_like(out, -3)
        _experts(cuda, x, off, w1, s1, w2, s2, ref)
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i
        assert (out[o[-1]:] == -3).all() and (out[:o[0]] == -3).all()


def test_side_streams(cuda):
    """Two streams at once on their own buffers give what one stream gives."""
    from h3_tp2_amd import ops
    g = gen(6)
    a, w, sa, sw = codes(g, 700, 1536), codes(g, 1536, 1536), scales(g, 700, 12), scales(g, 12, 12)
    ref = ops.gemm_blocks(a, w, sa, sw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.gemm_blocks(a, w, sa, sw))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ref) for y in got)


def test_side_streams_with_their_own_operands(cuda):
    """Four streams at once, each with operands and sizes of its own (other forms), written on that stream right before the calls
    and anew in every turn: each gives what the same calls give alone.  A call on another stream, or one that keeps anything
    of another call's, would show."""
    from h3_tp2_amd import ops
    K = 1536
    tab = torch.randn(256, 96, generator=gen(40), device=cuda)
    runs = []
    for i, (M, N, E) in enumerate(((9, 400, 2), (90, 1552, 5), (700, 2064, 6), (2050, 1280, 3))):
        g = gen(41 + i)
        fresh = [torch.randn(M, K, generator=g, device=cuda).to(BF16) for _ in range(3)]
        w, sw = ops.quant_blocks(torch.randn(E * N, K, generator=g, device=cuda) * 0.05, rows=128) if N % B == 0 else (
            codes(g, E * N, K), scales(g, E * cdiv(N, B), K // B))
        off = torch.randint(0, M + 1, (E + 1,), generator=g, device=cuda).sort()[0]
        off[0], off[-1] = 0, M
        norm = 1 + 0.1 * torch.randn(128, generator=g, device=cuda)
        pos = torch.randint(0, 256, (M,), generator=g, device=cuda)
        runs.append(dict(x=torch.zeros(M, K, dtype=BF16, device=cuda), fresh=fresh, w=w.view(E, N, K), sw=sw.view(E, -1, K // B), off=off,
                         norm=norm.to(BF16), pos=pos))

    def step(r, turn):
        r["x"].copy_(r["fresh"][turn])
        q, s = ops.quant_blocks(r["x"])
        y = ops.gemm_blocks(q, r["w"][0], s, r["sw"][0])
        z = ops.grouped_gemm_blocks(q, r["w"], s, r["sw"], r["off"])
        h, hs = ops.silu_mul_quant_blocks(r["x"])
        heads = r["x"].view(-1, 12, 128)
        qk = ops.qk_norm_rope(heads[:, :8], heads[:, 8:], r["norm"], r["norm"], tab, 1e-6, positions=r["pos"])
        return [t.contiguous().view(torch.uint8) for t in (q, s, y, z, h, hs, *qk)]

    alone = []
    for turn in range(3):
        for r in runs:
            alone.append(step(r, turn))
            torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device=cuda)
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = []
    for turn in range(3):
        for r, st in zip(runs, streams):
            with torch.cuda.stream(st):
                busy @ busy                                            # the stream is behind the host when its operands are written
                got.append(step(r, turn))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(got, alone)):
        assert all(torch.equal(x, y) for x, y in zip(a, b)), i


# ---- the native host path against the Python path ---------------------------------------------------------------------

def _outcome(f):
    try:
        out = f()
    except Exception as e:  # noqa: BLE001
        return type(e), str(e)
    return [(t.dtype, tuple(t.shape), t.stride(), t.contiguous().view(torch.uint8).cpu()) for t in (out if isinstance(out, tuple) else (out,))]


def test_native_and_python_host_paths_agree(cuda, monkeypatch):
    """The same outputs, strides among them, or the same refusal."""
    from h3_tp2_amd import ops
    g = gen(12)
    x = torch.randn(9, 544, generator=g, device=cuda).to(BF16)
    a, w, sa, sw = codes(g, 9, 272), codes(g, 400, 272), scales(g, 9, 3), scales(g, 4, 3)
    w3, sw3, off = codes(g, 800, 272).view(2, 400, 272), scales(g, 2, 4, 3), torch.tensor([0, 4, 9], device=cuda)
    bias = torch.randn(400, generator=g, device=cuda).to(FP16)
    q, k, wt = x[:, :256].view(9, 2, 128), x[:, 256:384].view(9, 1, 128), torch.ones(128, device=cuda, dtype=BF16)
    tab, pos = torch.randn(40, 96, generator=g, device=cuda), torch.arange(9, device=cuda) * 3
    calls = [lambda: ops.quant_blocks(x), lambda: ops.quant_blocks(x, rows=128), lambda: ops.quant_blocks(x[:1]),
             lambda: ops.quant_blocks(x.float()), lambda: ops.quant_blocks(x[:, 1:17]), lambda: ops.quant_blocks(x, rows=3),
             lambda: ops.quant_blocks(x[:0]), lambda: ops.silu_mul_quant_blocks(x), lambda: ops.silu_mul_quant_blocks(x[:, :40]),
             lambda: ops.silu_mul_quant_blocks(x.half()), lambda: ops.gemm_blocks(a, w, sa, sw),
             lambda: ops.gemm_blocks(a, w, sa, sw, FP16, bias), lambda: ops.gemm_blocks(a, w, sa, sw, BF16, bias),
             lambda: ops.gemm_blocks(a[:1], w, sa[:1], sw), lambda: ops.gemm_blocks(a, w, sa[:, :2], sw),
             lambda: ops.gemm_blocks(a, w, sa, sw, out=torch.empty(9, 416, device=cuda, dtype=BF16)[:, :400]),
             lambda: ops.gemm_blocks(a, w, sa, sw, out=torch.empty(9, 401, device=cuda, dtype=BF16)[:, :400]),
             lambda: ops.grouped_gemm_blocks(a, w3, sa, sw3, off), lambda: ops.grouped_gemm_blocks(a, w3, sa, sw3, off.int(), FP16),
             lambda: ops.grouped_gemm_blocks(a, w3[:1], sa, sw3[:1], off[:2]), lambda: ops.grouped_gemm_blocks(a, w3, sa, sw3, off[:2]),
             lambda: ops.qk_norm_rope(q, k, wt, wt, tab, 1e-6), lambda: ops.qk_norm_rope(q, k, wt, wt, tab, 1e-6, positions=pos),
             lambda: ops.qk_norm_rope(q[:1], k[:1], wt, wt, tab, 1e-6, positions=pos[:1].int(), interleaved=True),
             lambda: ops.qk_norm_rope(q, k, wt, wt, tab[:4], 1e-6), lambda: ops.qk_norm_rope(q, k, wt, wt, tab[:, :90], 1e-6)]
    for i, f in enumerate(calls):
        got = _outcome(f)
        with monkeypatch.context() as m:
            m.setattr(ops, "_host", None)
            ref = _outcome(f)
        assert type(got) is type(ref), (i, got, ref)
        if isinstance(got, tuple):
            assert got == ref, i
        else:
            assert all(x[:3] == y[:3] and torch.equal(x[3], y[3]) for x, y in zip(got, ref)) and len(got) == len(ref), i
