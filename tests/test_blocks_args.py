"""What the block-scaled operators and qk_norm_rope refuse (CPU): before any launch, in Python and again at the C entry."""
import ctypes

import pytest
import torch

from h3_tp2_amd import _lib, ops

E4M3, BF16, FP16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_call_on", lambda t, name, *args: seen.append((name, args)))
    return seen


def refused(f, *bad):
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            f(**kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU only"):
        ops.quant_blocks(torch.zeros(4, 64, dtype=BF16))


def test_quant_blocks(calls):
    x = torch.zeros(8, 272, dtype=BF16)
    q, s = ops.quant_blocks(x)
    assert q.shape == (8, 272) and s.shape == (8, 3) and s.stride() == (1, 8)
    q, s = ops.quant_blocks(x, rows=128)
    assert s.shape == (1, 3)
    q, s = ops.silu_mul_quant_blocks(x[:, :256])
    assert q.shape == (8, 128) and s.shape == (8, 1)
    n = len(calls)
    refused(lambda **kw: ops.quant_blocks(**{"x": x, **kw}), dict(x=x.int()), dict(x=x[0]), dict(x=x[:, :24]), dict(x=x.t()),
            dict(rows=2), dict(rows=0), dict(q=torch.empty(8, 256, dtype=E4M3)), dict(q=torch.empty(8, 272, dtype=torch.uint8)),
            dict(scale=torch.empty(8, 2)), dict(scale=torch.empty(8, 3, dtype=FP16)), dict(scale=torch.empty(1, 3).expand(8, 3)),
            dict(scale=torch.empty(8, 1).expand(8, 3)))
    refused(lambda **kw: ops.silu_mul_quant_blocks(**{"x": x, **kw}), dict(), dict(x=x[:, :256].float()), dict(x=x[:, :48]))
    assert len(calls) == n


def _operands(M=8, N=272, K=400):
    return dict(a=torch.zeros(M, K, dtype=E4M3), w=torch.zeros(N, K, dtype=E4M3), scale_a=torch.ones(M, 4),
                scale_b=torch.ones(3, 4))


def test_gemm_blocks(calls):
    ok = _operands()
    assert ops.gemm_blocks(**ok).shape == (8, 272)
    ops.gemm_blocks(**ok, out_dtype=FP16, bias=torch.zeros(272, dtype=FP16), out=torch.empty(8, 272, dtype=FP16))
    ops.gemm_blocks(**{**ok, "scale_a": torch.ones(1, 4).expand(8, 4)})
    n = len(calls)
    refused(lambda **kw: ops.gemm_blocks(**{**ok, **kw}), dict(a=torch.zeros(8, 400, dtype=BF16)), dict(a=torch.zeros(8, 384, dtype=E4M3)),
            dict(w=torch.zeros(3, 272, 400, dtype=E4M3)), dict(a=torch.zeros(400, 8, dtype=E4M3).t()),
            dict(scale_a=torch.ones(8, 1)), dict(scale_a=torch.ones(8, 3)), dict(scale_a=torch.ones(4, 8).t()[:4]),
            dict(scale_a=torch.ones(8, 4, dtype=FP16)), dict(scale_b=torch.ones(272, 4)), dict(scale_b=torch.ones(2, 4)),
            dict(out_dtype=F32), dict(bias=torch.zeros(272)), dict(bias=torch.zeros(270, dtype=BF16)),
            dict(out=torch.empty(8, 270, dtype=BF16)), dict(out=torch.empty(8, 272, dtype=FP16)),
            dict(out=torch.empty(272, 8, dtype=BF16).t()))
    assert len(calls) == n


def test_grouped_gemm_blocks(calls):
    o = _operands()
    ok = {**o, "w": torch.zeros(3, 272, 400, dtype=E4M3), "scale_b": torch.ones(3, 3, 4), "offsets": torch.zeros(4, dtype=torch.int32)}
    assert ops.grouped_gemm_blocks(**ok).shape == (8, 272)
    n = len(calls)
    refused(lambda **kw: ops.grouped_gemm_blocks(**{**ok, **kw}), dict(w=o["w"]), dict(scale_b=o["scale_b"]),
            dict(offsets=torch.zeros(3, dtype=torch.int32)), dict(offsets=torch.zeros(4)), dict(offsets=torch.zeros(8, dtype=torch.int64)[::2]),
            dict(offsets=[0, 1, 2, 3]), dict(w=torch.zeros(3, 400, 272, dtype=E4M3).transpose(1, 2)), dict(out_dtype=F32),
            dict(out=torch.empty(7, 272, dtype=BF16)))
    assert len(calls) == n


def test_qk_norm_rope(calls):
    q, k, w, tab = torch.zeros(5, 4, 128, dtype=BF16), torch.zeros(5, 2, 128, dtype=BF16), torch.ones(128, dtype=BF16), torch.zeros(9, 96)
    ok = dict(q=q, k=k, q_weight=w, k_weight=w, rope_table=tab, eps=1e-6)
    oq, okk = ops.qk_norm_rope(**ok)
    assert oq.shape == q.shape and okk.shape == k.shape
    ops.qk_norm_rope(**ok, positions=torch.zeros(5, dtype=torch.int32), interleaved=True, out=(q, k))
    n = len(calls)
    refused(lambda **kw: ops.qk_norm_rope(**{**ok, **kw}), dict(q=q.float()), dict(q=q[0]), dict(k=k[:4]), dict(k=k.half()),
            dict(q=q[..., :96], k=k[..., :96]), dict(q=q.transpose(1, 2)), dict(q_weight=w.float()), dict(k_weight=w[:64]),
            dict(rope_table=tab[:4]), dict(rope_table=tab.half()), dict(rope_table=torch.zeros(9, 160)), dict(rope_table=tab[:, :88]),
            dict(rope_table=torch.zeros(9, 95), interleaved=True), dict(positions=torch.zeros(4, dtype=torch.int64)),
            dict(positions=torch.zeros(5)), dict(out=(q, q)), dict(out=(q.half(), k)))
    assert len(calls) == n


def test_c_entries_refuse_without_a_gpu():
    """The same at the C ABI: status -22 and a message, nothing launched."""
    L = _lib.load()
    p, z = ctypes.c_void_p(4096), None

    def bad(name, args, text):
        assert getattr(L, name)(*args) == -22
        assert text in L.h3fp8_last_error().decode(), L.h3fp8_last_error()

    bad("h3fp8_quant_blocks", [p, 24, 0, 4, 24, 1, p, 24, p, 1, 4, z], "multiple of 16")
    bad("h3fp8_quant_blocks", [p, 32, 0, 4, 32, 3, p, 32, p, 1, 4, z], "1 or 128 rows")
    bad("h3fp8_quant_blocks", [p, 32, 7, 4, 32, 1, p, 32, p, 1, 4, z], "bad dtype")
    bad("h3fp8_quant_blocks", [ctypes.c_void_p(4098), 32, 0, 4, 32, 1, p, 32, p, 1, 4, z], "aligned")
    bad("h3fp8_quant_blocks", [p, 16, 0, 4, 32, 1, p, 32, p, 1, 4, z], "row stride of x")
    bad("h3fp8_silu_mul_quant_blocks", [p, 32, 0, 4, 32, p, 32, p, 1, 4, z], "row stride of x")
    bad("h3fp8_silu_mul_quant_blocks", [p, 64, 2, 4, 32, p, 32, p, 1, 4, z], "bad dtype")
    gemm = [p, 64, p, 64, p, 1, 8, p, 1, 1, z, p, 32, 0, 8, 32, 64, z]

    def gemm_with(**kw):
        names = ("a", "lda", "w", "ldw", "sa", "sa_m", "sa_k", "sw", "sw_n", "sw_k", "bias", "y", "ldy", "dt", "M", "N", "K", "st")
        return [kw.get(n, v) for n, v in zip(names, gemm)]

    bad("h3fp8_gemm_blocks", gemm_with(K=40), "multiples of 16")
    bad("h3fp8_gemm_blocks", gemm_with(K=0), "K must be positive")
    bad("h3fp8_gemm_blocks", gemm_with(dt=2), "bad out_dtype")
    bad("h3fp8_gemm_blocks", gemm_with(M=-1), "negative size")
    bad("h3fp8_gemm_blocks", gemm_with(a=z), "null pointer")
    bad("h3fp8_gemm_blocks", gemm_with(lda=56), "multiples of 16")
    bad("h3fp8_gemm_blocks", gemm_with(ldy=36), "row stride of y")
    bad("h3fp8_gemm_blocks", gemm_with(y=ctypes.c_void_p(4104)), "16-byte aligned")
    bad("h3fp8_gemm_blocks", gemm_with(sa_k=-1), "negative stride")
    bad("h3fp8_gemm_blocks", gemm_with(lda=1 << 24), "stride is too large")
    grouped = [p, 64, p, 2048, 64, p, 1, 8, p, 2, 1, 1, p, 4, p, 32, 0, 8, 32, 64, 3, z]
    bad("h3fp8_grouped_gemm_blocks", grouped[:12] + [p, 2] + grouped[14:], "int32 or int64")
    bad("h3fp8_grouped_gemm_blocks", grouped[:12] + [z, 4] + grouped[14:], "null offsets")
    bad("h3fp8_grouped_gemm_blocks", grouped[:12] + [ctypes.c_void_p(4098), 4] + grouped[14:], "misaligned offsets")
    bad("h3fp8_grouped_gemm_blocks", grouped[:12] + [ctypes.c_void_p(4100), 8] + grouped[14:], "misaligned offsets")
    f = ctypes.c_float(1e-6)
    qk = [p, 512, 128, p, 256, 128, 0, 5, 4, 2, 128, p, p, p, 96, 2, 9, 96, 0, z, 0, 8, f, p, 512, 128, p, 256, 128, z]
    bad("h3fp8_qk_norm_rope", qk[:10] + [96] + qk[11:], "head size")
    bad("h3fp8_qk_norm_rope", qk[:17] + [88] + qk[18:], "rotated dims")
    bad("h3fp8_qk_norm_rope", qk[:6] + [2] + qk[7:], "bad dtype")
    bad("h3fp8_qk_norm_rope", qk[:16] + [4] + qk[17:], "a row per token")
    bad("h3fp8_qk_norm_rope", qk[:1] + [516] + qk[2:], "multiples of 8")
    bad("h3fp8_qk_norm_rope", qk[:19] + [p, 1, 2] + qk[22:], "int32 or int64")


def test_more_threads_than_a_launch_holds_are_refused():
    """2^20 experts of one row by 1024 channels: 2^25 tiles of 128 threads are 2^32, past what one launch takes.  The library says
    so itself, as the quants and the rotation do, and does not leave it to the runtime."""
    L = _lib.load()
    p, z = ctypes.c_void_p(4096), None
    M = E = 1 << 20
    for n in (1024, 2048):
        rc = L.h3fp8_grouped_gemm_blocks(p, 16, p, 0, 16, p, 1, M, p, 0, 0, 0, p, 4, p, n, 0, M, n, 16, E, z)
        assert rc == -22 and "too many tiles for one launch" in L.h3fp8_last_error().decode(), L.h3fp8_last_error()
    assert L.h3fp8_quant_blocks(p, 512, 0, 1 << 27, 512, 1, p, 512, p, 1, 1 << 27, z) == -22


def test_outputs_that_share_memory_are_refused(calls):
    """Two entries in one place, an output over the other's input, an output shifted against its own input; in place and
    views that take turns are taken."""
    x = torch.zeros(8, 272, dtype=BF16)
    base = torch.zeros(64, dtype=F32)
    for st in ((1, 1), (0, 8), (2, 3)):
        with pytest.raises(ValueError, match="overlap"):
            ops.quant_blocks(x, scale=base.as_strided((8, 3), st))
    ops.quant_blocks(x, scale=base.as_strided((8, 3), (3, 1)))
    T, H, D = 5, 2, 64
    w, tab = torch.zeros(D, dtype=BF16), torch.zeros(T, D)
    qkv = torch.zeros(T, 3 * H * D, dtype=BF16)
    q, k, v = (qkv[:, i * H * D:(i + 1) * H * D].view(T, H, D) for i in range(3))
    pair = torch.zeros(T, H, 2, D, dtype=BF16)
    flat = torch.zeros(T * H * D + 8, dtype=BF16)
    run = lambda q, k, out: ops.qk_norm_rope(q, k, w, w, tab, 1e-6, out=out)            # noqa: E731
    for a, b, out in ((q, k, (q, k)), (q, k, (v, k)), (pair[:, :, 0], pair[:, :, 1], (pair[:, :, 0], pair[:, :, 1])),
                      (q[:1], k[:1], (q[:1], k[:1])), (q, k, (torch.empty_like(q), torch.empty_like(k))),
                      (q[:, :1], q[:, 1:], (q[:, :1], q[:, 1:]))):
        run(a, b, out)
    whole = torch.zeros(T, H, D, dtype=BF16)
    n = len(calls)
    for a, b, out in ((q, k, (k, q)), (q, q, (q, q)), (q, k, (v, v)), (q, k, (whole[:, :1].expand(T, H, D), k)),
                      (q, k, (k, torch.empty_like(k))),
                      (flat[:-8].view(T, H, D), k, (flat[8:].view(T, H, D), torch.empty_like(k)))):
        with pytest.raises(ValueError):
            run(a, b, out)
    assert len(calls) == n


def test_native_host_path_leaves_other_calls_to_python():
    h = _lib.host()
    assert h is not None, "the native host path is not built"
    x = torch.zeros(4, 64, dtype=BF16)
    assert h.quant_blocks(x, 1) is None and h.quant_blocks(x, 2) is None and h.quant_blocks(x, 2 ** 80) is None
    assert h.silu_mul_quant_blocks(x) is None
    assert h.gemm_blocks(x, x, x, x, BF16, None, None) is None and h.gemm_blocks(None, x, x, x, BF16, None, None) is None
    assert h.grouped_gemm_blocks(x, x, x, x, x, BF16, None) is None
    assert h.qk_norm_rope(x, x, x, x, x, 1e-6, None, False) is None and h.qk_norm_rope(x, x, x, x, x, 1, None, False) is None
    for f in (h.quant_blocks, h.silu_mul_quant_blocks, h.gemm_blocks, h.grouped_gemm_blocks, h.qk_norm_rope):
        assert f() is None
