"""What the router, the layer of experts and the product with an epilogue refuse (CPU): before any launch, in Python and again at
the C entry."""
import ctypes

import pytest
import torch

from h3_tp2_amd import _lib, ops
from test_blocks_args import _operands, refused

E4M3, BF16, FP16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_call_on", lambda t, name, *args: seen.append((name, args)))
    return seen


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU only"):
        ops.moe_route(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="GPU only"):
        ops.gemm_blocks_act(**_operands(), activation="silu")
    with pytest.raises(ValueError, match="GPU only"):
        ops.moe_blocks(**_layer())


def test_route(calls):
    x = torch.zeros(9, 24)
    r = ops.moe_route(x, 3)
    assert isinstance(r, ops.Routing)
    assert [tuple(t.shape) for t in r] == [(9, 3), (9, 3), (25,), (27,), (9, 3)]
    assert [t.dtype for t in r] == [F32] + 4 * [torch.int32]
    ops.moe_route(x.to(BF16), 1, "sigmoid", False, 2.5, torch.zeros(24))
    n = len(calls)
    refused(lambda **kw: ops.moe_route(**{"logits": x, "k": 3, **kw}), dict(k=0), dict(k=25), dict(k=17), dict(k=2.0), dict(logits=x[0]), dict(logits=x.t()),
            dict(logits=x.double()), dict(logits=torch.zeros(2, 513)), dict(logits=torch.zeros(2, 0)), dict(scoring="relu"),
            dict(bias=torch.zeros(23)), dict(bias=torch.zeros(24, dtype=BF16)), dict(bias=torch.zeros(48)[::2]))
    assert len(calls) == n


def _layer(T=6, E=4, k=2, H=272, F=144, dtype=BF16):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return dict(x=torch.zeros(T, H, dtype=dtype), w_gate_up=torch.zeros(E, 2 * F, H, dtype=E4M3), scale_gate_up=torch.ones(E, 3, 3),
                w_down=torch.zeros(E, H, F, dtype=E4M3), scale_down=torch.ones(E, 3, 2),
                routing=ops.Routing(torch.zeros(T, k), z(T, k), z(E + 1), z(T * k), z(T, k)))


def test_layer(calls):
    ok = _layer()
    assert ops.moe_blocks(**ok).shape == (6, 272)
    res = torch.zeros(6, 272, dtype=BF16)
    out = res.clone()
    assert ops.moe_blocks(**ok, residual=res, out=out) is out
    ops.moe_blocks(**ok, residual=out, out=out)
    ops.moe_blocks(**ok, residual=res[:1].expand(6, 272))
    n = len(calls)
    r = ok["routing"]
    refused(lambda **kw: ops.moe_blocks(**{**ok, **kw}), dict(x=ok["x"].float()), dict(x=ok["x"][0]), dict(x=torch.zeros(6, 256, dtype=BF16)),
            dict(x=torch.zeros(272, 6, dtype=BF16).t()), dict(w_gate_up=ok["w_gate_up"].view(torch.uint8)), dict(w_gate_up=ok["w_gate_up"][:, :144]),
            dict(w_down=ok["w_down"][:3]), dict(w_down=ok["w_down"][0]), dict(scale_gate_up=torch.ones(4, 3, 2)),
            dict(scale_down=torch.ones(4, 3, 2, dtype=BF16)), dict(residual=res.to(FP16)), dict(residual=res[:5]), dict(out=res.to(FP16)),
            dict(out=res[:5]), dict(routing=r._replace(weights=r.weights.to(BF16))), dict(routing=r._replace(experts=r.experts.long())),
            dict(routing=r._replace(offsets=r.offsets[:4])), dict(routing=r._replace(order=r.order[:-1])),
            dict(routing=r._replace(experts=torch.zeros(6, 4, dtype=torch.int32)[:, ::2])), dict(routing=r._replace(weights=torch.zeros(6, 5))))
    # rows that the output shares with the residual in part
    flat = torch.zeros(8 * 272, dtype=BF16)
    refused(lambda **kw: ops.moe_blocks(**{**ok, **kw}), dict(residual=flat[272:7 * 272].view(6, 272), out=flat[:6 * 272].view(6, 272)))
    with pytest.raises(ValueError, match="at most 128 tokens"):
        ops.moe_blocks(**_layer(T=129))
    assert len(calls) == n


def test_product_with_an_epilogue(calls):
    ok = _operands()
    assert ops.gemm_blocks_act(**ok, activation="gelu").shape == (8, 272)
    res = torch.zeros(8, 272, dtype=FP16)
    ops.gemm_blocks_act(**ok, out_dtype=FP16, bias=torch.zeros(272, dtype=FP16), residual=res, out=res)
    n = len(calls)
    flat = torch.zeros(10 * 272, dtype=BF16)
    refused(lambda **kw: ops.gemm_blocks_act(**{**ok, **kw}), dict(activation="tanh"), dict(activation=1), dict(residual=res),
            dict(residual=torch.zeros(8, 256, dtype=BF16)), dict(residual=torch.zeros(272, 8, dtype=BF16).t()), dict(out_dtype=F32),
            dict(bias=torch.zeros(272)), dict(a=ok["a"].to(BF16)), dict(scale_a=torch.ones(8, 3)),
            dict(residual=flat[272:9 * 272].view(8, 272), out=flat[:8 * 272].view(8, 272)))
    assert len(calls) == n


def test_c_entry_bounds_every_stride():
    """The experts' offsets, and strides whose products would pass 64 bits."""
    L = _lib.load()
    p = ctypes.c_void_p(4096)

    def layer(ldx=256, ld1=256, ld2=128, s1=(4, 2, 1), s2=(4, 2, 1)):
        return L.h3fp8_moe_blocks(p, ldx, 0, 4, 256, 128, 8, 2, p, 1 << 16, ld1, p, *s1, p, 1 << 16, ld2, p, *s2, p, p, p, p, None, 0, p, 256, p, 0, None)
    big = 1 << 28
    for kw in (dict(s1=(big, 2, 1)), dict(s2=(big, 2, 1)), dict(s1=(4, big, 1)), dict(s2=(4, big, 1)), dict(s1=(4, 2, big)), dict(s1=(1 << 62, 2, 1)),
               dict(s2=(1 << 62, 2, 1)), dict(s2=(4, 1 << 62, 1)), dict(s2=(4, 2, 1 << 62)), dict(ldx=1 << 62), dict(ld1=1 << 62), dict(ld2=1 << 62)):
        assert layer(**kw) == -22 and b"too large" in _lib.load().h3fp8_last_error(), kw


def test_c_entries():
    """The C side checks again, before any HIP call."""
    L = _lib.load()
    p = ctypes.c_void_p(4096)

    def route(logits=p, ld=64, dtype=2, T=4, E=64, k=2, scoring=0, out=p, offsets=p, ws=None, ws_bytes=0, bias=None):
        return L.h3fp8_moe_route(logits, ld, dtype, T, E, k, scoring, 1, 1.0, bias, out, out, offsets, out, out, ws, ws_bytes, None)
    for kw in (dict(T=-1), dict(E=0), dict(E=513), dict(k=0), dict(k=17), dict(E=4, k=5), dict(dtype=3), dict(scoring=2), dict(logits=None),
               dict(out=None), dict(offsets=None), dict(T=129), dict(T=129, ws=p, ws_bytes=3 * 68 * 4 - 1), dict(logits=ctypes.c_void_p(4098)),
               dict(bias=ctypes.c_void_p(4098)), dict(T=1 << 31), dict(ld=-1)):
        assert route(**kw) == -22, kw
    assert L.h3fp8_moe_route_workspace(128, 64) == 0 and L.h3fp8_moe_route_workspace(129, 64) == 3 * 68 * 4
    assert L.h3fp8_moe_route_workspace(1 << 24, 8) <= 512 * 12 * 4

    def layer(x=p, ldx=256, dtype=0, T=4, H=256, F=128, E=8, k=2, w=p, we=1 << 16, ld1=256, ld2=128, s=p, sn=2, sk=1, r=p, res=None, ldr=256, y=p,
              ldy=256, ws=p, ws_bytes=4 * 2 * 128 * 4):
        return L.h3fp8_moe_blocks(x, ldx, dtype, T, H, F, E, k, w, we, ld1, s, 4, sn, sk, w, we, ld2, s, 4, sn, sk, r, r, r, r, res, ldr, y, ldy, ws,
                                  ws_bytes, None)
    for kw in (dict(T=-1), dict(T=129), dict(E=0), dict(E=513), dict(k=0), dict(k=9), dict(k=17, E=32), dict(dtype=2), dict(H=0), dict(H=248), dict(F=120), dict(F=(1 << 22) + 16),
               dict(x=None), dict(w=None), dict(s=None), dict(r=None), dict(y=None), dict(ws=None), dict(ws_bytes=4095), dict(ldx=255), dict(ldx=252),
               dict(ldy=254), dict(ld1=240), dict(ld1=264), dict(ld2=120), dict(we=8), dict(we=-16), dict(sn=-1), dict(x=ctypes.c_void_p(4104)),
               dict(y=ctypes.c_void_p(4100)), dict(res=ctypes.c_void_p(4100)), dict(res=p, ldr=-4), dict(res=p, ldr=2), dict(s=ctypes.c_void_p(4098)),
               dict(r=ctypes.c_void_p(4098)), dict(ldx=1 << 24), dict(ld1=1 << 26), dict(sn=1 << 30)):
        assert layer(**kw) == -22, kw
    assert layer(T=0) == 0
    # h alone for a token or a few, else the pairs' results too
    ws = L.h3fp8_moe_blocks_workspace
    assert ws(1, 16, 256, 128, 32) == 16 * 4 * 128 and ws(2, 9, 256, 128, 32) == 18 * 4 * (128 + 256)
    assert ws(8, 1, 256, 128, 32) == 8 * 4 * 128 and ws(8, 1, 4096, 2048, 32) == 8 * 4 * (2048 + 4096) and ws(9, 1, 256, 128, 32) == 9 * 4 * (128 + 256)

    def act(bias=None, act=0, res=None, ldr=64, ldy=64, out_dtype=0, M=4, N=64, K=64):
        return L.h3fp8_gemm_blocks_act(p, 64, p, 64, p, 1, 1, p, 1, 1, bias, act, res, ldr, p, ldy, out_dtype, M, N, K, None)
    for kw in (dict(act=-1), dict(act=5), dict(bias=ctypes.c_void_p(4104)), dict(res=ctypes.c_void_p(4104)), dict(res=p, ldr=56), dict(res=p, ldr=68),
               dict(res=p, ldr=1 << 22), dict(res=p, ldr=-64), dict(N=72), dict(K=72), dict(ldy=56), dict(out_dtype=2)):
        assert act(**kw) == -22, kw
    assert act(M=0) == 0
