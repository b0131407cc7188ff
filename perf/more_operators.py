"""The measured cases of the expert layer's operators and of the block-scaled product with its epilogue.

Three operators, each over its range of sizes: the router, which picks every token's experts and sorts the tokens by expert
(``route``), the whole layer of block-scaled FP8 experts for a few tokens (``moe``), and the block-scaled FP8 product with bias,
activation and residual in its epilogue (``act``).

``run`` is one pass: with ``own`` through ``h3_tp2_amd.ops``, otherwise in elementary torch operations in fp32, rounded
once.  ``exact`` restates the definitions in float64.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
BLOCK = 128
FP8_MAX = 448.0
MIN_SCALE = 1.0 / (448.0 * 512.0)
INF = float("inf")
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decoded token
        dict(name="route_t1", kind="route", T=1, E=32, k=4, pad=0, scoring="softmax", renorm=True, bias=False, dtype="bf16"),
        # a captured decode step of 64 places, 59 of them taken; experts balanced by a bias that the weights do not see
        dict(name="route_t64", kind="route", T=64, E=256, k=8, pad=5, scoring="sigmoid", renorm=True, bias=True, dtype="bf16"),
        # a long prompt, the order in which the product by expert wants its rows
        dict(name="route_t32768", kind="route", T=32768, E=256, k=8, pad=0, scoring="softmax", renorm=False, bias=False,
             dtype="fp32"),
        # one token, two small experts: launches and latency
        dict(name="moe_t1_small", kind="moe", T=1, E=8, k=2, H=1536, F=2304, pad=0, residual=False, dtype="bf16"),
        # one token of a larger layer, onto the residual stream
        dict(name="moe_t1", kind="moe", T=1, E=32, k=4, H=4096, F=2048, pad=0, residual=True, dtype="bf16"),
        # decode of a ragged batch, widths that are no multiples of a block
        dict(name="moe_t37_odd", kind="moe", T=37, E=12, k=3, H=1200, F=1040, pad=2, residual=False, dtype="fp16"),
        # decode of 16 sequences: about two rows per expert, the time is that of the experts' weights
        dict(name="moe_t16", kind="moe", T=16, E=32, k=4, H=4096, F=2048, pad=0, residual=True, dtype="bf16"),
        # the largest batch that counts as few tokens: 32 rows per expert
        dict(name="moe_t128", kind="moe", T=128, E=32, k=8, H=4096, F=2048, pad=0, residual=True, dtype="bf16"),
        # one token through a wide first linear: the weight is read once
        dict(name="act_m1", kind="act", M=1, K=5376, N=21504, act="gelu_tanh", bias=True, residual=False, dtype="bf16"),
        # a short ragged sequence through the out projection onto the residual stream
        dict(name="act_m200", kind="act", M=200, K=7168, N=5376, act="none", bias=True, residual=True, dtype="fp16"),
        # a chunk of a prompt through a first linear
        dict(name="act_m4100", kind="act", M=4100, K=5376, N=14336, act="gelu", bias=True, residual=False, dtype="bf16"),
        # one rank's tokens of a clip through the second linear of the MLP, onto the residual stream
        dict(name="act_m18880", kind="act", M=18880, K=14336, N=5376, act="none", bias=True, residual=True, dtype="bf16"),
    ]


# (K, N) of the linears that the framework's models have, and of small and odd ones
_LINEARS = ((5376, 14336), (7168, 5376), (14336, 5376), (4096, 6144), (1536, 4608), (1536, 1536), (1200, 2064), (528, 720))
# (H, F) of an expert: hidden size, width of the gate and of the up product
_EXPERTS = ((4096, 2048), (4096, 1536), (2048, 2048), (1536, 2304), (2048, 768), (1200, 1040))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("route", "moe", "act"), (3, 5, 4))[0]
    dtype = "fp16" if rng.random() < 0.25 else "bf16"
    if kind == "route":
        T, E = _log_int(rng, 1, 32768), rng.choice((8, 32, 60, 100, 128, 256))
        return dict(kind=kind, T=T, E=E, k=rng.choice((1, 2, 4, 6, 8)), pad=rng.randrange(T // 8 + 1),
                    scoring=rng.choice(("softmax", "sigmoid")), renorm=rng.random() < 0.6, bias=T <= 8192 and rng.random() < 0.4,
                    dtype=rng.choice(("bf16", "fp16", "fp32")))
    if kind == "moe":
        (H, F), T = rng.choice(_EXPERTS), _log_int(rng, 1, 128)
        E = rng.choice((4, 12, 16, 32))
        return dict(kind=kind, T=T, E=E, k=min(E, rng.choice((1, 2, 3, 4, 8))), H=H, F=F, pad=rng.randrange(T // 8 + 1),
                    residual=rng.random() < 0.5, dtype=dtype)
    K, N = rng.choice(_LINEARS)
    act = rng.choice(("none", "silu", "gelu", "gelu_tanh", "relu"))
    return dict(kind=kind, M=_log_int(rng, 1, 18880), K=K, N=N, act=act, bias=rng.random() < 0.6,
                residual=rng.random() < (0.7 if act == "none" else 0.3), dtype=dtype)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, M, K):
    """fp32 activations [M, K] as a linear meets them: rows of log-normal magnitude, 0.1 % outlier channels x40."""
    x = _randn(g, M, K)
    x *= torch.exp(_randn(g, M, 1))
    x[:, torch.randperm(K, generator=g, device="cuda")[:max(1, K // 1000)]] *= 40.0
    return x


def _quant(x, rows):
    """e4m3 codes [M, K] and one fp32 scale per block of rows x 128."""
    M, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, -M % rows))
    b = b.view(b.shape[0] // rows, rows, b.shape[1] // BLOCK, BLOCK)
    s = (b.abs().amax(dim=(1, 3)) / FP8_MAX).clamp_min(MIN_SCALE)
    q = (b * (1.0 / s)[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).to(E4M3)
    return q.view(-1, b.shape[2] * BLOCK)[:M, :K].contiguous(), s


def _weights(g, E, N, K):
    """The block-scaled weights of E linears: [E, N, K] codes, [E, ceil(N / 128), ceil(K / 128)] scales."""
    w = torch.empty(E, N, K, dtype=E4M3, device="cuda")
    s = torch.empty(E, -(-N // BLOCK), -(-K // BLOCK), device="cuda")
    for e in range(E):
        w[e], s[e] = _quant(_randn(g, N, K) * 0.02, BLOCK)
    return w, s


def _logits(g, T, E, pad):
    """Router logits: tokens of unlike certainty, some experts liked more than others; places without a token are masked."""
    x = _randn(g, T, E) * torch.exp(0.3 * _randn(g, T, 1)) + 0.3 * _randn(g, E)
    if pad:
        x[torch.randperm(T, generator=g, device="cuda")[:pad]] = -INF
    return x


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    dt = _TYPES[case["dtype"]]
    st = dict(kind=kind)
    if kind == "route":
        st.update(k=case["k"], scoring=case["scoring"], renorm=case["renorm"], scale=2.5 if case["bias"] else 1.0)
        st["logits"] = _logits(g, case["T"], case["E"], case["pad"]).to(dt)
        st["bias"] = 0.05 * _randn(g, case["E"]) if case["bias"] else None
    elif kind == "moe":
        T, E, k, H, F = (case[n] for n in ("T", "E", "k", "H", "F"))
        # behind a norm: rows of like magnitude, some channels louder
        st["x"] = (_randn(g, T, H) * torch.exp(0.5 * _randn(g, H))).to(dt)
        st["w1"], st["s1"] = _weights(g, E, 2 * F, H)
        st["w2"], st["s2"] = _weights(g, E, H, F)
        # the router's answer
        st["routing"] = _route(_logits(g, T, E, case["pad"]), k, "softmax", True, 1.0, None)
        st["residual"] = _randn(g, T, H).to(dt) if case["residual"] else None
    else:
        M, K, N = case["M"], case["K"], case["N"]
        st["dtype"], st["act"] = dt, case["act"]
        st["a"], sa = _quant(_activations(g, M, K), 1)
        st["sa"] = sa.t().contiguous().t()
        w, s = _weights(g, 1, N, K)
        st["w"], st["sw"] = w[0], s[0]
        st["bias"] = _randn(g, N).mul_(0.1).to(dt) if case["bias"] else None
        st["residual"] = (_randn(g, M, N) * 2.0).to(dt) if case["residual"] else None
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------

def _ops():
    path = os.path.join(os.getcwd(), "minimax-h3-2x-dgx-spark-tp2_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from h3_tp2_amd import ops
    return ops


def run(st):
    return _run_own(st, _ops()) if own else _run_plain(st)


def _run_own(st, ops):
    if st["kind"] == "route":
        return tuple(ops.moe_route(st["logits"], st["k"], st["scoring"], st["renorm"], st["scale"], st["bias"]))
    if st["kind"] == "moe":
        return ops.moe_blocks(st["x"], st["w1"], st["s1"], st["w2"], st["s2"], ops.Routing(*st["routing"]), residual=st["residual"])
    return ops.gemm_blocks_act(st["a"], st["w"], st["sa"], st["sw"], st["dtype"], st["bias"],
                               None if st["act"] == "none" else st["act"], st["residual"])


def _route(logits, k, scoring, renorm, scale, bias):
    """(weights [T, k], experts [T, k], offsets [E + 1], order [T k], place [T, k]): the k best experts of every token, best first and
    the lower index first among equals; an expert at -inf is not chosen, places left over hold -1 with weight 0; the pairs
    (token, choice) sorted by expert, those without one last, and where each pair went."""
    T, E = logits.shape
    x = logits.float()
    top = x.amax(dim=1, keepdim=True)
    if scoring == "softmax":
        e = torch.exp(x - torch.where(top == -INF, 0.0, top))
        score = e / e.sum(dim=1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    key = x
    if bias is not None:                                  # a sum decides: in 64 bits
        d = x.double()
        if scoring == "softmax":
            e = torch.exp(d - torch.where(top == -INF, 0.0, top).double())
            d = e / e.sum(dim=1, keepdim=True)
        else:
            d = 1.0 / (1.0 + torch.exp(-d))
        key = torch.where(x == -INF, -INF, d + bias.double())
    key = key.clone()
    experts = torch.empty(T, k, dtype=torch.int64, device=x.device)
    for j in range(k):
        v, i = key.max(dim=1)
        experts[:, j] = torch.where(v > -INF, i, -1)
        key.scatter_(1, i[:, None], -INF)
    live = experts >= 0
    w = torch.where(live, score.gather(1, experts.clamp_min(0)), 0.0)
    if renorm:
        total = w.sum(dim=1, keepdim=True)
        w = torch.where(total > 0.0, w / total, 0.0)
    flat = torch.where(live, experts, E).view(-1)
    count = (flat[:, None] == torch.arange(E, device=x.device)).sum(dim=0) if T * k * E < 1 << 20 else \
        torch.zeros(E + 1, dtype=torch.int64, device=x.device).index_add_(0, flat, torch.ones_like(flat))[:E]
    offsets = torch.nn.functional.pad(count.cumsum(0), (1, 0))
    order = torch.sort(flat, stable=True)[1]
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device=x.device)
    return w * scale, experts.int(), offsets.int(), order.int(), place.view(T, k).int()


def _spread(s, rows, cols, r):
    """Block scales laid over the values they belong to, in the last two axes (blocks of r x 128)."""
    return s.repeat_interleave(r, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def _swiglu(g, F):
    return g[..., :F] / (1.0 + torch.exp(-g[..., :F])) * g[..., F:]


def _moe(st):
    x, w1, s1, w2, s2 = (st[n] for n in ("x", "w1", "s1", "w2", "s2"))
    weights, experts = st["routing"][:2]
    (T, H), (E, F2, _), k = x.shape, w1.shape, experts.shape[1]
    F, x = F2 // 2, x.float()
    if T * k <= E:                                        # the pairs' own experts
        e = experts.reshape(-1).clamp_min(0).long()
        a = w1.view(torch.uint8)[e].view(E4M3).float() * _spread(s1[e], F2, H, BLOCK)
        h = _swiglu((a * x.repeat_interleave(k, 0)[:, None, :]).sum(dim=2), F)
        a = w2.view(torch.uint8)[e].view(E4M3).float() * _spread(s2[e], H, F, BLOCK)
        y = (a * h[:, None, :]).sum(dim=2) * weights.view(-1, 1)
        y = y.view(T, k, H).sum(dim=1)
    else:                                                 # every expert on every token, weighted
        y = torch.zeros(T, H, device=x.device)
        for e in range(E):
            h = _swiglu(x @ (w1[e].float() * _spread(s1[e], F2, H, BLOCK)).t(), F)
            h = h @ (w2[e].float() * _spread(s2[e], H, F, BLOCK)).t()
            y += h * torch.where(experts == e, weights, 0.0).sum(dim=1, keepdim=True)
    return (y if st["residual"] is None else y + st["residual"].float()).to(st["x"].dtype)


def _activate(y, act):
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return y.clamp_min(0.0) if act == "relu" else y


def _run_plain(st):
    if st["kind"] == "route":
        return _route(st["logits"], st["k"], st["scoring"], st["renorm"], st["scale"], st["bias"])
    if st["kind"] == "moe":
        return _moe(st)
    (M, K), N = st["a"].shape, st["w"].shape[0]
    y = (st["a"].float() * _spread(st["sa"], M, K, 1)) @ (st["w"].float() * _spread(st["sw"], N, K, BLOCK)).t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    y = _activate(y, st["act"])
    return (y if st["residual"] is None else y + st["residual"].float()).to(st["dtype"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    e = 4 if case["dtype"] == "fp32" else 2
    if kind == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return dict(bytes=e * T * E + 16 * T * k + 4 * (E + 1), flops=T * E * (k + 4))
    if kind == "moe":
        T, E, k, H, F = (case[n] for n in ("T", "E", "k", "H", "F"))
        n = (T - case["pad"]) * k
        active = E * (1.0 - (1.0 - k / E) ** (T - case["pad"]))      # experts that some token chose, were all alike
        weights = 3 * H * F + 4 * (math.ceil(2 * F / BLOCK) * math.ceil(H / BLOCK) + math.ceil(H / BLOCK) * math.ceil(F / BLOCK))
        return dict(bytes=int(active * weights) + e * T * H * (3 if case["residual"] else 2) + 8 * T * k, flops=6 * n * H * F)
    M, K, N = case["M"], case["K"], case["N"]
    kb, nb = math.ceil(K / BLOCK), math.ceil(N / BLOCK)
    return dict(bytes=M * K + 4 * M * kb + N * K + 4 * nb * kb + e * M * N * (2 if case["residual"] else 1) + (e * N if case["bias"] else 0),
                flops=2 * M * N * K)


# ---- the same in float64 ---------------------------------------------------------------------------------------------

_CHUNK = 4096


def _product64(a, sa, w, sw):
    """Rows of a times the rows of w, block by block of 128; sa (or None): a scale per row and block."""
    N = w.shape[0]
    y = torch.zeros(a.shape[0], N, dtype=torch.float64, device=a.device)
    for b in range(sw.shape[1]):
        cols = slice(b * BLOCK, (b + 1) * BLOCK)
        part = a[:, cols].double() @ (w[:, cols].double().t() * sw[:, b].double().repeat_interleave(BLOCK)[:N])
        y += part if sa is None else part * sa[:, b, None].double()
    return y


def _sorted64(experts, E):
    """offsets, order and place from the chosen experts, by hand."""
    lists = [[] for _ in range(E + 1)]
    for p, e in enumerate(experts.flatten().tolist()):
        lists[e].append(p)                                # -1: the last list
    offsets, place = [0], [0] * experts.numel()
    for row in lists[:E]:
        offsets.append(offsets[-1] + len(row))
    order = [p for row in lists for p in row]
    for r, p in enumerate(order):
        place[p] = r
    at = dict(dtype=torch.int32, device=experts.device)
    return torch.tensor(offsets, **at), torch.tensor(order, **at), torch.tensor(place, **at).view(experts.shape)


def _route64(st):
    x, k = st["logits"].double(), st["k"]
    T, E = x.shape
    masked = x == -INF
    p = torch.softmax(x.masked_fill(masked.all(dim=1, keepdim=True), 0.0), dim=1) if st["scoring"] == "softmax" else torch.sigmoid(x)
    rank = x if st["bias"] is None else p + st["bias"].double()
    best = torch.sort(rank.masked_fill(masked, -INF), dim=1, descending=True, stable=True)[1][:, :k]
    none = masked.gather(1, best)
    w = p.gather(1, best).masked_fill(none, 0.0)
    if st["renorm"]:
        w = w / w.sum(dim=1, keepdim=True).clamp_min(1e-300)
    experts = best.masked_fill(none, -1).int()
    return (w * st["scale"], experts, *_sorted64(experts, E))


def _moe64(st):
    x, F = st["x"], st["w1"].shape[1] // 2
    weights, experts = st["routing"][:2]
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device) if st["residual"] is None else st["residual"].double()
    chosen = experts.tolist()
    for e in range(st["w1"].shape[0]):
        t = [i for i, row in enumerate(chosen) if e in row]
        if t:
            w = (weights[t].double() * (experts[t] == e)).sum(dim=1, keepdim=True)
            g = _product64(x[t], None, st["w1"][e], st["s1"][e])
            y[t] += w * _product64(g[:, :F] * torch.sigmoid(g[:, :F]) * g[:, F:], None, st["w2"][e], st["s2"][e])
    return y


def _act64(st):
    rows = []
    for m in range(0, st["a"].shape[0], _CHUNK):
        c = slice(m, m + _CHUNK)
        y = _product64(st["a"][c], st["sa"][c], st["w"], st["sw"])
        if st["bias"] is not None:
            y += st["bias"].double()
        if st["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif st["act"] == "gelu":
            y = 0.5 * y * torch.special.erfc(-y / math.sqrt(2.0))
        elif st["act"] == "gelu_tanh":
            y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
        elif st["act"] == "relu":
            y = torch.relu(y)
        rows.append(y if st["residual"] is None else y + st["residual"][c].double())
    return torch.cat(rows)


def exact(case, seed):
    st = prepare(case, seed)
    return {"route": _route64, "moe": _moe64, "act": _act64}[st["kind"]](st)
