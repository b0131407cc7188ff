"""Inputs and float64 references of the expert layer's tests."""
import torch

from _blocks import cdiv, spread

E4M3 = torch.float8_e4m3fn
INF = float("inf")


def route64(logits, k, scoring="softmax", renormalize=True, scale=1.0, bias=None):
    """The definition, token by token on the CPU: weights in float64, whole numbers as the kernel returns them."""
    x = logits.detach().cpu().double()
    T, E = x.shape
    weights, experts = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1, dtype=torch.int32)
    for t in range(T):
        row = x[t]
        top = row[row == row].max() if bool((row == row).any()) else torch.tensor(-INF)
        e = torch.exp(row - (0.0 if top == -INF else top))
        score = e / e.nansum() if scoring == "softmax" else 1.0 / (1.0 + torch.exp(-row))
        key = row if bias is None else torch.where(row > -INF, torch.nan_to_num(score, nan=0.0) + bias.cpu().double(), -INF)
        key = torch.where((row > -INF) & (key == key), key, torch.tensor(-INF, dtype=torch.float64))
        order = sorted((e for e in range(E) if key[e] > -INF), key=lambda e: (-float(key[e]), e))[:k]
        if order:
            experts[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
            w = score[order]
            if renormalize:
                total = w.sum()
                w = torch.zeros_like(w) if total == 0 else w / total
            weights[t, :len(order)] = float("nan") if bool((row != row).any()) else w * scale
    flat = experts.flatten().tolist()
    lists = [[p for p, e in enumerate(flat) if e == n] for n in (*range(E), -1)]
    order = [p for row in lists for p in row]
    offsets = [0]
    for row in lists[:E]:
        offsets.append(offsets[-1] + len(row))
    place = torch.empty(T * k, dtype=torch.int32)
    place[torch.tensor(order, dtype=torch.long)] = torch.arange(T * k, dtype=torch.int32)
    return weights, experts, torch.tensor(offsets, dtype=torch.int32), torch.tensor(order, dtype=torch.int32), place.view(T, k)


def expert_weights(g, E, N, K, device="cuda"):
    """e4m3 codes over their whole finite range [E, N, K] and block scales of uneven size."""
    w = (torch.randn(E, N, K, generator=g, device=device) * 60.0).clamp(-448.0, 448.0).to(E4M3)
    s = torch.exp(0.5 * torch.randn(E, cdiv(N, 128), cdiv(K, 128), generator=g, device=device)) * (1.0 / (60.0 * K ** 0.5))
    return w, s


def routing_of(ops, experts, weights, E):
    """A routing of given experts [T, k] (-1: none) and weights."""
    T, k = experts.shape
    flat = experts.flatten().tolist()
    order = sorted(range(T * k), key=lambda p: (flat[p] if flat[p] >= 0 else E, p))
    count = [sum(e == n for e in flat) for n in range(E)]
    offsets = torch.tensor([0, *count]).cumsum(0).to(torch.int32)
    place = torch.empty(T * k, dtype=torch.int32)
    place[torch.tensor(order, dtype=torch.long)] = torch.arange(T * k, dtype=torch.int32)
    dev = weights.device
    return ops.Routing(weights, experts.to(dev), offsets.to(dev), torch.tensor(order, dtype=torch.int32, device=dev), place.view(T, k).to(dev))


def moe64(x, w1, s1, w2, s2, weights, experts, residual=None):
    """(the layer in float64, a bound on what fp32 sums may be off by).

    A sum of up to 8192 products takes at most 4 MFMAs of 32 products (6 roundings each), 64 fmas and 7 additions per element
    before the next rounding: under 100 roundings of 2^-24, twice that if the MFMA cuts instead, 2^-16.3 of the sum of
    magnitudes: 2^-16.  h is carried to 2^-18 of itself, the SwiGLU's fp32 steps are some 2^-22."""
    T, H = x.shape
    E, F = w1.shape[0], w2.shape[2]
    eps = 2.0 ** -16
    y = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for e in range(E):
        gate = (weights.double() * (experts == e)).sum(dim=1)
        rows = ((experts == e).any(dim=1)).nonzero().flatten()
        if rows.numel() == 0:
            continue
        W1 = w1[e].double() * spread(s1[e].double(), 2 * F, H, 128)
        W2 = w2[e].double() * spread(s2[e].double(), H, F, 128)
        xr = x[rows].double()
        gu, mag = xr @ W1.t(), xr.abs() @ W1.abs().t()
        g, u = gu[:, :F], gu[:, F:]
        sig = torch.sigmoid(g)
        h = g * sig * u
        dh = eps * (1.1 * mag[:, :F] * u.abs() + (g * sig).abs() * mag[:, F:] + 2 * h.abs())
        w = gate[rows, None]
        y[rows] += w * (h @ W2.t())
        bound[rows] += w.abs() * (dh @ W2.abs().t() + eps * (h.abs() @ W2.abs().t()))
    if residual is not None:
        y += residual.double()
        bound += residual.double().abs() * 2.0 ** -23
    return y, bound


def check(y, y64, bound, dtype):
    """One rounding to the type on top of the bound."""
    info = torch.finfo(dtype)
    tol = (y64.abs() + bound) * (info.eps / 2) + bound + info.smallest_normal * info.eps
    bad = ~((y.double() - y64).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), float(((y.double() - y64).abs() / tol).max()))
