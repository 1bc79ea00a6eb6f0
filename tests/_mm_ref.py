"""The 16-bit products, their epilogues, gradients and the combine in 64 bits (torch, CPU), from their definitions; beside results the
magnitudes that their rounding errors scale with."""
import math

import torch

F8 = torch.float64
U = 2.0 ** -24                 # half an fp32 step
C, A = 2 * math.sqrt(2 / math.pi), 0.044715


def half(t):
    """half a step of the type, relative"""
    return torch.finfo(t).eps / 2


def sigma(t):
    return 1 / (1 + torch.exp(-t))


def arg(z, act):
    return z if act == "silu" else C * (z + A * z ** 3)


def act(z, kind):
    return z * sigma(arg(z, kind)) if kind else z


def slope(z, kind):
    if not kind:
        return torch.ones_like(z)
    t = arg(z, kind)
    d = torch.ones_like(z) if kind == "silu" else C * (1 + 3 * A * z ** 2)
    return sigma(t) + z * d * sigma(t) * sigma(-t)


def spans(offsets, n, ne):
    if offsets is None:
        return [(0, n)]
    o = [min(max(int(v), 0), n) for v in offsets]
    return [(o[e], max(o[e], o[e + 1])) for e in range(ne)]


def rows(x, perm, topk, a, b):
    """x's rows of slots a .. b - 1 in 64 bits, rows outside x as zeros"""
    if perm is None:
        return x[a:b].to(F8)
    r = perm[a:b].long() // topk
    ok = (r >= 0) & (r < x.shape[0])
    return torch.where(ok[:, None], x[r.clamp(0, max(0, x.shape[0] - 1))].to(F8), 0.0)


def products(x, W, offsets, perm=None, topk=1):
    """(z, sum |x w|) [n][R] of every slot an expert has, NaN elsewhere"""
    n = x.shape[0] if perm is None else perm.numel()
    Ws = W[None] if offsets is None else W
    z = torch.full((n, Ws.shape[1]), float("nan"), dtype=F8)
    m = z.clone()
    for e, (a, b) in enumerate(spans(offsets, n, Ws.shape[0])):
        if a < b:
            r, w = rows(x, perm, topk, a, b), Ws[e].to(F8)
            z[a:b], m[a:b] = r @ w.t(), r.abs() @ w.abs().t()
    return z, m


def grads(dz, x, W, offsets, perm=None, topk=1):
    """(dx, its magnitude, dW, its magnitude)"""
    n = dz.shape[0]
    Ws = W[None] if offsets is None else W
    dx = torch.full((n, Ws.shape[2]), float("nan"), dtype=F8)
    mx = dx.clone()
    dW, mW = torch.zeros(Ws.shape, dtype=F8), torch.zeros(Ws.shape, dtype=F8)
    for e, (a, b) in enumerate(spans(offsets, n, Ws.shape[0])):
        if a < b:
            d, r, w = dz[a:b].to(F8), rows(x, perm, topk, a, b), Ws[e].to(F8)
            dx[a:b], mx[a:b] = d @ w, d.abs() @ w.abs()
            dW[e], mW[e] = d.t() @ r, d.abs().t() @ r.abs()
    return (dx, mx, dW[0], mW[0]) if offsets is None else (dx, mx, dW, mW)


def combine(o, inv, w, sel, ne, residual):
    """(y, sum |w o| + |residual|)"""
    n, k = w.shape
    y = torch.zeros((n, o.shape[1]), dtype=F8) if residual is None else residual.to(F8)
    m = y.abs()
    inv = inv.view(n, k)
    for t in range(n):
        for j in range(k):
            if 0 <= int(sel[t, j]) < ne and 0 <= int(inv[t, j]) < o.shape[0]:
                v = float(w[t, j]) * o[int(inv[t, j])].to(F8)
                y[t] += v
                m[t] += v.abs()
    return y, m


def combine_grad(dy, o, inv, w, sel, ne):
    """(do, dw, dw's magnitude); slots of no pick NaN"""
    n, k = w.shape
    do = torch.full(o.shape, float("nan"), dtype=F8)
    dw, mw = torch.zeros((n, k), dtype=F8), torch.zeros((n, k), dtype=F8)
    inv = inv.view(n, k)
    for t in range(n):
        for j in range(k):
            s = int(inv[t, j])
            if 0 <= int(sel[t, j]) < ne and 0 <= s < o.shape[0]:
                do[s] = float(w[t, j]) * dy[t].to(F8)
                p = o[s].to(F8) * dy[t].to(F8)
                dw[t, j], mw[t, j] = p.sum(), p.abs().sum()
    return do, dw, mw


def order(sel, ne):
    """(offsets, perm, inv) of picks, pairs of no expert without a slot: their inv is -1, the last entries of perm -1"""
    flat = sel.reshape(-1).tolist()
    perm = [i for e in range(ne) for i, s in enumerate(flat) if s == e]
    off = [0]
    for e in range(ne):
        off.append(off[-1] + sum(s == e for s in flat))
    inv = [-1] * len(flat)
    for s, i in enumerate(perm):
        inv[i] = s
    perm += [-1] * (len(flat) - len(perm))
    return torch.tensor(off, dtype=torch.int32), torch.tensor(perm, dtype=torch.int32), torch.tensor(inv, dtype=torch.int32)
