"""The balance loss and the router's backward pass in 64 bits (numpy), from their definitions. `terms` returns, beside each
result, the magnitudes that its rounding errors scale with."""
import numpy as np

CLAMP = 2.0 ** -14


def sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-np.asarray(z, np.float64)))


def shares(z):
    """p_te = s_te / sum_j s_tj, through log s so that rows of tiny sigmoids keep their shares; a row of -inf is 0"""
    z = np.asarray(z, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        ls = np.where(z < -30, z, -np.log1p(np.exp(-np.maximum(z, -30.0))))
        m = ls.max(axis=1, keepdims=True)
        w = np.exp(ls - m)
        p = w / w.sum(axis=1, keepdims=True)
    return np.where(m == -np.inf, 0.0, p)


def balance(z, sel, alpha, seq, gloss=None):
    """(counts, loss, dz, scale of dz's rounding errors)"""
    z = np.asarray(z, np.float64)
    n, ne = z.shape
    topk, nseq = sel.shape[1], len(seq) - 1
    counts = np.zeros((nseq, ne), np.int32)
    loss, dz, mag = np.zeros(nseq), np.zeros((n, ne)), np.zeros((n, ne))
    for s in range(nseq):
        a, b = int(seq[s]), int(seq[s + 1])
        if a == b:
            continue
        picks = sel[a:b].ravel()
        picks = picks[(picks >= 0) & (picks < ne)]
        counts[s] = np.bincount(picks, minlength=ne)
        f = counts[s].astype(np.float64) * ne / (topk * (b - a))
        p = shares(z[a:b])
        loss[s] = alpha * float(f @ p.mean(axis=0))
        g = alpha / (b - a) * (1.0 if gloss is None else float(gloss[s]))
        om = sigmoid(-z[a:b])
        D = (p @ f)[:, None]
        dz[a:b] = g * p * om * (f[None] - D)
        mag[a:b] = abs(g) * p * om * (f[None] + D)
    return counts, loss, dz, mag


def route_dz(z, sel, dw, dz_in, scale):
    """(dz, scale of its rounding errors)"""
    z = np.asarray(z, np.float64)
    n, ne = z.shape
    dz = np.zeros((n, ne)) if dz_in is None else dz_in.astype(np.float64)
    mag = np.abs(dz)
    if dw is None:
        return dz, mag
    dw = dw.astype(np.float64)
    ok = (sel >= 0) & (sel < ne)
    zk = np.take_along_axis(z, np.where(ok, sel, 0), axis=1)
    sk = np.where(ok, sigmoid(zk), 0.0)
    om = np.where(ok, sigmoid(-zk), 0.0)
    dw = np.where(ok, dw, 0.0)
    S = sk.sum(axis=1, keepdims=True)
    D = (dw * sk).sum(axis=1, keepdims=True)
    A = (np.abs(dw) * sk).sum(axis=1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        big = S > CLAMP
        gz = np.where(big, scale / S * (dw - D / S), scale / CLAMP * dw) * sk * om
        gm = np.where(big, scale / S * (np.abs(dw) + A / S), scale / CLAMP * np.abs(dw)) * sk * om
    for k in range(sel.shape[1]):
        for t in np.nonzero(ok[:, k])[0]:
            dz[t, sel[t, k]] += gz[t, k]
            mag[t, sel[t, k]] += gm[t, k]
    return dz, mag


def weights(z, sel, scale):
    """the routing weights themselves (for differences)"""
    sk = np.take_along_axis(sigmoid(z), sel, axis=1)
    return scale * sk / np.maximum(sk.sum(axis=1, keepdims=True), CLAMP)
