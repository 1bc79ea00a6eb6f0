"""Q4_K matrices for tests, from the format's definition: 144 bytes = fp16 d, fp16 dmin, 12 bytes of 6-bit scales and mins, 128
bytes of quants (see dequant)."""
import numpy as np

from oracle import oracle as orc
from tests.golden import gen


def matrix(seed, R, K):
    """bytes of an R x K matrix: quant and scale bytes from hash words, d in [6e-5, 4e-3], dmin about 7 d"""
    nb = R * (K // 256)
    w = gen.words(seed, 77, nb * 19).reshape(nb, 19)
    b = w[:, :18].copy().view(np.uint8).reshape(nb, 144)
    d = (np.uint64(0x0C00) + w[:, 18] % np.uint64(0x1000)).astype(np.uint16)
    b[:, 0:2] = d.view(np.uint8).reshape(nb, 2)
    b[:, 2:4] = (7 * d.view(np.float16).astype(np.float32)).astype(np.float16).view(np.uint8).reshape(nb, 2)
    return b.reshape(-1)


def fields(w, R, K):
    """(d, dmin [R][nb], scales, mins [R][nb][8], quants [R][nb][8][32]) as integers and float64"""
    b = np.asarray(w, np.uint8).reshape(R, K // 256, 144)
    d = b[..., 0:2].copy().view(np.float16)[..., 0].astype(np.float64)
    m = b[..., 2:4].copy().view(np.float16)[..., 0].astype(np.float64)
    s = b[..., 4:16].astype(np.int64)
    sc, mn = np.empty(b.shape[:2] + (8,), np.int64), np.empty(b.shape[:2] + (8,), np.int64)
    for j in range(8):
        if j < 4:
            sc[..., j], mn[..., j] = s[..., j] % 64, s[..., j + 4] % 64
        else:
            sc[..., j] = s[..., j + 4] % 16 + 16 * (s[..., j - 4] // 64)
            mn[..., j] = s[..., j + 4] // 16 + 16 * (s[..., j] // 64)
    qs = b[..., 16:].reshape(R, K // 256, 4, 32).astype(np.int64)
    q = np.stack([qs % 16, qs // 16], axis=3).reshape(R, K // 256, 8, 32)
    return d, m, sc, mn, q


def dequant(w, R, K):
    d, m, sc, mn, q = fields(w, R, K)
    return ((d[..., None] * sc)[..., None] * q - (m[..., None] * mn)[..., None]).reshape(R, K)


def q8k_rows(n, K, seed, scale=3.0):
    return orc.quantize_q8k(gen.uniform(seed, 78, (n, K), scale))


def error_bound(w, R, K, q, d):
    """What the fp32 chain may be off by, [n][R]: per block isum, d * isum and the inner fma round once each, and each of the nb
    outer fmas rounds a partial sum: at most (nb + 3) half steps of sum_b |d8| (|d isum| + |dmin summ|), and second-order terms"""
    dd, m, sc, mn, qq = fields(w, R, K)
    nb, n = K // 256, q.shape[0]
    x = q.reshape(n, nb, 8, 32).astype(np.float64)
    isum = np.einsum("tbjl,rbjl->trb", x, (qq * sc[..., None]).astype(np.float64))
    summ = np.einsum("tbj,rbj->trb", x.sum(axis=3), mn.astype(np.float64))
    mag = (np.abs(d.astype(np.float64))[:, None] * (np.abs(dd[None] * isum) + np.abs(m[None] * summ))).sum(axis=2)
    return 1.01 * (nb + 3) * 2.0 ** -24 * mag + 1e-40
