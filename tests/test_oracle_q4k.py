"""CPU: the oracle's Q4_K against a 64-bit product of the dequantised matrix, built here from the format's definition."""
import numpy as np
import pytest

from oracle import oracle as orc
from tests._q4k import dequant, error_bound, matrix, q8k_rows

U = 2.0 ** -24


@pytest.mark.parametrize("R,K,n", [(3, 256, 2), (5, 2048, 3), (2, 7168, 1), (2, 18432, 2)])
def test_oracle_matches_the_definition(R, K, n):
    w = matrix(K + R, R, K)
    q, d, bs = q8k_rows(n, K, seed=K + n)
    y = orc.matvec_kq(orc.Q4K, w, R, K, q, d, bs)
    x = q.astype(np.float64) * np.repeat(d.astype(np.float64), 256, axis=1)
    want = x @ dequant(w, R, K).T
    assert np.all(np.abs(y - want) <= error_bound(w, R, K, q, d)), np.abs(y - want).max()


def test_oracle_dequantises():
    w = matrix(7, 4, 512)
    got = orc.dequant_kq(orc.Q4K, w, 512).astype(np.float64)
    want = dequant(w, 4, 512)
    # d * scale and dmin * min are exact in 17 bits, times q in 21: only the subtraction rounds
    assert np.all(np.abs(got - want) <= U * np.abs(want) * 1.001 + 1e-45)


def test_extremes_are_exact_integers():
    """all quants 15, scales 63, activations +-127: |isum| reaches 256 * 63 * 15 * 127 > 2^24, rounded to fp32 once"""
    K = 256
    b = np.full((2, 144), 0xFF, np.uint8)
    b[:, 0:2] = np.frombuffer(np.float16(1.0).tobytes(), np.uint8)
    b[:, 2:4] = np.frombuffer(np.float16(0.0).tobytes(), np.uint8)
    q = np.full((2, K), 127, np.int8); q[1] = -127
    d = np.ones((2, 1), np.float32)
    bs = q.reshape(2, 16, 16).sum(axis=2).astype(np.int16)
    y = orc.matvec_kq(orc.Q4K, b.ravel(), 2, K, q, d, bs)
    assert np.array_equal(y, np.array([[1, 1], [-1, -1]]) * np.float32(256 * 63 * 15 * 127))
