"""GPU: the balance loss over long sequences, held to a bound in which a single lost or doubled row of the longest sequence shows.

u = 2^-24. Every term is positive, so relative errors add up along the longest chain of additions: p 28 u (exp, sigmoid, the row's sum and
its reciprocal, as in test_gpu_router_train.py). A workgroup sums a chunk of T / chunks rows, each of its 16 waves 4 rows of every 64, one
after another, then its 16 waves, then the chunks in four slices and their join: 4 ceil(T / chunks / 64) + 16 + ceil(chunks / 4) + 4. The
mean's division, f and alpha 7 u, the sum over the experts 12 u. A row's own part of the loss is alpha f . p_t / T, which has to be
above twice the bound."""
import numpy as np
import pytest

from tests import _train_ref as ref
from tests.test_gpu_router_train import U, routed, run_balance

pytestmark = pytest.mark.gpu


def chunks(n, nseq):
    """workgroups a sequence of the sums (rows by the mean length; 512 in all where there are several)"""
    return 1 if n <= 128 * nseq else max(1, min(-(-n // (64 * nseq)), 512 // nseq, 256))


def one_long(n, nseq, long):
    """offsets of nseq sequences of n rows, the middle one `long`, the others sharing the rest"""
    rest = n - long
    cuts = [rest * i // (nseq - 1) for i in range(nseq)]
    m = nseq // 2
    return [c if i <= m else c + long for i, c in zip([*range(m + 1), *range(m + 1, nseq + 1)], cuts[:m + 1] + cuts[m:])]


@pytest.mark.parametrize("n,ne,topk,seq,shows", [
    (20011, 256, 8, [0, 1, 9000, 20011], True),
    (5000, 32, 2, [0, 4999, 5000], True),
    (16384, 130, 4, None, True),
    (8192, 64, 8, one_long(8192, 64, 8000), True),             # one workgroup a sequence: 125 turns of 64 rows
    (30000, 64, 2, one_long(30000, 200, 27000), False),        # two
    (40000, 20, 3, one_long(40000, 600, 39000), False)])       # nine tenths of the rows in one of very many
def test_long_sequences(ctx, n, ne, topk, seq, shows):
    rng, z, sel = routed(n, ne, topk, n + ne)
    print("balance n %d sequences %d" % (n, 1 if seq is None else len(seq) - 1), flush=True)
    seq = [0, n] if seq is None else seq
    nseq, T = len(seq) - 1, np.diff(seq)
    assert seq[-1] == n and np.all(T >= 0)
    alpha = np.float32(1e-3)
    gloss = rng.standard_normal(nseq).astype(np.float32)
    got = run_balance(ctx, z, sel, alpha, seq if nseq > 1 else None, gloss if nseq > 1 else None)
    counts, loss, dz, mag = ref.balance(z, sel, alpha, seq, gloss if nseq > 1 else None)
    c = chunks(n, nseq)
    tol = (28 + 4 * np.ceil(np.ceil(T / c) / 64) + 16 + np.ceil(c / 4) + 4 + 7 + 12) * U
    if shows:
        s = int(np.argmax(T))
        part = float(alpha) * (ref.shares(z[seq[s]:seq[s + 1]]) @ (counts[s] * ne / (topk * T[s]))) / T[s]
        assert part.min() > 2 * tol[s] * loss[s], (part.min(), tol[s] * loss[s])
    assert np.array_equal(got[0], counts)
    err = np.abs(got[1] - loss) / np.maximum(loss, 1e-44)
    print("loss error / bound %.3f" % (err / tol).max(), flush=True)
    assert np.all(err <= tol), (err / tol).max()
    assert np.all(np.abs(got[2] - dz) <= 90 * U * mag + 1e-44)
