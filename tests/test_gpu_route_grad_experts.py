"""GPU: the router's backward pass for experts whose gradients are of very different sizes: what the balance loss gives an expert that
no row picks is a million times and more below what a row's picks get, and is all that its row of dW consists of.

Tolerance of dW[e][j] against the 64-bit product of the kernel's own dlogits a and x, with u = 2^-24, A = max_t |a_te|, X = the largest
|x_tj| of the rows with a gradient, g_t = the largest |a_te| of t's aligned 8 rows:
  sums      an fp32 addition per term at most: (n + 16) u sum |a x|
  halves    an operand's two fp16 halves are off by 2^-11 2^-11 = 2^-22 of it, twice, and the product of the lower ones is left out: 3 * 2^-22
  dz        the lower half has steps of 2^-24 where the 8 rows' maximum is at 2^2 at least: half a step is 2^-27 g. Brought to the run's
            scale, A at 2^14 at least, both halves round to steps of 2^-24 again: 2 * 2^-25 / 2^14 = 2^-38 A; rows below 2^-36 A become 0
  x         steps of 2^-24 where X is at 2^14 at least: 2^-39 X
so 2^-27 sum g |x| + n (2^-36 + 2^-38 + 2^-39) A X more. No term is taken over experts."""
import numpy as np
import pytest

from tests import _train_ref as ref
from tests.test_gpu_router_train import U, gpu, inputs, routed, rule, run_grad  # noqa: F401

pytestmark = pytest.mark.gpu


def check_dW(x, a, dW):
    a, x = a.astype(np.float64), x.astype(np.float64)
    n, ne = a.shape
    on = np.any(a != 0, axis=1)
    ab, xb = np.abs(a), np.abs(x)
    g = np.maximum.reduceat(ab, np.arange(0, n, 8), axis=0)[np.arange(n) // 8]
    A, X = ab.max(axis=0)[:, None], (xb * on[:, None]).max(axis=0)[None]
    tol = ((n + 16) * U + 3 * 2.0 ** -22) * (ab[on].T @ xb[on]) + 2.0 ** -27 * (g[on].T @ xb[on]) + n * (2.0 ** -36 + 2.0 ** -38 + 2.0 ** -39) * A * X + 1e-40
    err = np.abs(dW - a[on].T @ x[on])
    assert np.all(err <= tol), ((err / tol).max(), np.unique(np.nonzero(err > tol)[0])[:20])


@pytest.mark.parametrize("n,ne,E", [(1, 20, 1024), (8, 64, 2048), (40, 64, 1024), (300, 130, 2048), (700, 256, 7168), (3001, 100, 4096)])
def test_experts_of_every_size(ctx, rule, n, ne, E):  # noqa: F811
    """columns of dz over 2^110: each expert's row of dW is as good as if it were alone"""
    rule(2)
    print("experts n %d ne %d E %d" % (n, ne, E), flush=True)
    W, x, z, sel, dw, dz = inputs(n, ne, 2, E, n + ne)
    rng = np.random.default_rng(n)
    dz = (dz * np.exp2(rng.integers(-90, 21, (1, ne)))).astype(np.float32)
    dl, dW, dx = run_grad(ctx, W, x, z, sel, None, dz)
    assert np.array_equal(dl, dz)
    check_dW(x, dz, dW)


def test_rows_and_experts_of_every_size(ctx, rule):  # noqa: F811
    """an expert's gradients over 2^24 from one group of 8 rows to the next, and a column of dz with one entry only"""
    rule(2)
    W, x, z, sel, dw, dz = inputs(520, 64, 2, 1024, 5)
    rng = np.random.default_rng(6)
    dz = (dz * np.exp2(rng.integers(-24, 1, (65, 64))).repeat(8, axis=0) * np.exp2(rng.integers(-40, 1, (1, 64)))).astype(np.float32)
    dz[:, 9] = 0
    dz[300, 9] = 3e-20
    dl, dW, dx = run_grad(ctx, W, x, z, sel, None, dz)
    check_dW(x, dz, dW)


@pytest.mark.parametrize("n,ne,E,masked", [(4096, 256, 1024, False), (4096, 256, 1024, True), (1001, 64, 2048, True)])
def test_experts_without_picks_learn_from_the_balance_loss(ctx, rule, n, ne, E, masked):  # noqa: F811
    """weights' gradients of order 1 beside the balance loss's own with alpha 1e-4, experts whose logits lie 3 to 20 lower (no row picks
    them; their entries are down to 2^-50 of the row's largest), rows of positive x, so that such an expert's terms, all of one sign, add
    up; masked: rows without a loss on their weights"""
    rng, z, sel = routed(n, ne, 8, 3)
    low = {3: 3, 10: 6, 20: 9, 33: 12, 40: 16, 63: 20}
    for e, d in low.items():
        z[:, e] = 0.3 * z[:, e] - d - 4
    sel = np.argsort(-z, axis=1, kind="stable")[:, :8].astype(np.int32)
    assert not np.any(np.isin(sel, list(low)))
    rule(8)
    W = (0.02 * rng.standard_normal((ne, E))).astype(np.float32)
    x = np.abs(rng.standard_normal((n, E))).astype(np.float32)
    dw = rng.standard_normal((n, 8)).astype(np.float32)
    if masked:
        dw[rng.random(n) < 0.5] = 0
    counts, _ = ctx.balance_loss(gpu(z), gpu(sel), 1e-4)
    bal = ctx.balance_loss_grad(gpu(z), counts, 8, 1e-4).cpu().numpy()
    dl, dW, dx = run_grad(ctx, W, x, z, sel, dw, bal)
    want, mag = ref.route_dz(z, sel, dw, bal, 2.5)
    assert np.all(np.abs(dl - want) <= 60 * U * mag + 1e-44)
    assert np.all(dl[:, list(low)] < 0) and np.abs(dl[:, 63]).max() < 2.0 ** -40 * np.abs(dl).max()
    check_dW(x, dl, dW)


def test_rows_without_a_gradient_cost_nothing(ctx, rule):  # noqa: F811
    """padding: what x holds in a row of zero gradients leaves the others' bits as they are, unless it is not finite, which is NaN as in
    the product itself, in its own column"""
    rule(2)
    W, x, z, sel, dw, dz = inputs(90, 48, 2, 1024, 7)
    pad = np.r_[0:5, 30:47, 80:90]
    dz[pad] = 0
    zero = x.copy(); zero[pad] = 0
    clean = run_grad(ctx, W, zero, z, sel, None, dz)
    big = x.copy(); big[pad] = 1e30; big[31] = -3e38
    got = run_grad(ctx, W, big, z, sel, None, dz)
    assert np.array_equal(got[1].view(np.uint32), clean[1].view(np.uint32)) and np.array_equal(got[2], clean[2])
    check_dW(x, dz, got[1])
    big[40, 17] = np.nan; big[85, 600] = np.inf
    got = run_grad(ctx, W, big, z, sel, None, dz)
    c = np.delete(np.arange(1024), [17, 600])
    assert np.all(np.isnan(got[1][:, [17, 600]])) and np.array_equal(got[1][:, c].view(np.uint32), clean[1][:, c].view(np.uint32))


def test_gradients_at_the_ends_of_the_range(ctx, rule):  # noqa: F811
    """experts near the smallest normal number and near the largest, and one of non-finite entries only: each row for itself"""
    rule(2)
    W, x, z, sel, dw, dz = inputs(64, 32, 2, 1024, 8)
    dz = (dz * 1e6).astype(np.float32)
    dz[:, 0] *= np.float32(2.0 ** -118)
    dz[:, 1] *= np.float32(2.0 ** 100)
    dz[:, 2] = 0; dz[9, 2] = np.nan
    dl, dW, dx = run_grad(ctx, W, x, z, sel, None, dz)
    e = np.arange(32) != 2
    assert np.all(np.isnan(dW[2])) and np.all(np.isfinite(dW[e]))
    check_dW(x, dz[:, e], dW[e])
