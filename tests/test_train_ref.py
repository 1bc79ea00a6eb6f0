"""CPU: the 64-bit references of the balance loss and of the router's backward pass against central differences of the values
they are gradients of, and what the entry points answer without a context."""
import ctypes

import numpy as np
import pytest

import loki_amd
from tests import _train_ref as ref


def case(n, ne, topk, seed, spread=1.5):
    rng = np.random.default_rng(seed)
    z = spread * rng.standard_normal((n, ne))
    sel = np.argsort(-z, axis=1, kind="stable")[:, :topk].astype(np.int32)
    return rng, z, sel


@pytest.mark.parametrize("n,ne,topk,seq", [(1, 8, 2, [0, 1]), (9, 16, 4, [0, 4, 4, 9]), (7, 5, 1, [1, 6])])
def test_balance_gradient_is_the_losses_derivative(n, ne, topk, seq):
    rng, z, sel = case(n, ne, topk, 3 + n)
    gloss = rng.standard_normal(len(seq) - 1)
    _, _, dz, _ = ref.balance(z, sel, 0.3, seq, gloss)
    h = 1e-5
    for t in range(n):
        for e in range(ne):
            v = []
            for sgn in (1, -1):
                y = z.copy(); y[t, e] += sgn * h
                v.append(float(ref.balance(y, sel, 0.3, seq)[1] @ gloss))
            # the difference's own error: h^2 / 6 of a third derivative of order 1, and eps / h
            assert abs((v[0] - v[1]) / (2 * h) - dz[t, e]) < 1e-8, (t, e)


@pytest.mark.parametrize("shift", [0.0, -18.0], ids=["normalised", "clamped"])
def test_route_gradient_is_the_weights_derivative(shift):
    rng, z, sel = case(6, 10, 3, 11)
    z = z + shift   # -18: the picked sigmoids' sum stays below 2^-14
    dw = rng.standard_normal(sel.shape)
    assert np.all((np.take_along_axis(ref.sigmoid(z), sel, 1).sum(1) < ref.CLAMP) == (shift < 0))
    dz, _ = ref.route_dz(z, sel, dw, None, 2.5)
    h = 1e-6
    for t in range(z.shape[0]):
        for e in range(z.shape[1]):
            v = []
            for sgn in (1, -1):
                y = z.copy(); y[t, e] += sgn * h
                v.append(float((ref.weights(y, sel, 2.5) * dw).sum()))
            assert abs((v[0] - v[1]) / (2 * h) - dz[t, e]) < 1e-6 * max(1.0, abs(dz[t, e])), (t, e)


def test_shares_of_tiny_rows():
    p = ref.shares(np.array([[-200.0, -201.0, -np.inf], [-np.inf] * 3, [50.0, 0.0, -np.inf]]))
    assert np.allclose(p[0], [1 / (1 + np.exp(-1)), 1 / (1 + np.exp(1)), 0], rtol=1e-12) and np.all(p[1] == 0)
    assert np.allclose(p[2], [2 / 3, 1 / 3, 0], rtol=1e-12)


def test_entry_points_without_a_context():
    L = loki_amd.lib()
    assert L.fl_balance_loss_dev(None, None, None, None, 0, 1, 8, 2, 1.0, None, None) == loki_amd.FL_EINVAL
    assert L.fl_balance_loss_grad_dev(None, None, None, None, None, 0, 1, 8, 2, 1.0, 0, None) == loki_amd.FL_EINVAL
    assert L.fl_route_grad_dev(None, None, None, None, None, None, None, 0, 8, 1024, None, None, 0, None) == loki_amd.FL_EINVAL


def test_wrappers_refuse_other_tensors():
    import torch
    need = loki_amd.Context._need
    with pytest.raises(loki_amd.LokiError, match="contiguous"):
        need(None, "x", (torch.zeros(4, 3), torch.float32, (4, 3)))          # not on the GPU
    with pytest.raises(loki_amd.LokiError, match="float32"):
        need(None, "x", (torch.zeros(4, 3, dtype=torch.float64), torch.float32, (4, 3)))
    need(None, "x", (None, torch.float32, (4, 3)))
