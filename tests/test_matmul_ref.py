"""CPU: the 64-bit references of the 16-bit products' gradients against central differences, and what the entry points and wrappers
refuse without a GPU."""
import pytest
import torch

import loki_amd
from tests import _mm_ref as ref

F8 = torch.float64


def rnd(seed, *shape):
    return torch.randn(shape, dtype=F8, generator=torch.Generator().manual_seed(seed))


def difference(f, v, i, h=1e-5):
    p, m = v.clone(), v.clone()
    p.view(-1)[i] += h
    m.view(-1)[i] -= h
    return float((f(p) - f(m)) / (2 * h))


@pytest.mark.parametrize("kind", [None, "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_layer_gradients_are_differences(kind, gated):
    """sum g * (act(z) (* z2)) over two experts' slots, to x, W and W2"""
    off, g = [1, 3, 6], rnd(1, 6, 4)
    x, W, W2 = rnd(2, 6, 5), rnd(3, 2, 4, 5), rnd(4, 2, 4, 5)
    g[0] = 0.0   # slot 0 belongs to no expert

    def value(x, W, W2):
        z, z2 = ref.products(x, W, off)[0], ref.products(x, W2, off)[0]
        y = ref.act(z, kind) * (z2 if gated else 1.0)
        return (g[1:] * y[1:]).sum()

    z, z2 = ref.products(x, W, off)[0], ref.products(x, W2, off)[0]
    dz, dz2 = g * ref.slope(z, kind) * (z2 if gated else 1.0), g * ref.act(z, kind)
    dx, _, dW, _ = ref.grads(dz, x, W, off)
    if gated:
        dxb, _, dW2, _ = ref.grads(dz2, x, W2, off)
        dx = dx + dxb
    for i in range(5, x.numel()):
        assert abs(difference(lambda v: value(v, W, W2), x, i) - float(dx.view(-1)[i])) < 1e-7
    for i in range(W.numel()):
        assert abs(difference(lambda v: value(x, v, W2), W, i) - float(dW.view(-1)[i])) < 1e-7
        if gated:
            assert abs(difference(lambda v: value(x, W, v), W2, i) - float(dW2.view(-1)[i])) < 1e-7


def test_combine_gradients_are_differences():
    sel = torch.tensor([[0, 1], [2, -1], [1, 1]], dtype=torch.int32)
    off, perm, inv = ref.order(sel, 3)
    o, w, dy = rnd(5, 6, 4), rnd(6, 3, 2), rnd(7, 3, 4)
    do, dw, _ = ref.combine_grad(dy, o, inv, w, sel, 3)
    for i in range(5 * 4):
        assert abs(difference(lambda v: (ref.combine(v, inv, w, sel, 3, None)[0] * dy).sum(), o, i) - float(do.view(-1)[i])) < 1e-8
    for i in range(w.numel()):
        assert abs(difference(lambda v: (ref.combine(o, inv, v, sel, 3, None)[0] * dy).sum(), w, i) - float(dw.view(-1)[i])) < 1e-8
    assert torch.isnan(do[5]).all() and float(dw[1, 1]) == 0


def test_order_is_a_dispatch():
    sel = torch.tensor([[3, 0], [-1, 3], [0, 9]], dtype=torch.int32)
    off, perm, inv = ref.order(sel, 4)
    assert off.tolist() == [0, 2, 2, 2, 4] and perm.tolist() == [1, 4, 0, 3, -1, -1] and inv.tolist() == [2, 0, -1, 3, 1, -1]


def test_entry_points_without_a_context():
    L, E = loki_amd.lib(), loki_amd.FL_EINVAL
    assert L.fl_matmul_dev(None, 18, 0, None, None, None, None, None, 0, 8, 8, 1, None, None, 1, 0, None, 18, None, None) == E
    assert L.fl_act_grad_dev(None, 18, 0, None, None, None, 0, 8, 1, None, None, None, None, 0) == E
    assert L.fl_matmul_grad_dev(None, 18, None, None, None, None, None, 0, 8, 8, 1, None, None, 1, 0, None, None, None, 18, 0) == E
    assert L.fl_combine_dev(None, 18, None, None, None, None, None, 0, 1, 1, 0, 8, None, 18) == E
    assert L.fl_combine_grad_dev(None, 18, None, None, None, None, None, 0, 1, 1, 0, 8, None, None) == E


class Bare(loki_amd.Context):
    """a context's checks without a GPU"""
    def __init__(self):
        self.torch, self.ctx, self._device = torch, None, 0


def test_wrappers_refuse():
    c, E = Bare(), loki_amd.LokiError
    x, W, W3 = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(2, 8, 16, dtype=torch.bfloat16)
    off = torch.tensor([0, 1, 4], dtype=torch.int32)
    with pytest.raises(E, match="bfloat16 or float16"):
        c.matmul(x.float(), W.float())
    with pytest.raises(E, match="bfloat16 or float16"):
        c.matmul(x.double(), W.double())
    with pytest.raises(E, match=r"\[n_exp\]"):
        c.expert_matmul(x, W, off)
    with pytest.raises(E, match="contiguous"):
        c.matmul(x, W)                                  # not on the GPU
    with pytest.raises(E, match="contiguous"):
        c.expert_matmul(x, W3, off)
    with pytest.raises(E, match="silu"):
        c.act_grad(x, x, "relu")
    with pytest.raises(E, match="contiguous"):
        c.act_grad(x, x, "silu")
    with pytest.raises(E, match="topk"):
        c.combine(x, torch.zeros(8, dtype=torch.int32))
    with pytest.raises(E, match="bfloat16 or float16"):
        c.combine(x.float(), torch.zeros(4, dtype=torch.int32), topk=2)
    with pytest.raises(E, match="contiguous"):
        c.combine_grad(x, x, torch.zeros(4, dtype=torch.int32), topk=1)
