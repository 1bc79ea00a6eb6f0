"""GPU: the 16-bit products' backward pass, the combine's and the dispatch where there are no rows, no slots or picks without one."""
import pytest
import torch

from loki_amd import FL_BF16, FL_EINVAL, LokiError, lib

pytestmark = pytest.mark.gpu
B, I = torch.bfloat16, torch.int32


def zeros(*shape, dtype=B):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def test_no_rows_in_the_backward_pass(ctx):
    """results of no elements have no address: such a call is one like any other, as the forward pass has it"""
    R, K, ne = 24, 40, 3
    dz, x, W, W3, off, perm = zeros(0, R), zeros(0, K), zeros(R, K), zeros(ne, R, K), zeros(ne + 1, dtype=I), zeros(0, dtype=I)
    for kw in (dict(), dict(offsets=off)):
        out, none, nb = ctx.act_grad(dz, dz, "silu", **kw)
        assert out.shape == (0, R) and none is None and nb is None
        out, out2, nb = ctx.act_grad(dz, dz, "gelu", z2=dz, **kw)
        assert out.shape == out2.shape == (0, R) and nb is None
    dx, none = ctx.matmul_grad(dz, x, W, need_dW=False)
    assert dx.shape == (0, K) and none is None
    dx, none, none2 = ctx.matmul_grad(dz, x, W, dz2=dz, up=W, need_dW=False)
    assert dx.shape == (0, K) and none is None and none2 is None
    for kw in (dict(), dict(perm=perm, topk=2)):
        dx, none = ctx.expert_matmul_grad(dz, x, W3, off, need_dW=False, **kw)
        assert dx.shape == (0, K) and none is None
    dx, dW = ctx.expert_matmul_grad(dz, x, W3, off, perm=perm, topk=2)
    ctx.sync()
    assert dx.shape == (0, K) and not bool(dW.any())


def test_no_rows_or_slots_in_the_combines_gradient(ctx):
    o, none = zeros(4, 40), zeros(0, dtype=I)
    do, dw = ctx.combine_grad(zeros(0, 40), o, none, topk=2, need_do=False)
    assert do is None and dw.shape == (0, 2)
    do, dw = ctx.combine_grad(zeros(0, 40), o, none, topk=2, need_dw=False)
    assert do.shape == (4, 40) and dw is None
    do, dw = ctx.combine_grad(zeros(2, 40), zeros(0, 40), zeros(4, dtype=I), topk=2, need_dw=False)   # rows, but no slot
    assert do.shape == (0, 40) and dw is None
    do, dw = ctx.combine_grad(zeros(2, 40), zeros(0, 40), zeros(4, dtype=I), topk=2)
    ctx.sync()
    assert do.shape == (0, 40) and not bool(dw.any())


def test_nothing_to_compute_is_still_refused(ctx):
    """where there are rows; and without rows sizes and types are checked all the same"""
    dz, x, W = zeros(4, 24), zeros(4, 40), zeros(24, 40)
    with pytest.raises(LokiError, match="nothing to compute"):
        ctx.matmul_grad(dz, x, W, need_dx=False, need_dW=False)
    with pytest.raises(LokiError, match="nothing to compute"):
        ctx.combine_grad(zeros(2, 40), zeros(4, 40), zeros(4, dtype=I), topk=2, need_do=False, need_dw=False)
    L, c = lib(), ctx.ctx
    assert L.fl_act_grad_dev(c, FL_BF16, 1, dz.data_ptr(), dz.data_ptr(), None, 4, 24, 1, None, None, None, None, 0) == FL_EINVAL
    assert L.fl_act_grad_dev(c, FL_BF16, 9, None, None, None, 0, 24, 1, None, None, None, None, 0) == FL_EINVAL
    assert L.fl_act_grad_dev(c, FL_BF16, 1, None, None, None, 0, 12, 1, None, None, None, None, 0) == FL_EINVAL
    assert L.fl_matmul_grad_dev(c, 0, None, None, None, None, None, 0, 24, 40, 1, None, None, 1, 0, None, None, None, FL_BF16, 0) == FL_EINVAL
    assert L.fl_combine_grad_dev(c, FL_BF16, None, None, None, None, None, 0, 2, 1, 4, 12, None, None) == FL_EINVAL
