"""GPU: the dispatch of picks that no expert has (-1, or n_exp and above), and of no rows: in one workgroup (up to 4096 pairs) and in several."""
import pytest
import torch

from loki_amd import lib
from tests import _mm_ref as ref

pytestmark = pytest.mark.gpu


def dropped(n, topk, ne, seed):
    g = torch.Generator().manual_seed(seed)
    sel = torch.topk(torch.randn((n, ne), generator=g), topk, dim=1).indices.to(torch.int32)
    sel[torch.rand(sel.shape, generator=g) < 0.3] = -1
    sel[torch.rand(sel.shape, generator=g) < 0.1] = ne
    return sel


@pytest.mark.parametrize("n,topk,ne", [(1, 4, 8), (5, 8, 64), (512, 8, 256), (513, 8, 9), (3000, 3, 200)])
def test_a_pair_without_a_slot_is_told_by_inv(ctx, n, topk, ne):
    sel = dropped(n, topk, ne, n)
    off, perm, inv = ref.order(sel, ne)
    P, full = n * topk, lambda k: torch.full((k,), 2, dtype=torch.int32, device="cuda")   # noqa: E731
    counts, offsets, gp, gi, act, nact, gs = full(ne), full(ne + 1), full(P), full(P), full(ne), full(1), sel.cuda()
    ctx.check(lib().fl_dispatch_dev(ctx.ctx, gs.data_ptr(), n, topk, ne, *[t.data_ptr() for t in (counts, offsets, gp, gi, act, nact)]))
    ctx.sync()
    used = int(off[-1])
    assert torch.equal(offsets.cpu(), off) and torch.equal(gp.cpu()[:used], perm[:used]) and bool((gp[used:] == 2).all())
    assert torch.equal(gi.cpu(), inv)


@pytest.mark.parametrize("n", [7, 700])
def test_combine_by_inv_alone(ctx, n):
    """a row's sum over its slots needs no picks beside the dispatch's inv"""
    topk, ne, E = 8, 16, 24
    sel = dropped(n, topk, ne, n).cuda()
    _, _, _, inv, _, _ = ctx.dispatch(sel, n_exp=ne)
    o = torch.randint(-9, 10, (n * topk, E), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    a, b = ctx.combine(o, inv, topk=topk, dtype=torch.float32), ctx.combine(o, inv, sel=sel, n_exp=ne, dtype=torch.float32)
    ctx.sync()
    s = sel.cpu()
    want = torch.where(((s >= 0) & (s < ne))[:, :, None], o.cpu().float()[inv.cpu().view(n, topk).long().clamp(0, n * topk - 1)], 0.0).sum(1)
    assert torch.equal(b.cpu(), want) and torch.equal(a, b)


def test_dispatch_of_no_rows(ctx):
    counts, offsets, perm, inv, _, nact = ctx.dispatch(torch.zeros((0, 8), dtype=torch.int32, device="cuda"), n_exp=16)
    ctx.sync()
    assert not bool(counts.any()) and not bool(offsets.any()) and int(nact) == 0 and perm.numel() == inv.numel() == 0


def test_no_rows_through_the_layer(ctx):
    """route, dispatch, the experts, the combine and all of it backwards, for a batch without rows: no results but zeros for the matrices"""
    ne, k, E, H, T, F = 16, 4, 1024, 24, torch.bfloat16, torch.float32
    z = lambda *s, dtype=T: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    x, x32, Wr, Wg, Wd = z(0, E), z(0, E, dtype=F), z(ne, E, dtype=F), z(ne, H, E), z(ne, E, H)
    ctx.set_routing(1, 1, k, 2.5)
    try:
        logits, _, sel, w = ctx.route(Wr, z(ne, dtype=F), x32, topk=k)
        _, off, perm, inv, _, _ = ctx.dispatch(sel, n_exp=ne)
        h, p, p2 = ctx.expert_matmul(x, Wg, off, up=Wg, act="silu", perm=perm, topk=k, keep=True)
        o = ctx.expert_matmul(h, Wd, off)
        y = ctx.combine(o, inv, w, sel=sel, n_exp=ne, residual=x)
        do, dw = ctx.combine_grad(y, o, inv, w, sel=sel, n_exp=ne)
        dh, dWd = ctx.expert_matmul_grad(do, h, Wd, off)
        dz, dz2, _ = ctx.act_grad(dh, p, "silu", z2=p2, offsets=off)
        dxs, dWg, dWu = ctx.expert_matmul_grad(dz, x, Wg, off, dz2=dz2, up=Wg, perm=perm, topk=k)
        dx = ctx.combine(dxs, inv, sel=sel, n_exp=ne, residual=y, dtype=F)
        dl, dWr, dxr = ctx.route_grad(Wr, x32, logits, sel, dw)
        ctx.sync()
    finally:
        ctx.set_routing()
    assert y.shape == dx.shape == dxr.shape == (0, E) and dw.shape == (0, k) and dl.shape == (0, ne) and dxs.shape == (0, E) and do.shape == (0, E)
    assert not any(bool(t.any()) for t in (dWd, dWg, dWu, dWr))
