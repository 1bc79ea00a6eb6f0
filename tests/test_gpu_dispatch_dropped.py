"""GPU: the dispatch of picks that no expert has (-1, or n_exp and above): in one workgroup (up to 4096 pairs) and in several."""
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
