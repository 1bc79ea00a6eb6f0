"""GPU: the 16-bit products at sizes that reach every kernel, tile and split (_mm_cases.py; the rules' CPU test says that they do), in whole numbers.

x, W, dz are -1, 0 or 1, biases and residuals small whole numbers: every product, partial sum and result before its last rounding is a whole
number below 2^24 whatever the order, so float32 results equal the definition's and 16-bit ones its nearest value, bit for bit: (16-bit
results of a sum split into parts as well.) A gated result is a product of two sums: below 2^24 as both are below 2^12 (K up to 7176 terms of
variance 4/9: 56 on average, 20 times that is 1130)."""
import pytest
import torch

import loki_amd
from loki_amd import FL_BF16, FL_ENOMEM, LokiError, lib
from tests import _mm_cases as cases
from tests import _mm_ref as ref

pytestmark = pytest.mark.gpu
B, F4 = torch.bfloat16, torch.float32


def whole(seed, *shape, dtype=B, most=1):
    return torch.randint(-most, most + 1, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def mm(a, b):
    """a b^T in float32 (exact); the operands' whole numbers in float32 too"""
    return a.float() @ b.float().t().contiguous()


def same(got, want):
    w = want.to(got.dtype)
    assert torch.equal(got, w), (int((got != w).sum()), (got != w).nonzero()[:3].tolist())


def dims(n, ne, first=3, after=5):
    c = cases.counts(n, ne)
    off = [first + sum(c[:e]) for e in range(ne + 1)]
    return off, torch.tensor(off, dtype=torch.int32, device="cuda"), off[-1] + after


def test_matmul_kernels_dense(ctx):
    for i, (n, R, K) in enumerate(cases.DENSE):
        print("n %d R %d K %d" % (n, R, K), flush=True)
        T = (B, torch.float16)[i % 2]
        x, W, W2, bias, res = whole(1, n, K, dtype=T), whole(2, R, K, dtype=T), whole(3, R, K, dtype=T), whole(4, R, dtype=F4, most=99), whole(5, n, R, dtype=T, most=99)
        z, z2 = mm(x, W), mm(x, W2)
        same(ctx.matmul(x, W, bias=bias, residual=res, dtype=F4), z + bias + res.float())
        same(ctx.matmul(x, W), z)
        y, kz, kz2 = ctx.matmul(x, W, up=W2, residual=res, dtype=F4, keep=True)
        same(y, z * z2 + res.float())
        same(kz, z)
        same(kz2, z2)
        dz, dz2 = whole(6, n, R, dtype=T), whole(7, n, R, dtype=T)
        dx, dW = ctx.matmul_grad(dz, x, W, dw_dtype=F4)
        same(dx, mm(dz, W.t()))
        same(dW, mm(dz.t(), x.t()))
        add, add2 = whole(8, R, K, dtype=F4, most=99), whole(9, R, K, dtype=F4, most=99)
        w, w2 = add.clone(), add2.clone()
        dx, dW, dW2 = ctx.matmul_grad(dz, x, W, dz2=dz2, up=W2, dW=w, dW2=w2)
        same(dx, mm(dz, W.t()) + mm(dz2, W2.t()))
        same(dW, add + mm(dz.t(), x.t()))
        same(dW2, add2 + mm(dz2.t(), x.t()))
        same(ctx.matmul_grad(dz, x, W, need_dx=False)[1], mm(dz.t(), x.t()))


@pytest.mark.parametrize("through", [False, True])
def test_matmul_kernels_experts(ctx, through):
    for i, (n, ne, R, K) in enumerate(cases.EXPERTS):
        print("n %d experts %d R %d K %d%s" % (n, ne, R, K, " through perm" if through else ""), flush=True)
        T = (torch.float16, B)[i % 2]
        off, offsets, slots = dims(n, ne)
        topk = 3 if through else 1
        x = whole(1, -(-slots // topk), K, dtype=T) if through else whole(1, slots, K, dtype=T)
        perm = torch.randperm(x.shape[0] * topk, generator=torch.Generator().manual_seed(2))[:slots].to(torch.int32).cuda() if through else None
        rows = x[perm.long() // topk] if through else x
        W, W2, bias, res = whole(3, ne, R, K, dtype=T), whole(4, ne, R, K, dtype=T), whole(5, ne, R, dtype=F4, most=99), whole(6, slots, R, dtype=T, most=99)
        dz, dz2 = whole(7, slots, R, dtype=T), whole(8, slots, R, dtype=T)
        z, z2 = torch.full((slots, R), 77.0, device="cuda"), torch.full((slots, R), 77.0, device="cuda")
        b, d, d2 = torch.zeros_like(z), torch.full((slots, K), 77.0, device="cuda"), torch.full((slots, K), 77.0, device="cuda")
        w, w2 = torch.zeros((ne, R, K), device="cuda"), torch.zeros((ne, R, K), device="cuda")
        for e in range(ne):
            s = slice(off[e], off[e + 1])
            if off[e] < off[e + 1]:
                z[s], z2[s], b[s], d[s] = mm(rows[s], W[e]), mm(rows[s], W2[e]), bias[e], mm(dz[s], W[e].t())
                d2[s] = d[s] + mm(dz2[s], W2[e].t())
                w[e], w2[e] = mm(dz[s].t(), rows[s].t()), mm(dz2[s].t(), rows[s].t())
        live = slice(off[0], off[-1])
        outside = torch.ones(slots, dtype=torch.bool, device="cuda")
        outside[live] = False
        kw = dict(perm=perm, topk=topk)

        def check(got, want):
            same(got[live], want[live])
            assert bool((got[outside] == 77.0).all())

        out = lambda cols, dtype=T: torch.full((slots, cols), 77.0, dtype=dtype, device="cuda")  # noqa: E731
        check(ctx.expert_matmul(x, W, offsets, bias=bias, residual=res, y=out(R, F4), **kw), z + b + res.float())
        check(ctx.expert_matmul(x, W, offsets, y=out(R), **kw), z)
        for got, want in zip(ctx.expert_matmul(x, W, offsets, up=W2, y=out(R, F4), z=out(R), z2=out(R), **kw), (z * z2, z, z2)):
            check(got, want)
        dx, dW = ctx.expert_matmul_grad(dz, x, W, offsets, dx=out(K), dw_dtype=F4, **kw)
        check(dx, d)
        same(dW, w)
        a, a2 = whole(9, ne, R, K, dtype=F4, most=99), whole(10, ne, R, K, dtype=F4, most=99)
        dx, dW, dW2 = ctx.expert_matmul_grad(dz, x, W, offsets, dz2=dz2, up=W2, dx=out(K), dW=a.clone(), dW2=a2.clone(), **kw)
        check(dx, d2)
        same(dW, a + w)
        same(dW2, a2 + w2)
        same(ctx.expert_matmul_grad(dz, x, W, offsets, need_dx=False, **kw)[1], w)
        torch.cuda.empty_cache()


def test_tiles_hold_nan_and_infinities_apart(ctx):
    """rows, experts and columns outside a tile are not touched: what is not finite in one expert stays there at every tile size"""
    for n, ne, R, K in ((2100, 5, 4104, 72), (4200, 5, 264, 520), (8500, 5, 1032, 2056)):
        off, offsets, slots = dims(n, ne)
        x, W, dz = whole(1, slots, K), whole(2, ne, R, K), whole(3, slots, R)
        clean = [ctx.expert_matmul(x, W, offsets)] + list(ctx.expert_matmul_grad(dz, x, W, offsets))
        x[off[2]:off[3]], dz[off[2]:off[3]], W[2] = float("inf"), float("nan"), float("nan")
        for t in (x, dz):
            t[:off[0]], t[off[-1]:] = float("nan"), float("nan")
        got = [ctx.expert_matmul(x, W, offsets)] + list(ctx.expert_matmul_grad(dz, x, W, offsets))
        ctx.sync()
        for i in (0, 1):
            for s in (slice(off[0], off[2]), slice(off[3], off[-1])):
                assert torch.equal(got[i][s], clean[i][s])
        for e in (0, 1, 3, 4):
            assert torch.equal(got[2][e], clean[2][e])


def test_offsets_past_32_bits(ctx):
    """rows, weights and results beyond 2^32 bytes and 2^32 values from their first"""
    n, R, K = (1 << 19) + 40, 8200, 8       # y: 8.6 GB
    x, W = whole(1, n, K), whole(2, R, K)
    y = ctx.matmul(x, W)
    s = slice(n - 300, n)
    same(y[s], mm(x[s], W))
    same(y[:300], mm(x[:300], W))
    dx, dW = ctx.matmul_grad(y, x, W, need_dW=False), None   # sums of 8200 terms below 2^24: at most 8 * 8200
    same(dx[0][s], mm(y[s], W.t()))
    t = ctx.matmul(y, W.t().contiguous(), dtype=F4)           # x: 8.6 GB
    same(t[s], mm(y[s], W.t()))
    del y, dx, dW, t
    torch.cuda.empty_cache()
    ne, R, K, n = 40, 8200, 8200, 90                             # W, dW: 5.4 GB
    W = torch.empty((ne, R, K), dtype=B, device="cuda")
    for e in range(ne):
        W[e] = whole(e, R, K)
    offsets = torch.tensor([min(e, 30) for e in range(ne)] + [n], dtype=torch.int32, device="cuda")
    x, dz = whole(100, n, K), whole(101, n, R)
    y = ctx.expert_matmul(x, W, offsets, dtype=F4)
    dx, dW = ctx.expert_matmul_grad(dz, x, W, offsets)
    a = slice(30, n)
    same(y[a], mm(x[a], W[-1]))
    same(dx[a], mm(dz[a], W[-1].t()))
    same(dW[-1], mm(dz[a].t(), x[a].t()))
    same(dW[29], mm(dz[29:30].t(), x[29:30].t()))
    assert not bool(dW[30:-1].any())
    del W, dW
    torch.cuda.empty_cache()
    pairs, E = (1 << 19) + 24, 8200                               # o: 8.6 GB
    o = torch.empty((pairs, E), dtype=B, device="cuda")
    o[:300], o[-300:] = whole(1, 300, E), whole(2, 300, E)
    inv = torch.arange(pairs - 1, -1, -1, dtype=torch.int32, device="cuda").view(-1, 8)
    y = ctx.combine(o, inv, topk=8, dtype=F4)
    same(y[:30], o[inv[:30].long()].float().sum(1))
    same(y[-30:], o[inv[-30:].long()].float().sum(1))


def test_equal_calls_equal_bits(ctx):
    """sums have one order: the same call gives the same bits, whatever ran before and whichever workgroup took a tile"""
    g = torch.Generator(device="cuda").manual_seed(1)
    for n, ne, R, K in ((8500, 5, 1032, 2056), (1400, 5, 520, 7176), (70, 1, 4104, 7176), (4200, 5, 72, 72)):
        off, offsets, slots = dims(n, ne)
        r = lambda *s: torch.randn(s, generator=g, device="cuda").to(B)  # noqa: E731
        x, W, dz, bias = r(slots, K), r(ne, R, K), r(slots, R), r(ne, R).float()
        def run():
            y = torch.zeros((slots, R), dtype=B, device="cuda")
            dx = torch.zeros((slots, K), dtype=B, device="cuda")
            ctx.expert_matmul(x, W, offsets, bias=bias, act="gelu", y=y)
            _, dW = ctx.expert_matmul_grad(dz, x, W, offsets, dx=dx)
            db = ctx.act_grad(dz, None, None, bias=True, offsets=offsets, dz=torch.zeros_like(dz))[2]
            return y, dx, dW, db
        first = run()
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_two_contexts_at_once(ctx):
    """two contexts on streams of their own, their tiles' counters and workspaces apart"""
    n, R, K = 1400, 1032, 7176
    cs = [(loki_amd.Context(), torch.cuda.Stream()) for _ in range(2)]
    data = [(whole(i, n, K), whole(i + 5, R, K), whole(i + 9, n, R)) for i in range(2)]
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(3):
        for i, (c, s) in enumerate(cs):
            with torch.cuda.stream(s):
                x, W, dz = data[i]
                c.check(lib().fl_set_stream(c.ctx, s.cuda_stream))
                out[i].append((c.matmul(x, W), *c.matmul_grad(dz, x, W)))
    torch.cuda.synchronize()
    for i, (x, W, dz) in enumerate(data):
        want = mm(x, W), mm(dz, W.t()), mm(dz.t(), x.t())
        for got in out[i]:
            for a, b in zip(got, want):
                same(a, b)
    for c, _ in cs:
        c.close()


def test_split_sums_captured(ctx):
    """sums in parts need the context's workspace: a capture on a fresh context is refused and goes on, one after an eager call runs; replays with
    eager calls between them give the eager result every time (the tiles' counters are back at 0 after each)"""
    n, R, K = 70, 4104, 7176
    c, s = loki_amd.Context(), torch.cuda.Stream()
    x, W, dz = whole(1, n, K), whole(2, R, K), whole(3, n, R)
    y, dx = torch.zeros((n, R), device="cuda"), torch.zeros((n, K), dtype=B, device="cuda")
    torch.cuda.synchronize()
    c.check(lib().fl_set_stream(c.ctx, s.cuda_stream))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        rc = lib().fl_matmul_dev(c.ctx, FL_BF16, 0, x.data_ptr(), W.data_ptr(), None, None, None, n, R, K, 1, None, None, 1, 0, y.data_ptr(), 16, None, None)
        y.add_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    assert rc == FL_ENOMEM and bool((y == 1.0).all())

    def step():
        c.matmul(x, W, y=y, dtype=F4)
        c.matmul_grad(dz, x, W, dx=dx, need_dW=False)

    with torch.cuda.stream(s):
        step()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
    for i in range(4):
        x.copy_(whole(20 + i, n, K))
        dz.copy_(whole(30 + i, n, R))
        y.zero_()
        dx.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(y, mm(x, W))
        same(dx, mm(dz, W.t()))
        with torch.cuda.stream(s):
            c.matmul(dz, W.t().contiguous())
        torch.cuda.synchronize()
    c.close()


def test_offsets_that_are_none(ctx):
    """offsets outside 0 .. n or out of order: nothing outside the buffers is read or written, slots of no expert stay"""
    n, R, K = 600, 264, 72
    x, W, dz = whole(1, n, K), whole(2, 4, R, K), whole(3, n, R)
    for bad in ([-5, 10, 20, 30, 40], [0, 100, 50, 700, 650], [2 ** 31 - 1, 3, -2 ** 31, 9, 2 ** 31 - 1], [40, 30, 20, 10, 0]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        y = torch.full((n, R), 77.0, dtype=B, device="cuda")
        dx = torch.full((n, K), 77.0, dtype=B, device="cuda")
        ctx.expert_matmul(x, W, offsets, y=y)
        _, dW = ctx.expert_matmul_grad(dz, x, W, offsets, dx=dx)
        ctx.sync()
        used = torch.zeros(n, dtype=torch.bool, device="cuda")
        for a, b in ref.spans(offsets.cpu(), n, 4):
            used[a:b] = True
        assert bool((y[~used] == 77.0).all()) and bool((dx[~used] == 77.0).all()) and bool(torch.isfinite(dW).all())


def test_wrapper_refusals(ctx):
    x, W = whole(1, 4, 16), whole(2, 24, 16)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    W3, dz = whole(3, 2, 24, 16), whole(4, 4, 24)
    for call in (lambda: ctx.matmul(x.float(), W), lambda: ctx.matmul(x, W.half()), lambda: ctx.matmul(x, W[:, :8]), lambda: ctx.matmul(x.cpu(), W), lambda: ctx.matmul(x, W, act="relu"),
                 lambda: ctx.matmul(x, W, residual=dz.float()), lambda: ctx.matmul(x, W, bias=whole(5, 24)), lambda: ctx.matmul(x, W, y=whole(6, 5, 24)),
                 lambda: ctx.matmul(x, W, up=W, bias=whole(5, 24, dtype=F4)), lambda: ctx.matmul(x.t().contiguous().t(), W), lambda: ctx.expert_matmul(x, W, off),
                 lambda: ctx.expert_matmul(x, W3, off[:2]), lambda: ctx.expert_matmul(x, W3, off.long()), lambda: ctx.expert_matmul(x, W3, off, perm=off.long()),
                 lambda: ctx.matmul(x, W, dtype=torch.float64), lambda: ctx.matmul_grad(dz[:3], x, W), lambda: ctx.matmul_grad(dz, x, W, dw_dtype=torch.float16),
                 lambda: ctx.matmul_grad(dz, x, W, need_dx=False, need_dW=False), lambda: ctx.act_grad(dz, None, "silu"), lambda: ctx.combine(x.float(), off, topk=1),
                 lambda: ctx.combine(x, off, topk=2), lambda: ctx.combine(x, off), lambda: ctx.combine(x, off[:2].contiguous(), topk=2, residual=x)):
        with pytest.raises(LokiError):
            call()
    ctx.sync()
    assert torch.equal(ctx.matmul(x, W), mm(x, W).to(B))


def test_entry_refusals(ctx):
    """a bias inside a result, picks beyond 2^28 pairs; a gradient whose matrices' parts do not fit the workspace under capture writes nothing"""
    t = torch.zeros(1 << 16, dtype=B, device="cuda")
    p = t.data_ptr()
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda").data_ptr()
    assert lib().fl_matmul_dev(ctx.ctx, FL_BF16, 0, p, p + 8192, None, p + 16384, None, 4, 16, 16, 1, None, None, 1, 0, p + 16384, FL_BF16, None, None) == loki_amd.FL_EINVAL
    assert lib().fl_matmul_dev(ctx.ctx, FL_BF16, 0, p, p + 8192, None, None, None, 4, 16, 8, 1, off, off, 8, (1 << 25) + 1, p + 16384, FL_BF16, None, None) == loki_amd.FL_ERANGE
    c, s = loki_amd.Context(), torch.cuda.Stream()
    n, R, K = 8500, 72, 72
    dz, x, W = whole(1, n, R), whole(2, n, K), whole(3, R, K)
    dx, dW = torch.full((n, K), 77.0, dtype=B, device="cuda"), torch.full((R, K), 77.0, dtype=B, device="cuda")
    torch.cuda.synchronize()
    c.check(lib().fl_set_stream(c.ctx, s.cuda_stream))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        rc = lib().fl_matmul_grad_dev(c.ctx, FL_BF16, dz.data_ptr(), None, x.data_ptr(), W.data_ptr(), None, n, R, K, 1, None, None, 1, 0, dx.data_ptr(), dW.data_ptr(), None, FL_BF16, 0)
        dW.add_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    assert rc == FL_ENOMEM and bool((dx == 77.0).all()) and bool((dW == 78.0).all())
    c.close()


@pytest.mark.parametrize("n,ne,topk", [(1, 8, 2), (70, 16, 4), (900, 200, 6)])
def test_layer_with_dropped_picks(ctx, n, ne, topk):
    """the layer forward and backward on dispatch()'s tables where picks were dropped (-1): two linear products, so that everything stays a whole
    number below 2^11 where it is float16 and below 2^24 where it is float32"""
    T, E, H = torch.float16, 24, 16
    g = torch.Generator().manual_seed(n)
    sel = torch.topk(torch.randn((n, ne), generator=g), topk, dim=1).indices.to(torch.int32)
    sel[torch.rand(sel.shape, generator=g) < 0.3] = -1
    sel[-1] = -1
    sel = sel.cuda()
    x, Wg, Wd, w, dy, res = whole(1, n, E, dtype=T), whole(2, ne, H, E, dtype=T), whole(3, ne, E, H, dtype=T), whole(4, n, topk, dtype=F4, most=2), whole(5, n, E, dtype=T), whole(6, n, E, dtype=T)
    _, off, perm, inv, _, _ = ctx.dispatch(sel, n_exp=ne)
    h = ctx.expert_matmul(x, Wg, off, perm=perm, topk=topk)
    o = ctx.expert_matmul(h, Wd, off)
    y = ctx.combine(o, inv, w, sel=sel, n_exp=ne, residual=res, dtype=F4)
    do, dw = ctx.combine_grad(dy, o, inv, w, sel=sel, n_exp=ne)
    dh, dWd = ctx.expert_matmul_grad(do, h, Wd, off, dw_dtype=F4)
    dxs, dWg = ctx.expert_matmul_grad(dh, x, Wg, off, perm=perm, topk=topk, dw_dtype=F4)
    dx = ctx.combine(dxs, inv, sel=sel, n_exp=ne, topk=topk, dtype=F4)
    ctx.sync()
    a = [t.double().cpu().requires_grad_(True) for t in (x, Wg, Wd, w)]
    want = res.double().cpu()
    for k in range(topk):
        e = sel[:, k].cpu().long()
        z = torch.einsum("te,the->th", a[0], a[1][e.clamp(min=0)])
        want = want + torch.einsum("th,teh->te", z, a[2][e.clamp(min=0)]) * (a[3][:, k] * (e >= 0))[:, None]
    (want * dy.double().cpu()).sum().backward()
    for got, t in ((y, want.detach()), (dx, a[0].grad), (dWg, a[1].grad), (dWd, a[2].grad), (dw, a[3].grad)):
        assert got.dtype is F4 and torch.equal(got.cpu(), t.float())


def test_combine_of_more_rows_than_workgroups(ctx):
    """a launch has 2^22 workgroups at most: more rows take more than one"""
    n = (1 << 22) + 9
    for E, P in ((2048, 50), (8, n)):
        o, w = whole(1, P, E), whole(2, n, 1, dtype=F4, most=3)
        inv = torch.randint(0, P, (n,), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda", dtype=torch.int32) if P < n else torch.arange(n, dtype=torch.int32, device="cuda").flip(0).contiguous()
        y = ctx.combine(o, inv, w)
        for s in (slice(0, 20), slice(n - 30, n)):
            same(y[s], o[inv[s].long()].float() * w[s])
        if P == n:   # (each slot once)
            dy = whole(4, n, E)
            do, dw = ctx.combine_grad(dy, o, inv, w)
            same(do, (dy.float() * w).flip(0))
            same(dw, (o.flip(0).float() * dy.float()).sum(1, keepdim=True))
        del y
        torch.cuda.empty_cache()


def test_results_on_tables_are_refused(ctx):
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = t.data_ptr()
    E = loki_amd.FL_EINVAL
    mm = lambda y, z=None: lib().fl_matmul_dev(ctx.ctx, FL_BF16, 0, p, p + 4096, None, None, None, 8, 16, 16, 2, p + 8192, p + 12288, 1, 8, y, FL_BF16, z, None)  # noqa: E731
    gr = lambda dx=None, dW=None: lib().fl_matmul_grad_dev(ctx.ctx, FL_BF16, p, None, p + 2048, p + 4096, None, 8, 16, 16, 2, p + 8192, p + 12288, 1, 8, dx, dW, None, FL_BF16, 0)  # noqa: E731
    ag = lambda dz=None, db=None: lib().fl_act_grad_dev(ctx.ctx, FL_BF16, 0, p, None, None, 8, 16, 2, p + 8192, dz, None, db, 0)  # noqa: E731
    cb = lambda y: lib().fl_combine_dev(ctx.ctx, FL_BF16, p, p + 4096, p + 8192, p + 12288, None, 8, 2, 4, 16, 16, y, FL_BF16)  # noqa: E731
    cg = lambda do=None, dw=None: lib().fl_combine_grad_dev(ctx.ctx, FL_BF16, p, p + 2048, p + 4096, p + 8192, p + 12288, 8, 2, 4, 16, 16, do, dw)  # noqa: E731
    for y in (p + 8192, p + 12288):
        assert mm(y) == E and mm(p + 20480, z=y) == E and gr(dx=y) == E and gr(dW=y) == E and cb(y) == E and cg(do=y) == E and cg(dw=y) == E
    assert ag(dz=p + 8192) == E and ag(db=p + 8192) == E and cb(p + 4096) == E and cg(do=p + 4096) == E and cg(dw=p + 4096) == E
    assert mm(p + 20480) == 0 and gr(dx=p + 20480) == 0 and ag(dz=p + 20480) == 0 and cb(p + 20480) == 0 and cg(do=p + 20480) == 0
    ctx.sync()


@pytest.mark.parametrize("n", [1, 40, 600])
def test_fp16_below_its_normal_range(ctx, n):
    """fp16 operands and results below 2^-14 keep their bits: whole multiples of 2^-24, exact in every form"""
    R, K = 72, 136
    x, W = whole(1, n, K, dtype=torch.float16), whole(2, R, K, dtype=torch.float16)
    tiny = (x.float() * 2.0 ** -24).half()
    same(ctx.matmul(tiny, W), mm(x, W) * 2.0 ** -24)
    same(ctx.matmul(x, (W.float() * 2.0 ** -24).half(), dtype=F4), mm(x, W) * 2.0 ** -24)
    dz = whole(3, n, R, dtype=torch.float16)
    dx, dW = ctx.matmul_grad((dz.float() * 2.0 ** -24).half(), x, W)
    same(dx, mm(dz, W.t()) * 2.0 ** -24)
    same(dW, mm(dz.t(), x.t()) * 2.0 ** -24)
    same(ctx.combine(tiny, torch.arange(n, dtype=torch.int32, device="cuda"), topk=1), x.float() * 2.0 ** -24)


def test_first_call_of_a_context_captured(ctx):
    """a product without parts needs nothing of the context but its counters: the first call of a context may be the captured one"""
    n, R, K = 2100, 4104, 72
    c, s = loki_amd.Context(), torch.cuda.Stream()
    x, W = whole(1, n, K), whole(2, R, K)
    y = torch.zeros((n, R), dtype=B, device="cuda")
    torch.cuda.synchronize()
    c.check(lib().fl_set_stream(c.ctx, s.cuda_stream))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        c.matmul(x, W, y=y)
        c.matmul(x, W, y=y, residual=y)
    for i in range(3):
        x.copy_(whole(10 + i, n, K))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(y, 2 * mm(x, W))
    c.close()
