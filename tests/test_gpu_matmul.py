"""GPU: the 16-bit products with their epilogues, dense and by expert, their backward pass, and the combine of picks with its gradients,
against their definitions in 64 bits (_mm_ref.py).

Tolerances, with u = 2^-24 (half an fp32 step) and h = half a step of the type (bf16 2^-8, fp16 2^-11, fp32 u):
  product  operands' products are exact in fp32, K terms are added in some order: an addition each, of up to 2 u as the matrix cores may
           truncate: (2 K + 16) u of sum |x w|. The result is rounded once: h of it (below fp16's normal range 2^-25).
  act      silu: t = z; gelu: t of six roundings. e^-t: its argument's rounding, 2 |t| u, and the instruction, 2 u; 1 + e^-t and the division
           2 u; what an error of t does to s(t) is s (1 - s) |t| <= 0.224 of it: below 8 u |z| for the value with the product. z's own error
           passes on by at most |act'| <= 1.13.
  slope    s + z d s (1 - s): |z d s (1 - s)| <= 0.67, its relative error 2 |t| * 8 u and t^2 s (1 - s) <= 0.44, so 11 u; s 5 u; the sums and
           products 8 u: below 32 u.
  dbias    sums of len terms in fp32: (len + 8) u of sum |dz| and each dz's own 34 u |dy| (|z2| has no bias).
  combine  eight fused products and sums at most: 16 u of sum |w o| + |residual|; d_o one product and one rounding; dw's sum (E + 16) u."""
import numpy as np
import pytest
import torch

from loki_amd import FL_ACT, FL_BF16, FL_EINVAL, FL_ENOMEM, FL_ERANGE, FL_F32, LokiError, lib
from tests import _mm_ref as ref

pytestmark = pytest.mark.gpu
U, F8, TYPES = ref.U, ref.F8, {"bf16": torch.bfloat16, "f16": torch.float16}


def rnd(seed, *shape, dtype=torch.bfloat16, by=1.0):
    return (by * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def near(got, want, err):
    """within err (before rounding) and the rounding to got's type"""
    got = got.cpu()
    h = ref.half(got.dtype)
    tiny = 2.0 ** -25 if got.dtype is torch.float16 else 1e-38
    bound = err + h * (want.abs() + err) + tiny
    d = (got.to(F8) - want).abs()
    ok = ~torch.isnan(want)
    worst = (d / bound)[ok]
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, (float(worst.max()), float(d[ok].max()))
    assert torch.isfinite(got.to(F8)[ok]).all()


def forward(ctx, x, W, W2, bias, kind, residual, offsets, perm, topk, dtype):
    """checks one product with everything kept; slots of no expert stay as they were"""
    g = lambda t: None if t is None else t.cuda()  # noqa: E731
    T = x.dtype
    n = x.shape[0] if perm is None else perm.numel()
    R, K = W.shape[-2:]
    y = torch.full((n, R), 77.0, dtype=dtype or T, device="cuda")
    z, z2 = torch.full((n, R), 78.0, dtype=T, device="cuda"), torch.full((n, R), 79.0, dtype=T, device="cuda") if W2 is not None else None
    if offsets is None:
        ctx.matmul(g(x), g(W), up=g(W2), bias=g(bias), act=kind, residual=g(residual), y=y, z=z, z2=z2)
    else:
        ctx.expert_matmul(g(x), g(W), g(offsets), up=g(W2), bias=g(bias), act=kind, residual=g(residual), perm=g(perm), topk=topk, y=y, z=z, z2=z2)
    ctx.sync()
    wz, mz = ref.products(x, W, offsets, perm, topk)
    ez = (2 * K + 16) * U * mz
    if bias is not None:
        for e, (a, b) in enumerate(ref.spans(offsets, n, 1 if offsets is None else W.shape[0])):
            bb = (bias if offsets is None else bias[e]).to(F8)
            wz[a:b] += bb
            ez[a:b] += U * wz[a:b].abs() + 4 * U * bb.abs()
    near(z, wz, ez)
    wy, ey = ref.act(wz, kind), 1.13 * ez + (8 * U * wz.abs() if kind else 0.0)
    if W2 is not None:
        w2, m2 = ref.products(x, W2, offsets, perm, topk)
        e2 = (2 * K + 16) * U * m2
        near(z2, w2, e2)
        ey = ey * (w2.abs() + e2) + wy.abs() * e2 + U * (wy * w2).abs()
        wy = wy * w2
    if residual is not None:
        wy = wy + residual.to(F8)
        ey = ey + U * wy.abs()
    near(y, wy, ey)
    gone = torch.isnan(wz)
    for t, v in ((y, 77.0), (z, 78.0), (z2, 79.0)):
        assert t is None or bool((t.cpu()[gone] == v).all())


DENSE = [(1, 8, 8), (1, 2048, 264), (2, 136, 72), (5, 72, 1000), (16, 64, 520), (17, 200, 264), (33, 520, 40), (64, 128, 32), (65, 72, 2056), (130, 264, 1032),
         (257, 520, 136), (300, 1000, 2048), (515, 264, 64)]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n,R,K", DENSE)
def test_matmul(ctx, n, R, K, kind):
    T, s = TYPES[kind], n + R + K
    x, W, W2 = rnd(s, n, K, dtype=T), rnd(s + 1, R, K, dtype=T, by=K ** -0.5), rnd(s + 2, R, K, dtype=T, by=K ** -0.5)
    bias, res = rnd(s + 3, R, dtype=torch.float32), rnd(s + 4, n, R, dtype=T)
    print("matmul n %d R %d K %d %s" % (n, R, K, kind), flush=True)
    forward(ctx, x, W, None, bias, "gelu", res, None, None, 1, None)
    forward(ctx, x, W, W2, None, "silu", None, None, None, 1, torch.float32)
    forward(ctx, x, W, None, None, None, res, None, None, 1, torch.float32)


GROUPS = {   # name: (slots of each expert, first slot, slots behind the last)
    "one": ([1], 0, 0), "empty": ([0, 0, 0], 2, 3), "first_empty": ([0, 5, 0, 1], 0, 2), "ragged": ([3, 0, 17, 64, 65, 1, 130], 4, 9),
    "many": ([(7 * i) % 5 for i in range(256)], 0, 1), "one_large": ([0, 600, 2], 1, 0), "middle": ([40, 33, 31, 32, 47, 90], 0, 5)}


def group(name):
    counts, first, after = GROUPS[name]
    off = torch.tensor([first + sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32)
    return len(counts), off, first + sum(counts) + after


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("R,K", [(8, 16), (200, 136), (264, 520)])
def test_expert_matmul(ctx, name, R, K, kind):
    T, (ne, off, n) = TYPES[kind], group(name)
    x, W, W2 = rnd(n, n, K, dtype=T), rnd(n + 1, ne, R, K, dtype=T, by=K ** -0.5), rnd(n + 2, ne, R, K, dtype=T, by=K ** -0.5)
    bias, res = rnd(n + 3, ne, R, dtype=torch.float32), rnd(n + 4, n, R, dtype=T)
    x[:int(off[0])] = float("nan")   # slots of no expert are not read
    x[int(off[-1]):] = float("nan")
    print("expert_matmul %s R %d K %d %s" % (name, R, K, kind), flush=True)
    forward(ctx, x, W, None, bias, "silu", res, off, None, 1, None)
    forward(ctx, x, W, W2, None, "gelu", None, off, None, 1, None)


def routed(n, ne, topk, seed, drop=0.15):
    g = torch.Generator().manual_seed(seed)
    sel = torch.topk(torch.randn((n, ne), generator=g), topk, dim=1).indices.to(torch.int32)
    sel[torch.rand(sel.shape, generator=g) < drop] = -1
    return sel


@pytest.mark.parametrize("n,ne,topk,R,K", [(1, 8, 8, 72, 64), (6, 256, 8, 136, 264), (40, 5, 3, 264, 136), (200, 7, 2, 520, 72), (700, 3, 1, 64, 136)])
def test_expert_matmul_through_perm(ctx, n, ne, topk, R, K):
    sel = routed(n, ne, topk, n)
    off, perm, _ = ref.order(sel, ne)
    perm[int(off[-1]):] = 2 ** 30   # entries that no expert has are not read
    x, W, W2 = rnd(n, n, K), rnd(n + 1, ne, R, K, by=K ** -0.5), rnd(n + 2, ne, R, K, by=K ** -0.5)
    print("through perm n %d ne %d topk %d" % (n, ne, topk), flush=True)
    forward(ctx, x, W, W2, None, "silu", None, off, perm, topk, None)
    forward(ctx, x, W, None, None, None, None, off, perm, topk, torch.float32)


def test_rows_outside_x_count_as_zeros(ctx):
    off, perm = torch.tensor([0, 3, 6], dtype=torch.int32), torch.tensor([0, 9, -1, 3, 2 ** 31 - 1, 1], dtype=torch.int32)
    x, W = rnd(1, 2, 40), rnd(2, 2, 24, 40)
    forward(ctx, x, W, None, None, None, None, off, perm, 2, None)   # rows 0, 4, .., 1, .., 0: those above 1 are not there


def backward(ctx, dz, dz2, x, W, W2, offsets, perm, topk, dtype, add=False):
    T = x.dtype
    g = lambda t: None if t is None else t.cuda()  # noqa: E731
    n, R, K = dz.shape[0], *W.shape[-2:]
    dx = torch.full((n, K), 77.0, dtype=T, device="cuda")
    base, base2 = rnd(5, *W.shape, dtype=dtype or T), rnd(6, *W.shape, dtype=dtype or T)
    args = dict(dz2=g(dz2), up=g(W2), dx=dx)
    if add:
        args.update(dW=g(base), dW2=g(base2) if W2 is not None else None)
    else:
        args.update(dw_dtype=dtype)
    out = ctx.matmul_grad(g(dz), g(x), g(W), **args) if offsets is None else ctx.expert_matmul_grad(g(dz), g(x), g(W), g(offsets), perm=g(perm), topk=topk, **args)
    ctx.sync()
    wx, mx, wW, mW = ref.grads(dz, x, W, offsets, perm, topk)
    terms = R
    if W2 is not None:
        wx2, mx2, wW2, mW2 = ref.grads(dz2, x, W2, offsets, perm, topk)
        wx, mx, terms = wx + wx2, mx + mx2, 2 * R
    near(out[0], wx, (2 * terms + 16) * U * mx)
    assert bool((out[0].cpu()[torch.isnan(wx)] == 77.0).all())
    most = max(b - a for a, b in ref.spans(offsets, n, 1 if offsets is None else W.shape[0]))
    sums = [(out[1], wW, mW, base)] + ([(out[2], wW2, mW2, base2)] if W2 is not None else [])
    for got, w, m, b in sums:
        e = (2 * most + 16) * U * m
        if add:
            w = w + b.to(F8)
            e = e + U * w.abs()
        near(got, w, e)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n,R,K", DENSE)
def test_matmul_grad(ctx, n, R, K, kind):
    T, s = TYPES[kind], n + R + K
    dz, dz2, x = rnd(s, n, R, dtype=T), rnd(s + 1, n, R, dtype=T), rnd(s + 2, n, K, dtype=T)
    W, W2 = rnd(s + 3, R, K, dtype=T, by=R ** -0.5), rnd(s + 4, R, K, dtype=T, by=R ** -0.5)
    print("matmul_grad n %d R %d K %d %s" % (n, R, K, kind), flush=True)
    backward(ctx, dz, None, x, W, None, None, None, 1, None)
    backward(ctx, dz, dz2, x, W, W2, None, None, 1, torch.float32)
    backward(ctx, dz, None, x, W, None, None, None, 1, torch.float32, add=True)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("R,K", [(8, 16), (200, 136), (264, 520)])
def test_expert_matmul_grad(ctx, name, R, K, kind):
    T, (ne, off, n) = TYPES[kind], group(name)
    dz, dz2, x = rnd(n, n, R, dtype=T), rnd(n + 1, n, R, dtype=T), rnd(n + 2, n, K, dtype=T)
    W, W2 = rnd(n + 3, ne, R, K, dtype=T, by=R ** -0.5), rnd(n + 4, ne, R, K, dtype=T, by=R ** -0.5)
    for t in (dz, dz2, x):
        t[:int(off[0])] = float("nan")
        t[int(off[-1]):] = float("nan")
    print("expert_matmul_grad %s R %d K %d %s" % (name, R, K, kind), flush=True)
    backward(ctx, dz, dz2, x, W, W2, off, None, 1, None)
    backward(ctx, dz, None, x, W, None, off, None, 1, torch.float32, add=True)
    backward(ctx, dz, None, x, W, None, off, None, 1, None, add=True)


def test_an_experts_nan_stays_its_own(ctx):
    """NaN and infinities in one expert's rows and matrix reach no other expert, also inside a tile that holds both"""
    ne, off, n = group("ragged")
    dz, x, W = rnd(1, n, 72), rnd(2, n, 136), rnd(3, ne, 72, 136)
    clean = [t.clone() for t in ctx.expert_matmul_grad(dz.cuda(), x.cuda(), W.cuda(), off.cuda())] + [ctx.expert_matmul(x.cuda(), W.cuda(), off.cuda())]
    a, b = int(off[2]), int(off[3])
    x[a:b], dz[a + 1:b, 3] = float("inf"), float("nan")
    W[2] = float("nan")
    dx, dW = ctx.expert_matmul_grad(dz.cuda(), x.cuda(), W.cuda(), off.cuda())
    y = ctx.expert_matmul(x.cuda(), W.cuda(), off.cuda())
    ctx.sync()
    live = [i for i in range(int(off[0]), int(off[-1])) if not a <= i < b]
    others = [e for e in range(ne) if e != 2]
    assert torch.equal(dx[live], clean[0][live]) and torch.equal(dW[others], clean[1][others]) and torch.equal(y[live], clean[2][live])
    assert bool(torch.isnan(y[a:b]).all())


@pytest.mark.parametrize("n,ne,topk,R,K", [(3, 8, 2, 72, 64), (40, 5, 3, 264, 136), (200, 7, 2, 136, 520), (700, 3, 1, 64, 136)])
def test_expert_matmul_grad_through_perm(ctx, n, ne, topk, R, K):
    sel = routed(n, ne, topk, n)
    off, perm, _ = ref.order(sel, ne)
    P = perm.numel()
    dz, dz2, x, W, W2 = rnd(n, P, R), rnd(n + 1, P, R), rnd(n + 2, n, K), rnd(n + 3, ne, R, K, by=R ** -0.5), rnd(n + 4, ne, R, K, by=R ** -0.5)
    print("grad through perm n %d ne %d topk %d" % (n, ne, topk), flush=True)
    backward(ctx, dz, dz2, x, W, W2, off, perm, topk, None)
    backward(ctx, dz, None, x, W, None, off, perm, topk, torch.float32)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("n,R", [(1, 8), (3, 136), (70, 520), (1000, 72), (600, 2056), (5000, 264)])
def test_act_grad(ctx, n, R, act, kind):
    T = TYPES[kind]
    dy, z, z2 = rnd(n, n, R, dtype=T), rnd(n + 1, n, R, dtype=T, by=3.0), rnd(n + 2, n, R, dtype=T)
    z.view(-1)[:6] = torch.tensor([0.0, -0.0, 60.0, -60.0, 200.0, -200.0], dtype=T)
    d8, z8, zz = dy.to(F8), z.to(F8), z2.to(F8)
    sl, e = ref.slope(z8, act), 32 * U if act else 0.0
    base = rnd(4, R, dtype=torch.float32)
    dz, none, db = ctx.act_grad(dy.cuda(), z.cuda(), act, bias=True, dbias=base.cuda())
    assert none is None
    near(dz, d8 * sl, d8.abs() * (e + 2 * U))
    near(db, (d8 * sl).sum(0) + base.to(F8), (d8.abs() * (34 * U + (n + 8) * U * sl.abs())).sum(0) + U * base.to(F8).abs())
    dz, dz2, none = ctx.act_grad(dy.cuda(), z.cuda(), act, z2=z2.cuda())
    assert none is None
    near(dz, d8 * sl * zz, (d8 * zz).abs() * (e + 4 * U))
    near(dz2, d8 * ref.act(z8, act), (d8 * z8).abs() * 10 * U)
    a, b, c = dy.cuda(), z.cuda(), z2.cuda()   # in place
    ctx.act_grad(a, b, act, z2=c, dz=b, dz2=a)
    ctx.sync()
    assert torch.equal(b, dz) and torch.equal(a, dz2)


def test_act_grad_by_expert(ctx):
    ne, off, n = group("ragged")
    R = 136
    dy, z = rnd(1, n, R), rnd(2, n, R)
    dy[:int(off[0])] = float("nan")
    dy[int(off[-1]):] = float("nan")
    out = torch.full((n, R), 77.0, dtype=torch.bfloat16, device="cuda")
    dz, _, db = ctx.act_grad(dy.cuda(), z.cuda(), "silu", bias=True, offsets=off.cuda(), dz=out)
    d = dy.to(F8) * ref.slope(z.to(F8), "silu")
    live = slice(int(off[0]), int(off[-1]))
    near(dz[live], d[live], dy[live].to(F8).abs() * 34 * U)
    assert bool((out[:int(off[0])] == 77.0).all()) and bool((out[int(off[-1]):] == 77.0).all())
    for e, (a, b) in enumerate(ref.spans(off, n, ne)):
        near(db[e], d[a:b].sum(0), ((b - a + 8) * U * d[a:b].abs() + 34 * U * dy[a:b].to(F8).abs()).sum(0))
    out.fill_(77.0)   # without the bias
    ctx.act_grad(dy.cuda(), z.cuda(), "silu", offsets=off.cuda(), dz=out)
    ctx.sync()
    assert torch.equal(out[live], dz[live]) and bool((out[:int(off[0])] == 77.0).all()) and bool((out[int(off[-1]):] == 77.0).all())


def test_slope_where_a_factor_vanishes(ctx):
    """far out on both sides, where the sigmoid or its complement is 0: slope 1 or 0, nothing infinite or NaN"""
    z = torch.tensor([3e38, -3e38, 1e30, -1e30, 1e4, -1e4, 100.0, -100.0], dtype=torch.bfloat16, device="cuda")[None]
    one = torch.ones_like(z)
    for act in ("silu", "gelu"):
        dz, _, _ = ctx.act_grad(one, z, act)
        ctx.sync()
        assert torch.equal(dz, (z > 0).to(dz.dtype)), (act, dz)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n,ne,topk,E", [(1, 4, 1, 8), (3, 8, 8, 72), (17, 256, 6, 520), (70, 16, 2, 2056), (600, 9, 3, 136), (530, 32, 8, 1032)])
def test_combine(ctx, n, ne, topk, E, kind):
    T, sel = TYPES[kind], routed(n, ne, topk, n)
    if n > 2:
        sel[1] = -1                    # a row that no expert takes
        sel[2] = sel[2, 0].item()      # the same expert again and again
        sel[0, 0] = ne                 # and one that is none
    off, perm, inv = ref.order(sel, ne)
    P = perm.numel()
    garbage = inv.clone()
    garbage[inv < 0] = P // 2          # a pair without a slot is told by sel, whatever inv holds
    o, w, res, dy = rnd(n, P, E, dtype=T), rnd(n + 1, n, topk, dtype=torch.float32), rnd(n + 2, n, E, dtype=T), rnd(n + 3, n, E, dtype=T)
    print("combine n %d topk %d E %d" % (n, topk, E), flush=True)
    for r, dt in ((res, None), (None, torch.float32)):
        y = ctx.combine(o.cuda(), garbage.cuda(), w.cuda(), sel=sel.cuda(), n_exp=ne, residual=None if r is None else r.cuda(), dtype=dt)
        ctx.sync()
        wy, m = ref.combine(o, inv, w, sel, ne, r)
        near(y, wy, 16 * U * m)
    do = torch.full((P, E), 77.0, dtype=T, device="cuda")
    do, dw = ctx.combine_grad(dy.cuda(), o.cuda(), garbage.cuda(), w.cuda(), sel=sel.cuda(), n_exp=ne, do=do)
    ctx.sync()
    wo, ww, mw = ref.combine_grad(dy, o, inv, w, sel, ne)
    near(do, wo, U * wo.abs())
    assert bool((do.cpu()[torch.isnan(wo)] == 77.0).all())
    near(dw, ww, (E + 16) * U * mw)
    y = ctx.combine(o.cuda(), inv.cuda(), topk=topk)   # ones, and slots outside 0 .. P - 1 are skipped
    ctx.sync()
    wy, m = ref.combine(o, inv, torch.ones((n, topk)), sel, ne, None)
    near(y, wy, 16 * U * m)


def test_no_rows(ctx):
    """no rows: nothing is written, a matrix's gradient is 0 or stays"""
    x, W, dz = torch.zeros((0, 40), dtype=torch.bfloat16, device="cuda"), rnd(1, 24, 40).cuda(), torch.zeros((0, 24), dtype=torch.bfloat16, device="cuda")
    assert ctx.matmul(x, W).shape == (0, 24)
    dx, dW = ctx.matmul_grad(dz, x, W)
    assert dx.shape == (0, 40) and bool((dW == 0).all())
    base = rnd(2, 24, 40).cuda()
    assert torch.equal(ctx.matmul_grad(dz, x, W, dW=base.clone())[1], base)
    assert bool((ctx.act_grad(dz, None, None, bias=True)[2] == 0).all())
    inv = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert ctx.combine(rnd(3, 4, 40).cuda(), inv, topk=2).shape == (0, 40)


def test_refusals(ctx):
    L, c = lib(), ctx.ctx
    t = torch.zeros(1 << 16, dtype=torch.bfloat16, device="cuda")
    p = t.data_ptr()
    x, W, y, z = p, p + 8192, p + 16384, p + 24576
    mm = lambda ty=FL_BF16, act=0, x=x, W=W, W2=None, b=None, r=None, n=4, R=16, K=16, ne=1, o=None, pm=None, k=1, xr=4, y=y, yt=FL_BF16, z=None, z2=None: \
        L.fl_matmul_dev(c, ty, act, x, W, W2, b, r, n, R, K, ne, o, pm, k, xr, y, yt, z, z2)   # noqa: E731
    assert mm() == 0
    for kw in (dict(ty=0), dict(ty=FL_F32), dict(act=3), dict(act=-1), dict(R=0), dict(R=12), dict(K=4), dict(K=-8), dict(K=65544), dict(ne=2), dict(ne=0), dict(ne=257, o=p),
               dict(yt=17), dict(x=None), dict(W=None), dict(y=None), dict(x=p + 8), dict(y=y + 2), dict(W2=W, b=p), dict(z2=z), dict(pm=p), dict(o=p, pm=p, k=0),
               dict(o=p, pm=p, k=9), dict(y=x), dict(y=W + 16), dict(z=y), dict(r=y, yt=FL_F32), dict(r=y + 16), dict(n=1 << 20)):
        assert mm(**kw) == FL_EINVAL, kw
        assert L.fl_last_error(c)
    assert mm(n=-1) == FL_ERANGE and mm(n=(1 << 24) + 1) == FL_ERANGE and mm(o=p, pm=p, xr=2 ** 30) == FL_ERANGE and mm(o=p, pm=p, xr=-1) == FL_ERANGE
    assert mm(n=0, x=None, W=None, y=None) == 0 and mm(r=y) == 0
    gr = lambda ty=FL_BF16, dz=x, dz2=None, x=W, W=z, W2=None, n=4, R=16, K=16, ne=1, o=None, dx=y, dW=None, dW2=None, dt=FL_BF16: \
        L.fl_matmul_grad_dev(c, ty, dz, dz2, x, W, W2, n, R, K, ne, o, None, 1, 0, dx, dW, dW2, dt, 0)   # noqa: E731
    assert gr() == 0
    for kw in (dict(dx=None), dict(dz=None), dict(W=None), dict(dz2=p), dict(dx=None, dW=y, x=None), dict(dW2=p + 32768), dict(dt=17), dict(dx=x), dict(dW=y), dict(dx=y + 8), dict(n=1 << 20)):
        assert gr(**kw) == FL_EINVAL, kw
    ag = lambda act=1, dy=x, z=z, z2=None, n=4, R=16, o=None, dz=y, dz2=None, db=None: L.fl_act_grad_dev(c, FL_BF16, act, dy, z, z2, n, R, 1, o, dz, dz2, db, 0)   # noqa: E731
    assert ag() == 0 and ag(dz=x) == 0
    for kw in (dict(act=9), dict(dz=None), dict(z=None), dict(dy=None), dict(dz2=W), dict(z2=W, db=p + 32768), dict(dz=x + 16), dict(dz=y, db=y), dict(db=x, dz=None), dict(n=1 << 20)):
        assert ag(**kw) == FL_EINVAL, kw
    iv = torch.zeros(64, dtype=torch.int32, device="cuda").data_ptr()
    cb = lambda o=x, inv=iv, n=4, k=2, ne=4, P=8, E=16, y=y, yt=FL_BF16, r=None: L.fl_combine_dev(c, FL_BF16, o, inv, None, iv, r, n, k, ne, P, E, y, yt)   # noqa: E731
    assert cb() == 0 and cb(r=y) == 0
    for kw in (dict(o=None), dict(inv=None), dict(ne=0), dict(ne=300), dict(E=12), dict(E=0), dict(y=x), dict(yt=17), dict(r=y + 16), dict(y=None), dict(P=1 << 22)):
        assert cb(**kw) == FL_EINVAL, kw
    assert cb(k=9) == FL_ERANGE and cb(n=-1) == FL_ERANGE and cb(P=-1) == FL_ERANGE
    cg = lambda dy=W, o=x, do=y, dw=None, n=4: L.fl_combine_grad_dev(c, FL_BF16, dy, o, iv, None, iv, n, 2, 4, 8, 16, do, dw)   # noqa: E731
    assert cg() == 0 and cg(do=x) == 0
    for kw in (dict(dy=None), dict(do=None), dict(do=W), dict(do=x + 16), dict(dw=W), dict(n=1 << 20)):
        assert cg(**kw) == FL_EINVAL, kw
    ctx.sync()
    with pytest.raises(LokiError, match="go together"):
        ctx.matmul_grad(t[:64].view(4, 16), t[:64].view(4, 16), t[:256].view(16, 16), dz2=t[:64].view(4, 16))


@pytest.mark.parametrize("n,R,K", [(1, 136, 264), (40, 264, 136), (300, 520, 264)])
def test_captured_calls(ctx, n, R, K):
    """a product with its backward pass captured once and replayed, with other work between, is the eager result every time"""
    import loki_amd
    c = loki_amd.Context()
    s = torch.cuda.Stream()
    x, W, dy, bias = rnd(1, n, K).cuda(), rnd(2, R, K, by=K ** -0.5).cuda(), rnd(3, n, R).cuda(), rnd(4, R, dtype=torch.float32).cuda()
    y, z = torch.empty((n, R), dtype=torch.bfloat16, device="cuda"), torch.empty((n, R), dtype=torch.bfloat16, device="cuda")
    dz, dx, dW, db = torch.empty_like(y), torch.empty_like(x), torch.zeros_like(W), torch.zeros_like(bias)

    def step():
        c.matmul(x, W, bias=bias, act="silu", y=y, z=z)
        c.act_grad(dy, z, "silu", dz=dz, dbias=db)
        c.matmul_grad(dz, x, W, dW=dW, dx=dx)

    torch.cuda.synchronize()
    c.check(lib().fl_set_stream(c.ctx, s.cuda_stream))
    with torch.cuda.stream(s):
        step()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
    for i in range(4):
        x.copy_(rnd(10 + i, n, K)); dW.zero_(); db.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, z, dz, dx, dW, db)]
        dW.zero_(); db.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (y, z, dz, dx, dW, db)))
    c.close()


def test_workspace_under_capture(ctx):
    """a bias's gradient that needs a larger workspace than the context has is refused under capture, and the capture goes on"""
    import loki_amd
    c = loki_amd.Context()
    s = torch.cuda.Stream()
    dy, out = rnd(1, 4000, 264).cuda(), torch.zeros(264, device="cuda")
    torch.cuda.synchronize()
    c.check(lib().fl_set_stream(c.ctx, s.cuda_stream))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            rc = lib().fl_act_grad_dev(c.ctx, FL_BF16, 0, dy.data_ptr(), None, None, 4000, 264, 1, None, None, None, out.data_ptr(), 0)
            out.add_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    assert rc == FL_ENOMEM and bool((out == 1.0).all())
    c.close()


def test_training_step(ctx):
    """route, dispatch, the experts, the combine and all of it backwards to the rows, the experts' matrices and the router, as a program runs
    it, against 64-bit autograd. Each of the chain's roundings to bfloat16 (x, the two products kept, h, o, y; do, dz, dz2, dx, its sum; the
    matrices' own) is half a step at most, 2^-8 of what it rounds, and six of them meet in any one result: 6 * 2^-8 of its norm, twice that
    where a slope or a difference of picks passes an error on (the router's gradient is of differences between picks)."""
    n, ne, topk, E, H = 48, 16, 4, 1024, 264
    x = rnd(1, n, E)
    Wr, bias = rnd(2, ne, E, dtype=torch.float32, by=0.05), torch.zeros(ne)
    Wg, Wu, Wd = rnd(3, ne, H, E, by=E ** -0.5), rnd(4, ne, H, E, by=E ** -0.5), rnd(5, ne, E, H, by=H ** -0.5)
    dy = rnd(6, n, E)
    g = [t.cuda() for t in (x, Wr, bias, Wg, Wu, Wd, dy)]
    gx, gr, gb, gg, gu, gd, gy = g
    ctx.set_routing(1, 1, topk, 2.5)
    try:
        xf = gx.float()
        logits, _, sel, w = ctx.route(gr, gb, xf, topk=topk)
        _, off, perm, inv, _, _ = ctx.dispatch(sel, n_exp=ne)
        h, z, z2 = ctx.expert_matmul(gx, gg, off, up=gu, act="silu", perm=perm, topk=topk, keep=True)
        o = ctx.expert_matmul(h, gd, off)
        y = ctx.combine(o, inv, w, sel=sel, n_exp=ne, residual=gx)
        do, dw = ctx.combine_grad(gy, o, inv, w, sel=sel, n_exp=ne)
        dh, dWd = ctx.expert_matmul_grad(do, h, gd, off, dw_dtype=torch.float32)
        dz, dz2, _ = ctx.act_grad(dh, z, "silu", z2=z2, offsets=off)
        dxs, dWg, dWu = ctx.expert_matmul_grad(dz, gx, gg, off, dz2=dz2, up=gu, perm=perm, topk=topk)
        dx = ctx.combine(dxs, inv, sel=sel, n_exp=ne, residual=gy, dtype=torch.float32)
        dl, dWr, dxr = ctx.route_grad(gr, xf, logits, sel, dw)
        dx += dxr
        ctx.sync()
    finally:
        ctx.set_routing()
    leaf = lambda t: t.to(F8).requires_grad_(True)  # noqa: E731
    a = [leaf(t) for t in (x, Wr, Wg, Wu, Wd)]
    s = torch.sigmoid(a[0] @ a[1].t())
    pick = sel.cpu().long()
    sk = s.gather(1, pick)
    wk = 2.5 * sk / sk.sum(1, keepdim=True)
    out = a[0]
    for k in range(topk):
        gk, uk, dk = a[2][pick[:, k]], a[3][pick[:, k]], a[4][pick[:, k]]
        zz = torch.einsum("te,the->th", a[0], gk)
        hh = zz * torch.sigmoid(zz) * torch.einsum("te,the->th", a[0], uk)
        out = out + wk[:, k:k + 1] * torch.einsum("th,teh->te", hh, dk)
    (out * dy.to(F8)).sum().backward()
    for name, got, want, times in (("y", y, out.detach(), 1), ("dx", dx, a[0].grad, 2), ("dWr", dWr, a[1].grad, 2), ("dWg", dWg, a[2].grad, 2), ("dWu", dWu, a[3].grad, 2),
                                   ("dWd", dWd, a[4].grad, 2)):
        far = float((got.cpu().to(F8) - want).norm() / want.norm())
        assert far <= 6 * times * 2.0 ** -8, (name, far)
