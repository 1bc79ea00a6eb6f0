"""GPU: the balance loss with its counts and gradient, and the router's backward pass, against their definitions in 64 bits
(_train_ref.py).

Tolerances, with u = 2^-24 (half an fp32 step):
  loss    every term is positive, so relative errors add up along the longest chain. p: exp (3 u), 1 + t, a reciprocal of 2 u and a
          product (7 u in all), the row's sum (4 + 7 adds, and its terms' 7 u), its reciprocal and a product (3 u): 28 u. The mean:
          rows of a wave one after another (at most n / 16 + 4), 16 waves, chunks / 4 + 3 <= 67, the division. f and alpha: 6 u; the
          experts' sum: 12. (130 + n) u is an upper bound from n = 5 on, and below there is one chunk: 28 + n + 16 + 21 u.
  dlogits a product of p (28 u), 1 - s (7 u), k (4 u) and f - D: f 3 u, D = sum f p 28 + 3 + 12 u, relative to f + D, and three
          roundings: within 90 u of |k| p (1 - s) (f + D).
  dz      s and 1 - s 5 u each, S and D over at most 8 picks: 60 u of scale / S (|dw| + sum |dw| s / S) s (1 - s), and one rounding
          for dz_in.
  dW, dx  against the 64-bit product of the kernel's own dlogits: per product 3 * 2^-22 (operands in two 11-bit halves, the product
          of the lower ones left out), an fp32 addition per term at most: (K + 16) u + 3 * 2^-22 of sum |a b| + what the halves' scale
          leaves of the smallest values, 2^-39 of the row's largest |dz| times the largest |x| or |W|, per term."""
import ctypes

import numpy as np
import pytest

from tests import _train_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def routed(n, ne, topk, seed, spread=1.7):
    rng = np.random.default_rng(seed)
    z = (spread * rng.standard_normal((n, ne)) + 0.5 * rng.standard_normal(ne)).astype(np.float32)
    sel = np.argsort(-z, axis=1, kind="stable")[:, :topk].astype(np.int32)
    return rng, z, sel


def gpu(a):
    import torch
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def run_balance(ctx, z, sel, alpha, seq=None, gloss=None):
    dz_, ds, dq, dg = gpu(z), gpu(sel), gpu(None if seq is None else np.asarray(seq, np.int32)), gpu(gloss)
    counts, loss = ctx.balance_loss(dz_, ds, alpha, seq=dq)
    grad = ctx.balance_loss_grad(dz_, counts, sel.shape[1], alpha, seq=dq, gloss=dg)
    ctx.sync()
    return counts.cpu().numpy(), loss.cpu().numpy(), grad.cpu().numpy()


def check_balance(got, z, sel, alpha, seq, gloss=None):
    counts, loss, dz, mag = ref.balance(z, sel, alpha, seq, gloss)
    n = z.shape[0]
    assert np.array_equal(got[0], counts)
    assert np.all(np.abs(got[1] - loss) <= (130 + n) * U * np.abs(loss) + 1e-44), np.abs(got[1] - loss).max()
    assert np.all(np.abs(got[2] - dz) <= 90 * U * mag + 1e-44), (np.abs(got[2] - dz) / np.maximum(90 * U * mag, 1e-44)).max()


@pytest.mark.parametrize("n,ne,topk,seq", [
    (1, 1, 1, None), (1, 256, 8, None), (2, 63, 3, None), (17, 64, 8, None), (129, 65, 5, None), (300, 160, 6, None), (1000, 255, 8, None),
    (40, 256, 8, [0, 13, 13, 40]),              # an empty sequence
    (700, 256, 8, [30, 31, 500, 640]),          # rows of no sequence on both sides
    (5000, 32, 2, [0, 4999, 5000]),             # a long and a short one
    (3000, 128, 4, list(range(0, 3001, 10))),   # 300 of them: one workgroup each
    (9, 16, 2, [4, 4])])                        # no rows at all
def test_balance(ctx, n, ne, topk, seq):
    rng, z, sel = routed(n, ne, topk, n + ne)
    print("balance n %d ne %d" % (n, ne), flush=True)
    gloss = None if seq is None else (rng.standard_normal(len(seq) - 1)).astype(np.float32)
    got = run_balance(ctx, z, sel, 0.01, seq, gloss)
    check_balance(got, z, sel, np.float32(0.01), [0, n] if seq is None else seq, gloss)


def test_balance_long(ctx):
    rng, z, sel = routed(20011, 256, 8, 5)
    seq = [0, 1, 9000, 20011]
    check_balance(run_balance(ctx, z, sel, 1e-4, seq), z, sel, np.float32(1e-4), seq)


def test_balance_masked_and_extreme_rows(ctx):
    """-inf columns (masked experts), rows of -inf only, the type's lowest value, tiny and huge logits, +inf"""
    rng, z, sel = routed(96, 64, 4, 8)
    low = np.finfo(np.float32).min
    z[:, 7] = -np.inf
    z[3] = -np.inf
    z[4] = low
    z[5, :] -= 200.0
    z[6, :] += 200.0
    z[8, 10] = np.inf
    z[9, 1:] = low
    z[10] = -60.0
    z[11, :32] = -35.0; z[11, 32:] = -20.0
    got = run_balance(ctx, z, sel, 0.5, [0, 50, 96])
    assert np.all(np.isfinite(got[1])) and np.all(np.isfinite(got[2]))
    want = ref.balance(np.where(z == low, -np.inf, z), sel, 0.5, [0, 50, 96])
    z4 = z.copy(); z4[4] = -5.0   # equal logits have equal shares, whatever their size
    p4 = ref.balance(z4, sel, 0.5, [0, 50, 96])
    assert np.abs(got[1] - p4[1]).max() <= 300 * U * p4[1].max()
    rows = [t for t in range(96) if t not in (4,)]
    assert np.all(np.abs(got[2][rows] - want[2][rows]) <= 90 * U * want[3][rows] + 1e-44)
    assert np.all(got[2][3] == 0)


def test_balance_nan_stays_in_its_sequence(ctx):
    rng, z, sel = routed(60, 32, 2, 9)
    clean = run_balance(ctx, z, sel, 0.5, [0, 20, 40, 60])
    z[25, 3] = np.nan
    got = run_balance(ctx, z, sel, 0.5, [0, 20, 40, 60])
    assert np.isnan(got[1][1]) and np.array_equal(got[1][[0, 2]], clean[1][[0, 2]])
    keep = np.arange(60) != 25
    assert np.array_equal(got[2][keep], clean[2][keep]) and np.all(np.isnan(got[2][25]))


def test_balance_picks_outside_and_twice(ctx):
    """picks of -1 or n_exp and above count for no expert; the same expert twice in a row counts twice"""
    rng, z, sel = routed(33, 40, 4, 10)
    sel[2] = -1; sel[5, 1] = 40; sel[6] = 7; sel[7, 0] = 2 ** 30
    check_balance(run_balance(ctx, z, sel, 0.25), z, sel, 0.25, [0, 33])


def test_balance_padding_is_not_read_and_adds_stay(ctx):
    """NaN in the rows of no sequence; with a tensor to add to, those rows stay and the others get the sum"""
    import torch
    rng, z, sel = routed(50, 24, 3, 11)
    seq = np.array([5, 20, 44], np.int32)
    zz = z.copy(); zz[:5] = np.nan; zz[44:] = np.nan
    got = run_balance(ctx, zz, sel, 0.5, seq)
    check_balance(got, z, sel, 0.5, seq)
    assert np.all(got[2][:5] == 0) and np.all(got[2][44:] == 0)
    base = rng.standard_normal(z.shape).astype(np.float32)
    out = ctx.balance_loss_grad(gpu(zz), gpu(got[0]), 3, 0.5, seq=gpu(seq), dlogits=gpu(base))
    ctx.sync()
    assert np.array_equal(out.cpu().numpy(), (base + got[2]).astype(np.float32))


def test_balance_bad_offsets_stay_in_bounds(ctx):
    """offsets past the ends are clamped; nothing outside the outputs is written"""
    import torch
    rng, z, sel = routed(30, 16, 2, 12)
    got = run_balance(ctx, z, sel, 0.5, [-5, 10, 10 ** 6])
    check_balance(got, z, sel, 0.5, [0, 10, 30])
    n, ne = z.shape
    buf = torch.full((n * ne + 64,), 3.0, device="cuda")
    cnt = torch.full((ne + 8,), 9, dtype=torch.int32, device="cuda"); loss = torch.full((9,), 4.0, device="cuda")
    from loki_amd import lib
    P = lambda t, o=0: ctypes.c_void_p(t.data_ptr() + 4 * o)   # noqa: E731
    zt, st, sq = gpu(z), gpu(sel), gpu(np.array([20, 3], np.int32))   # descending
    ctx.check(lib().fl_balance_loss_dev(ctx.ctx, P(zt), P(st), P(sq), n, 1, ne, 2, 0.5, P(cnt, 4), P(loss, 4)))
    ctx.check(lib().fl_balance_loss_grad_dev(ctx.ctx, P(zt), P(cnt, 4), P(sq), None, n, 1, ne, 2, 0.5, 0, P(buf, 32)))
    ctx.sync()
    assert torch.all(buf[:32] == 3) and torch.all(buf[-32:] == 3) and torch.all(cnt[:4] == 9) and torch.all(cnt[-4:] == 9)
    assert torch.all(loss[:4] == 4) and torch.all(loss[5:] == 4)


# ---------------------------------------------------------------- the router's backward pass
def check_products(W, x, dz, dW, dx, base=None):
    dz8, W8, x8 = dz.astype(np.float64), W.astype(np.float64), x.astype(np.float64)
    n, ne = dz.shape
    a = np.abs(dz8)
    rowmax = a.max(axis=1, keepdims=True) if n else a[:, :1]
    if dx is not None:
        tol = ((ne + 16) * U + 3 * 2.0 ** -22) * (a @ np.abs(W8)) + ne * 2.0 ** -39 * rowmax * np.abs(W8).max() + 1e-40
        err = np.abs(dx - dz8 @ W8)
        assert np.all(err <= tol), (err / tol).max()
    if dW is not None:
        tol = ((n + 16) * U + 3 * 2.0 ** -22) * (a.T @ np.abs(x8)) + (2.0 ** -39 * n * (rowmax * np.abs(x8)).max() if n else 0) + 1e-40
        want = dz8.T @ x8
        if base is not None:
            want = want + base
            tol = tol + U * np.abs(want)
        err = np.abs(dW - want)
        assert np.all(err <= tol), (err / tol).max()


def run_grad(ctx, W, x, z, sel, dw, dz, **kw):
    out = ctx.route_grad(gpu(W), gpu(x), gpu(z), gpu(sel), gpu(dw), gpu(dz), **kw)
    ctx.sync()
    return [None if t is None else t.cpu().numpy() for t in out]


def inputs(n, ne, topk, E, seed):
    rng, z, sel = routed(n, ne, topk, seed)
    W = (0.02 * rng.standard_normal((ne, E))).astype(np.float32)
    x = rng.standard_normal((n, E)).astype(np.float32)
    dw = (1e-3 * rng.standard_normal((n, topk))).astype(np.float32)
    dz = (1e-6 * rng.standard_normal((n, ne))).astype(np.float32)
    return W, x, z, sel, dw, dz


@pytest.fixture
def rule(ctx):
    yield lambda topk, scale=2.5: ctx.set_routing(1, 1, topk, scale)
    ctx.set_routing(8, 4, 8, 2.5)


@pytest.mark.parametrize("n,ne,topk,E", [(1, 2, 1, 1024), (1, 256, 8, 7168), (3, 17, 4, 2048), (16, 64, 8, 1024), (33, 255, 8, 4096), (100, 160, 6, 5120),
                                         (129, 256, 8, 7168), (515, 96, 2, 1024), (1030, 256, 8, 2048)])
def test_route_grad(ctx, rule, n, ne, topk, E):
    rule(topk)
    W, x, z, sel, dw, dz = inputs(n, ne, topk, E, n + ne + E)
    print("route_grad n %d ne %d E %d" % (n, ne, E), flush=True)
    dl, dW, dx = run_grad(ctx, W, x, z, sel, dw, dz)
    want, mag = ref.route_dz(z, sel, dw, dz, 2.5)
    assert np.all(np.abs(dl - want) <= 60 * U * mag + 1e-44), (np.abs(dl - want) / (60 * U * mag + 1e-44)).max()
    check_products(W, x, dl, dW, dx)


def test_route_grad_parts(ctx, rule):
    """either gradient alone, each output alone, the sum into a given dW, the logits' gradient in place"""
    import torch
    from loki_amd import lib
    rule(4, 1.5)
    W, x, z, sel, dw, dz = inputs(70, 48, 4, 1024, 3)
    full = run_grad(ctx, W, x, z, sel, dw, dz)
    only_w = run_grad(ctx, W, x, z, sel, dw, None)
    assert np.all(np.abs(only_w[0] - ref.route_dz(z, sel, dw, None, 1.5)[0]) <= 60 * U * ref.route_dz(z, sel, dw, None, 1.5)[1] + 1e-44)
    only_z = run_grad(ctx, W, x, z, sel, None, dz)
    assert np.array_equal(only_z[0], dz)
    check_products(W, x, dz, only_z[1], only_z[2])
    no_w = run_grad(ctx, W, x, z, sel, dw, dz, need_dW=False)
    assert no_w[1] is None and np.array_equal(no_w[2], full[2])
    no_x = run_grad(ctx, W, x, z, sel, dw, dz, need_dx=False)
    assert no_x[2] is None and np.array_equal(no_x[1], full[1])
    base = np.random.default_rng(4).standard_normal(W.shape).astype(np.float32)
    add = run_grad(ctx, W, x, z, sel, dw, dz, dW=gpu(base))
    check_products(W, x, full[0], add[1], None, base=base)
    # dW alone with the library's own logits' gradient; dz in place
    t = {k: gpu(v) for k, v in dict(W=W, x=x, z=z, sel=sel, dw=dw, dz=dz).items()}
    P = lambda k: ctypes.c_void_p(t[k].data_ptr())   # noqa: E731
    t["dW"] = torch.empty_like(t["W"])
    ctx.check(lib().fl_route_grad_dev(ctx.ctx, None, P("x"), P("z"), P("sel"), P("dw"), P("dz"), 70, 48, 1024, None, P("dW"), 0, None))
    ctx.check(lib().fl_route_grad_dev(ctx.ctx, None, None, P("z"), P("sel"), P("dw"), P("dz"), 70, 48, 1024, P("dz"), None, 0, None))
    ctx.sync()
    assert np.array_equal(t["dW"].cpu().numpy(), full[1]) and np.array_equal(t["dz"].cpu().numpy(), full[0])


def test_route_grad_clamped_sums_and_picks(ctx, rule):
    """rows whose picked sigmoids sum below 2^-14, rows without picks, the same expert twice, picks outside, masked logits"""
    rule(4)
    W, x, z, sel, dw, dz = inputs(40, 32, 4, 1024, 6)
    z[0] -= 25.0; z[1] -= 120.0; z[2] = -np.inf
    sel[3] = -1; sel[4] = 5; sel[5, 2] = 32
    dl, dW, dx = run_grad(ctx, W, x, z, sel, dw, dz)
    want, mag = ref.route_dz(z, sel, dw, dz, 2.5)
    assert np.all(np.abs(dl - want) <= 60 * U * mag + 1e-44)
    assert np.array_equal(dl[3], dz[3]) and np.array_equal(dl[2], dz[2])
    check_products(W, x, dl, dW, dx)


@pytest.mark.parametrize("wide", [1e-30, 1e-12, 1.0, 1e12, 1e28])
def test_route_grad_ranges(ctx, rule, wide):
    """gradients and rows of any size: per-row gradients over 2^40, columns of x over 2^20, all scaled together"""
    rule(2)
    rng = np.random.default_rng(14)
    W, x, z, sel, dw, dz = inputs(300, 40, 2, 1024, 15)
    dz = (dz * 1e6 * np.exp2(rng.integers(-20, 21, (300, 1)))).astype(np.float32) * np.float32(wide)
    x = (x * np.exp2(rng.integers(-10, 11, (1, 1024)))).astype(np.float32)
    dl, dW, dx = run_grad(ctx, W, x, z, sel, None, dz)
    assert np.array_equal(dl, dz)
    check_products(W, x, dz, dW, dx)


def test_route_grad_zero_rows_and_growing_rows(ctx, rule):
    """zero gradients, a zero x, and rows whose size grows along the batch (a running scale has to follow)"""
    rule(2)
    W, x, z, sel, dw, dz = inputs(400, 64, 2, 2048, 16)
    dz[:130] = 0
    x[:, :64] = 0
    x *= np.exp2(np.arange(400) // 16)[:, None].astype(np.float32)
    dl, dW, dx = run_grad(ctx, W, x, z, sel, None, dz)
    assert np.all(dx[:130] == 0) and np.all(dW[:, :64] == 0)
    check_products(W, x, dz, dW, dx)


def test_route_grad_non_finite_rows(ctx, rule):
    """an infinite or NaN gradient or row: its own dx row and dW's affected entries are non-finite, the rest as without it"""
    rule(2)
    W, x, z, sel, dw, dz = inputs(64, 32, 2, 1024, 17)
    clean = run_grad(ctx, W, x, z, sel, None, dz)
    bad = dz.copy(); bad[9, 4] = np.nan
    got = run_grad(ctx, W, x, z, sel, None, bad)
    rows = np.arange(64) != 9
    assert np.all(np.isnan(got[2][9])) and np.array_equal(got[2][rows], clean[2][rows])
    e = np.arange(32) != 4
    assert np.all(np.isnan(got[1][4]))
    check_products(W, x, dz[:, e], got[1][e], None)
    xb = x.copy(); xb[11, 70] = np.inf
    got = run_grad(ctx, W, xb, z, sel, None, dz)
    c = np.arange(1024) != 70
    assert not np.any(np.isfinite(got[1][:, 70]))
    check_products(W[:, c], x[:, c], dz, got[1][:, c], None)


def test_route_grad_no_rows(ctx, rule):
    import torch
    rule(2)
    W = torch.ones((8, 1024), device="cuda"); e = lambda *s, **k: torch.empty(s, device="cuda", **k)   # noqa: E731
    dl, dW, dx = ctx.route_grad(W, e(0, 1024), e(0, 8), e(0, 2, dtype=torch.int32), e(0, 2))
    keep = torch.full((8, 1024), 2.0, device="cuda")
    ctx.route_grad(W, e(0, 1024), e(0, 8), e(0, 2, dtype=torch.int32), e(0, 2), dW=keep)
    ctx.sync()
    assert torch.all(dW == 0) and torch.all(keep == 2) and dx.shape == (0, 1024)


def test_refusals(ctx, rule):
    import torch
    from loki_amd import FL_EINVAL, FL_ERANGE, LokiError, lib
    rule(2)
    L = lib()
    z = torch.zeros((4, 8), device="cuda"); sel = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    c = torch.zeros((1, 8), dtype=torch.int32, device="cuda"); loss = torch.zeros(1, device="cuda"); x = torch.zeros((4, 1024), device="cuda")
    W = torch.zeros((8, 1024), device="cuda"); dw = torch.zeros((4, 2), device="cuda"); dW = torch.empty_like(W); dx = torch.empty_like(x)
    P = lambda t: ctypes.c_void_p(t.data_ptr())   # noqa: E731
    loss_call = lambda n=4, nseq=1, ne=8, k=2, al=0.5, seq=None, zz=P(z): L.fl_balance_loss_dev(ctx.ctx, zz, P(sel), seq, n, nseq, ne, k, al, P(c), P(loss))   # noqa: E731
    assert loss_call(n=-1) == FL_ERANGE and loss_call(k=0) == FL_ERANGE and loss_call(k=9) == FL_ERANGE and loss_call(n=1 << 24) == FL_ERANGE
    assert loss_call(ne=0) == FL_EINVAL and loss_call(ne=257) == FL_EINVAL and loss_call(nseq=0) == FL_EINVAL and loss_call(nseq=2) == FL_EINVAL
    assert loss_call(al=float("nan")) == FL_EINVAL and loss_call(al=float("inf")) == FL_EINVAL and loss_call(zz=None) == FL_EINVAL
    assert loss_call(n=1 << 20) == FL_EINVAL and b"smaller" in L.fl_last_error(ctx.ctx)
    grad = lambda n=4, ne=8, E=1024, d=P(dw), dl=P(z), w=P(dW), o=P(dx), xx=P(x): L.fl_route_grad_dev(ctx.ctx, P(W), xx, P(z), P(sel), d, None, n, ne, E, dl, w, 0, o)   # noqa: E731
    assert grad(n=-1) == FL_ERANGE and grad(n=65537) == FL_ERANGE and grad(ne=300) == FL_EINVAL and grad(E=1000) == FL_EINVAL and grad(E=0) == FL_EINVAL
    assert grad(d=None) == FL_EINVAL and grad(dl=None, w=None, o=None) == FL_EINVAL and grad(xx=None) == FL_EINVAL
    assert grad(o=P(x)) == FL_EINVAL and grad(w=P(W)) == FL_EINVAL and grad(ne=256, E=65536) == FL_EINVAL
    with pytest.raises(LokiError, match="contiguous"):
        ctx.balance_loss(z.t(), sel, 0.5)
    with pytest.raises(LokiError, match="picks a row"):
        ctx.route_grad(W, x, z, torch.zeros((4, 3), dtype=torch.int32, device="cuda"), torch.zeros((4, 3), device="cuda"))
    ctx.sync()


# ---------------------------------------------------------------- as they are used
def step(c, W, bias, x, alpha, seq, gout):
    """a router's training step: route, the balance loss and its gradient, the backward pass from the weights' gradient"""
    logits, _, sel, w = c.route(W, bias, x)
    counts, loss = c.balance_loss(logits, sel, alpha, seq=seq)
    dz = c.balance_loss_grad(logits, counts, sel.shape[1], alpha, seq=seq)
    return (counts, loss) + c.route_grad(W, x, logits, sel, gout, dz=dz)


def test_training_step_eager_and_captured(ctx):
    """route -> balance -> backward on one context: against the 64-bit formulas on the router's own logits and picks, equal bits
    when run again and on another context's stream, and captured into a graph replayed over changed rows between eager calls"""
    import torch
    from loki_amd import Context, lib
    n, ne = 600, 64
    ctx.set_routing(8, 4, 8, 2.5)
    g = torch.Generator(device="cuda").manual_seed(3)
    W = 0.02 * torch.randn((ne, 7168), device="cuda", generator=g); bias = 0.05 * torch.randn(ne, device="cuda", generator=g)
    xs = [torch.randn((n, 7168), device="cuda", generator=g) for _ in range(2)]
    gout = 1e-3 * torch.randn((n, 8), device="cuda", generator=g)
    seq = torch.tensor([0, 250, 251, 590], dtype=torch.int32, device="cuda")
    want = []
    for x in xs:
        out = step(ctx, W, bias, x, 1e-3, seq, gout)
        ctx.sync()
        want.append([t.cpu().numpy() for t in out])
    logits, _, sel, _ = ctx.route(W, bias, xs[0])
    ctx.sync()
    z, s = logits.cpu().numpy(), sel.cpu().numpy()
    cnt, loss, dz, mag = ref.balance(z, s, np.float32(1e-3), seq.cpu().numpy())
    assert np.array_equal(want[0][0], cnt) and np.all(np.abs(want[0][1] - loss) <= 1000 * U * np.abs(loss))
    full, fmag = ref.route_dz(z, s, gout.cpu().numpy(), dz, 2.5)
    assert np.all(np.abs(want[0][2] - full) <= 60 * U * fmag + 90 * U * mag + 1e-44)
    check_products(W.cpu().numpy(), xs[0].cpu().numpy(), *want[0][2:])
    other = Context()
    try:
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        other.check(lib().fl_set_stream(other.ctx, ctypes.c_void_p(side.cuda_stream)))
        x_in = xs[0].clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = step(other, W, bias, x_in, 1e-3, seq, gout)   # workspaces grow here, before the capture
        torch.cuda.synchronize()
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(eager, want[0]))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(other, W, bias, x_in, 1e-3, seq, gout)
        for rep in range(2):
            for i, x in enumerate(xs):
                x_in.copy_(x)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(out, want[i])), (rep, i)
                again = step(ctx, W, bias, x, 1e-3, seq, gout)
                ctx.sync()
                assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(again, want[i]))
        del graph
    finally:
        torch.cuda.synchronize()
        other.close()


def test_workspace_is_not_grown_under_capture(ctx):
    """a captured call that would have to allocate is refused by its code, and the capture goes on: the graph holds what came before
    and after it"""
    import torch
    from loki_amd import FL_ENOMEM, Context, lib
    n, ne = 4000, 64
    z = torch.randn((n, ne), device="cuda"); sel = torch.zeros((n, 8), dtype=torch.int32, device="cuda")
    counts = torch.empty((1, ne), dtype=torch.int32, device="cuda"); loss = torch.empty(1, device="cuda")
    x = torch.zeros(1000, device="cuda")
    c = Context()
    try:
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        c.check(lib().fl_set_stream(c.ctx, side.cuda_stream))
        call = lambda: lib().fl_balance_loss_dev(c.ctx, z.data_ptr(), sel.data_ptr(), None, n, 1, ne, 8, 1e-3, counts.data_ptr(), loss.data_ptr())   # noqa: E731
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            x += 1
            rc = call()
            x += 1
        assert rc == FL_ENOMEM and b"capture" in lib().fl_last_error(c.ctx)
        for rep in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.all(x == 2 * (rep + 1))
        with torch.cuda.stream(side):
            assert call() == 0
        torch.cuda.synchronize()
        assert counts[0, 0].item() == 8 * n
        del graph
    finally:
        torch.cuda.synchronize()
        c.close()


# several tiles of rows a wave, with experts that fill their steps of 32 or do not, and dx's parts beside dW for many rows
@pytest.mark.parametrize("n,ne,topk,E", [(3001, 130, 4, 7168), (2100, 100, 8, 16384), (5003, 64, 6, 8192), (4100, 256, 8, 7168), (2900, 30, 5, 2048)])
def test_route_grad_many_rows(ctx, rule, n, ne, topk, E):
    rule(topk)
    W, x, z, sel, dw, dz = inputs(n, ne, topk, E, n + ne + E)
    print("route_grad n %d ne %d E %d" % (n, ne, E), flush=True)
    dl, dW, dx = run_grad(ctx, W, x, z, sel, dw, dz)
    check_products(W, x, dl, dW, dx)
    _, _, alone = run_grad(ctx, W, x, z, sel, dw, dz, need_dW=False)
    assert np.array_equal(alone.view(np.uint32), dx.view(np.uint32))   # a row's dx has the same bits however the rows are shared out
    for kw in ({"need_dx": False}, {"need_dW": False, "need_dx": False}):   # dW alone (cut into runs of its own), dlogits alone
        dl2, dW2, _ = run_grad(ctx, W, x, z, sel, dw, dz, **kw)
        assert np.array_equal(dl2.view(np.uint32), dl.view(np.uint32))
        check_products(W, x, dl, dW2, None)
    _, _, tail = run_grad(ctx, W, x[-70:], z[-70:], sel[-70:], dw[-70:], dz[-70:], need_dW=False)
    assert np.array_equal(tail.view(np.uint32), dx[-70:].view(np.uint32))


def test_offsets_past_32_bits(ctx, rule):
    """rows behind 2^32 bytes of logits, gradients, x and dx: as the same rows alone"""
    import torch
    rule(2)
    n, ne, T = 1 << 23, 160, 100   # 5.4 GB of logits
    g = torch.Generator(device="cuda").manual_seed(4)
    z = torch.randn((T, ne), device="cuda", generator=g); sel = torch.topk(z, 2, dim=1).indices.to(torch.int32).contiguous()
    big = torch.zeros((n, ne), device="cuda"); big[-T:] = z
    bsel = torch.zeros((n, 2), dtype=torch.int32, device="cuda"); bsel[-T:] = sel
    seq = torch.tensor([n - T - 5, n - T, n], dtype=torch.int32, device="cuda")
    counts, loss = ctx.balance_loss(big, bsel, 0.5, seq=seq)
    grad = ctx.balance_loss_grad(big, counts, 2, 0.5, seq=seq)
    c1, l1 = ctx.balance_loss(z, sel, 0.5)
    g1 = ctx.balance_loss_grad(z, c1, 2, 0.5)
    ctx.sync()
    assert torch.equal(counts[1], c1[0])
    check_balance((c1.cpu().numpy(), l1.cpu().numpy(), g1.cpu().numpy()), z.cpu().numpy(), sel.cpu().numpy(), np.float32(0.5), [0, T])
    assert abs(loss[1].item() - l1.item()) <= 460 * U * l1.item()   # two orders of the same sum, (130 + 100) u each
    assert torch.equal(grad[-T:].view(torch.int32), g1.view(torch.int32)) and not torch.any(grad[:-T - 5])
    del big, bsel, grad
    n, ne, E, T = 65536, 8, 20480, 64   # 5.4 GB of x and of dx
    W = 0.02 * torch.randn((ne, E), device="cuda", generator=g)
    x = torch.zeros((n, E), device="cuda"); x[-T:] = torch.randn((T, E), device="cuda", generator=g)
    z = torch.randn((n, ne), device="cuda", generator=g); sel = torch.topk(z, 2, dim=1).indices.to(torch.int32).contiguous()
    dz = torch.zeros((n, ne), device="cuda"); dz[-T:] = 1e-3 * torch.randn((T, ne), device="cuda", generator=g)
    dl, dW, dx = ctx.route_grad(W, x, z, sel, dz=dz)
    ctx.sync()
    assert not torch.any(dx[:-T]) and torch.equal(dl, dz)
    check_products(W.cpu().numpy(), x[-T:].cpu().numpy(), dz[-T:].cpu().numpy(), dW.cpu().numpy(), dx[-T:].cpu().numpy())
    del x, dx
    torch.cuda.empty_cache()
