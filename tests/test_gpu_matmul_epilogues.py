"""GPU: the 16-bit products' epilogues at sizes that reach every kernel, tile and split (_mm_cases.py; the rules' CPU test says that they do),
and rows picked through perm over the whole of what an entry point takes.

x is -1, 0 or 1 and W as many times a power of two, the bias whole multiples of it: z, z2 and z + bias are exact, whatever the order of the
sums, and only what comes after them has a tolerance, with u = 2^-24: the activation 8 u |z| (as derived for the products of few rows: the
sigmoid's argument, its two instructions and the product with z), the gate's product and the residual's sum u of their results, and the last
rounding half a step of the type."""
import math

import pytest
import torch

from tests import _mm_cases as cases
from tests import _mm_ref as ref
from tests.test_gpu_matmul_kernels import dims, mm, same, whole

pytestmark = pytest.mark.gpu
B, H, F4, F8, U = torch.bfloat16, torch.float16, torch.float32, torch.float64, ref.U


def near(got, want, err):
    h, tiny = ref.half(got.dtype), 2.0 ** -25 if got.dtype is H else 1e-38
    far = (got.to(F8) - want).abs() / (err + h * (want.abs() + err) + tiny)
    assert bool(torch.isfinite(got).all()) and float(far.max()) <= 1.0, float(far.max())


def unit(K):
    """a power of two that gives a sum of K terms a spread of 2 to 4"""
    return 2.0 ** -(round(math.log2(math.sqrt(K * 4 / 9))) - 1)


def check(call, z, z2, bias, res, act, T, outside, R):
    """call(**kw) fills y, z and z2: act(z + bias) + res, and act(z) z2; rows of `outside` stay"""
    slots = z.shape[0]
    live = slice(None) if outside is None else ~outside
    out = lambda dtype: torch.full((slots, R), 77.0, dtype=dtype, device="cuda")  # noqa: E731
    y, kz, kz2 = out(F4), out(T), out(T)
    call(bias=bias, act=act, residual=res, y=y, z=kz)
    zb = z + bias if outside is None else z + bias_of(bias, z, outside)
    want = ref.act(zb.to(F8), act)
    near(y[live], (want + res.to(F8))[live], (8 * U * zb.abs() + U * (want + res.to(F8)).abs())[live])
    same(kz[live], zb[live])
    y16 = out(T)
    call(bias=bias, act=act, residual=None, y=y16, z=None)
    near(y16[live], want[live], (8 * U * zb.abs())[live])
    yg = out(F4)
    call(up=True, act=act, residual=res, y=yg, z=kz, z2=kz2)
    g = ref.act(z.to(F8), act) * z2.to(F8)
    near(yg[live], (g + res.to(F8))[live], (8 * U * (z * z2).abs().to(F8) + U * g.abs() + U * (g + res.to(F8)).abs())[live])
    same(kz[live], z[live])
    same(kz2[live], z2[live])
    if outside is not None:
        for t in (y, kz, kz2, y16, yg):
            assert bool((t[outside] == 77.0).all())


def bias_of(bias, z, outside):
    """the bias of each slot, laid out by the caller"""
    b = torch.zeros_like(z)
    b[~outside] = torch.repeat_interleave(bias, bias_of.counts, 0)
    return b


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_epilogues_dense(ctx, act):
    for i, (n, R, K) in enumerate(cases.DENSE):
        print("%s n %d R %d K %d" % (act, n, R, K), flush=True)
        T = (B, H)[(i + (act == "gelu")) % 2]
        s = unit(K)
        x, W, W2, bias, res = whole(1, n, K, dtype=T), whole(2, R, K, dtype=T) * s, whole(3, R, K, dtype=T) * s, whole(4, R, dtype=F4, most=9) * s, whole(5, n, R, dtype=T, most=9)

        def call(up=None, **kw):
            ctx.matmul(x, W, up=W2 if up else None, **kw)
        check(call, mm(x, W), mm(x, W2), bias, res, act, T, None, R)


@pytest.mark.parametrize("through", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_epilogues_experts(ctx, act, through):
    for i, (n, ne, R, K) in enumerate(cases.EXPERTS):
        print("%s n %d experts %d R %d K %d%s" % (act, n, ne, R, K, " through perm" if through else ""), flush=True)
        T = (H, B)[(i + (act == "gelu")) % 2]
        off, offsets, slots = dims(n, ne)
        topk, s = 3 if through else 1, unit(K)
        x = whole(1, -(-slots // topk), K, dtype=T)
        perm = torch.randperm(x.shape[0] * topk, generator=torch.Generator().manual_seed(2))[:slots].to(torch.int32).cuda() if through else None
        rows = x[perm.long() // topk] if through else x
        W, W2, bias, res = whole(3, ne, R, K, dtype=T) * s, whole(4, ne, R, K, dtype=T) * s, whole(5, ne, R, dtype=F4, most=9) * s, whole(6, slots, R, dtype=T, most=9)
        z, z2 = torch.zeros((slots, R), device="cuda"), torch.zeros((slots, R), device="cuda")
        for e in range(ne):
            if off[e] < off[e + 1]:
                a = slice(off[e], off[e + 1])
                z[a], z2[a] = mm(rows[a], W[e]), mm(rows[a], W2[e])
        outside = torch.ones(slots, dtype=torch.bool, device="cuda")
        outside[off[0]:off[-1]] = False
        bias_of.counts = (offsets[1:] - offsets[:-1]).long()

        def call(up=None, **kw):
            ctx.expert_matmul(x, W, offsets, up=W2 if up else None, perm=perm, topk=topk, **kw)
        check(call, z, z2, bias, res, act, T, outside, R)
        torch.cuda.empty_cache()


@pytest.mark.parametrize("topk", [1, 3])
def test_rows_picked_from_all_that_is_allowed(ctx, topk):
    """x of 2^31 - 2^16 values, close to 4 GiB: rows on both sides of 2^31 bytes and the last ones, picked by every kernel that reads through perm"""
    K = 8192
    xr = (2 ** 31 - 2 ** 16) // K
    x = torch.empty((xr, K), dtype=B, device="cuda")
    x.fill_(3.0)
    at = torch.cat([torch.arange(a, a + 100) for a in (0, 2 ** 31 // (2 * K) - 50, 3 * xr // 4, xr - 100)])
    x[at.cuda()] = whole(1, 400, K)
    for n, ne, R in ((300, 3, 72), (300, 3, 264), (2000, 2, 520), (2000, 2, 4104)):   # few rows / tiles; dW of 128 x 128, few rows, 256 x 256
        print("n %d experts %d R %d topk %d" % (n, ne, R, topk), flush=True)
        g = torch.Generator().manual_seed(n + R)
        row = at[torch.randint(0, 400, (n,), generator=g)]
        row[-1] = xr - 1
        perm = (row * topk + torch.randint(0, topk, (n,), generator=g)).to(torch.int32).cuda()
        cut = [0, n // 3, n] if ne == 2 else [0, 7, n // 2, n]
        offsets = torch.tensor(cut, dtype=torch.int32, device="cuda")
        W, W2, dz, rows = whole(2, ne, R, K), whole(3, ne, R, K), whole(4, n, R), x[row.cuda()]
        y, z, z2 = ctx.expert_matmul(x, W, offsets, up=W2, perm=perm, topk=topk, keep=True, dtype=F4)
        p = ctx.expert_matmul(x, W, offsets, perm=perm, topk=topk, dtype=F4)
        dW = ctx.expert_matmul_grad(dz, x, W, offsets, perm=perm, topk=topk, need_dx=False, dw_dtype=F4)[1]
        for e in range(ne):
            a = slice(cut[e], cut[e + 1])
            w, w2 = mm(rows[a], W[e]), mm(rows[a], W2[e])
            same(p[a], w)
            same(y[a], w * w2)
            same(z[a], w)
            same(z2[a], w2)
            same(dW[e], mm(dz[a].t(), rows[a].t()))
    del x
    torch.cuda.empty_cache()
