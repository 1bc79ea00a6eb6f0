"""GPU: products of Q4_K matrices (fl_kq_matvec_dev with FL_Q4K, and as a format of the device-resident block) against the CPU
oracle, bit for bit: the integer sums are exact and the fp32 chain over the blocks is the same in every kernel, so a row's output
has the same bits whatever n and R. The oracle itself is held to a 64-bit product on the CPU (test_oracle_q4k.py)."""
import ctypes

import numpy as np
import pytest

from oracle import oracle as orc
from tests._q4k import matrix, q8k_rows
from tests.test_q4k_rules import SIZES

pytestmark = pytest.mark.gpu

E, H, KE = 7168, 2048, 8


def product(ctx, w, R, K, q, d):
    import torch
    y = ctx.kq_matvec(orc.Q4K, torch.from_numpy(w).cuda(), R, K, torch.from_numpy(q).cuda(), torch.from_numpy(d).cuda())
    ctx.sync()
    return y.cpu().numpy()


def same(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


# blocks per row: one, under and over a wave's 8, every wave split (1, 2, 3, 4 waves and several passes), the largest
@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 9, 16, 17, 33, 70, 130])
@pytest.mark.parametrize("R,K", [(1, 256), (15, 768), (16, 2048), (33, 2304), (130, 4608), (66, 7168), (257, 1024), (40, 16640)])
def test_products(ctx, R, K, n):
    w = matrix(R + K, R, K)
    q, d, bs = q8k_rows(n, K, seed=K + n)
    print("q4_K R %d K %d n %d" % (R, K, n), flush=True)
    assert same(product(ctx, w, R, K, q, d), orc.matvec_kq(orc.Q4K, w, R, K, q, d, bs))


def test_longest_rows(ctx):
    R, K = 5, 65536
    w = matrix(9, R, K)
    for n in (1, 7, 20):
        q, d, bs = q8k_rows(n, K, seed=n)
        print("q4_K longest n %d" % n, flush=True)
        assert same(product(ctx, w, R, K, q, d), orc.matvec_kq(orc.Q4K, w, R, K, q, d, bs))


def test_extremes(ctx):
    """the largest block sums (every quant 15, scale and min 63, |x| = 127) and zero scales, in every kernel"""
    R, K = 24, 512
    b = np.full((R, K // 256, 144), 0xFF, np.uint8)
    b[..., 0:2] = np.frombuffer(np.float16(0.01).tobytes(), np.uint8)
    b[..., 2:4] = np.frombuffer(np.float16(0.07).tobytes(), np.uint8)
    b[3, :, 4:16] = 0
    w = b.reshape(-1)
    for n in (1, 6, 12, 40):
        q = np.where(np.arange(n)[:, None] % 2 == 0, 127, -127).astype(np.int8) * np.ones((1, K), np.int8)
        q[n - 1, 256:] = 0
        d = np.full((n, K // 256), 0.03, np.float32)
        bs = q.reshape(n, K // 16, 16).sum(axis=2).astype(np.int16)
        print("q4_K extremes n %d" % n, flush=True)
        assert same(product(ctx, w, R, K, q, d), orc.matvec_kq(orc.Q4K, w, R, K, q, d, bs))


def test_non_finite_scales_stay_in_their_rows(ctx):
    """a row of infinite d or NaN d8: its outputs as the oracle's, the others' untouched"""
    R, K = 20, 1024
    w = matrix(12, R, K).reshape(R, -1).copy()
    w[5, 0:2] = np.frombuffer(np.float16(np.inf).tobytes(), np.uint8)
    w = w.reshape(-1)
    for n in (2, 10, 37):
        q, d, bs = q8k_rows(n, K, seed=40 + n)
        d[1, 2] = np.nan
        got, want = product(ctx, w, R, K, q, d), orc.matvec_kq(orc.Q4K, w, R, K, q, d, bs)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])


def test_batch_does_not_change_a_row(ctx):
    """row t of a batch of any size has the bits that it has alone, and a slice of the matrix's rows too"""
    import torch
    R, K, N = 300, 2048, 150
    w = matrix(5, R, K)
    q, d, _ = q8k_rows(N, K, seed=6)
    whole = product(ctx, w, R, K, q, d)
    for n in (1, 2, 4, 7, 15, 16, 31, 64, 65, 128, 129):
        assert same(product(ctx, w, R, K, q[:n], d[:n]), whole[:n]), n
    rb = K // 256 * 144
    for a, b in ((0, 17), (16, 80), (250, 300)):
        assert same(product(ctx, w[a * rb:b * rb], b - a, K, q, d), np.ascontiguousarray(whole[:, a:b])), (a, b)


@pytest.mark.parametrize("n", [1, 6, 24, 130])
def test_unaligned_start_and_untouched_surroundings(ctx, n):
    """a matrix 4 bytes off a 16-byte boundary inside a larger buffer, the output inside another: nothing around it is written"""
    import torch
    R, K = 77, 2048
    w = matrix(21, R, K)
    q, d, bs = q8k_rows(n, K, seed=22)
    buf = torch.zeros(len(w) + 64, dtype=torch.uint8, device="cuda")
    buf[4:4 + len(w)] = torch.from_numpy(w).cuda()
    out = torch.full((n * R + 32,), -7.0, device="cuda")
    ctx.kq_matvec(orc.Q4K, buf[4:4 + len(w)], R, K, torch.from_numpy(q).cuda(), torch.from_numpy(d).cuda(), out[16:16 + n * R])
    ctx.sync()
    o = out.cpu().numpy()
    assert np.all(o[:16] == -7.0) and np.all(o[16 + n * R:] == -7.0)
    assert same(o[16:16 + n * R].reshape(n, R), orc.matvec_kq(orc.Q4K, w, R, K, q, d, bs))


@pytest.mark.parametrize("name", SIZES)
def test_every_kernel(ctx, name):
    """ragged sizes that the launch rule gives each of the kernels for many tokens (test_q4k_rules.py holds it to that), the matrix 4
    bytes off a 16-byte boundary; the largest block sums in three rows and two tokens"""
    import torch
    for R, K, n in SIZES[name]:
        w = matrix(R + 7, R, K).reshape(R, K // 256, 144).copy()
        for r in (0, 17, R - 1):
            w[r, :, 4:] = 0xFF
        w = w.reshape(-1)
        q, d, _ = q8k_rows(n, K, seed=R + n)
        q[0], q[n - 1] = 127, -127
        bs = q.reshape(n, K // 16, 16).sum(axis=2).astype(np.int16)
        buf = torch.zeros(len(w) + 64, dtype=torch.uint8, device="cuda")
        buf[4:4 + len(w)] = torch.from_numpy(w).cuda()
        out = torch.full((n * R + 32,), -7.0, device="cuda")
        print("q4_K %s R %d K %d n %d" % (name, R, K, n), flush=True)
        ctx.kq_matvec(orc.Q4K, buf[4:4 + len(w)], R, K, torch.from_numpy(q).cuda(), torch.from_numpy(d).cuda(), out[16:16 + n * R])
        ctx.sync()
        o = out.cpu().numpy()
        assert np.all(o[:16] == -7.0) and np.all(o[16 + n * R:] == -7.0)
        assert same(o[16:16 + n * R].reshape(n, R), orc.matvec_kq(orc.Q4K, w, R, K, q, d, bs)), (R, K, n)


def test_offsets_past_32_bits(ctx):
    """the last rows of a 4.8 GB matrix, and outputs behind 2^32 bytes of others, as from those rows alone"""
    import torch
    R, K, T = 1200007, 7168, 45
    rb = K // 256 * 144
    tail = matrix(81, T, K)
    w = torch.zeros(R * rb + 1, dtype=torch.uint8, device="cuda")[:R * rb]
    w[(R - T) * rb:] = torch.from_numpy(tail).cuda()
    for n in (1, 5, 40, 1000):
        q, d, bs = q8k_rows(n, K, seed=82 + n)
        print("q4_K 4.8 GB n %d" % n, flush=True)
        y = ctx.kq_matvec(orc.Q4K, w, R, K, torch.from_numpy(q).cuda(), torch.from_numpy(d).cuda())
        ctx.sync()
        want = orc.matvec_kq(orc.Q4K, tail, T, K, q, d, bs)
        assert same(np.ascontiguousarray(y[:, R - T:].cpu().numpy()), want), n
        assert not torch.any(y[:, :R - T]), n
        del y
    del w
    torch.cuda.empty_cache()


def test_refusals(ctx):
    import torch
    from loki_amd import FL_EINVAL, FL_OK, FL_Q4K, lib
    L = lib()
    w = torch.zeros(2 * 144 + 4, dtype=torch.uint8, device="cuda")
    q = torch.zeros((2, 256), dtype=torch.int8, device="cuda"); d = torch.zeros((2, 1), device="cuda"); y = torch.zeros((2, 2), device="cuda")
    P = lambda t, o=0: ctypes.c_void_p(t.data_ptr() + o)   # noqa: E731
    call = lambda R, K, n, wp=None, yp=None: L.fl_kq_matvec_dev(ctx.ctx, FL_Q4K, wp or P(w), R, K, P(q), P(d), n, yp or P(y))   # noqa: E731
    assert call(0, 256, 1) == FL_EINVAL and call(2, 0, 1) == FL_EINVAL and call(2, 300, 1) == FL_EINVAL and call(2, 256, -1) == FL_EINVAL
    assert call(1, 65792, 1) == FL_EINVAL and b"65536" in L.fl_last_error(ctx.ctx)
    assert call(2, 256, 1, wp=P(w, 2)) == FL_EINVAL and b"4-byte" in L.fl_last_error(ctx.ctx)
    big = 1 << 26
    assert call(big, 256, 1) == FL_EINVAL and b"smaller" in L.fl_last_error(ctx.ctx)
    assert L.fl_kq_matvec_dev(ctx.ctx, FL_Q4K, None, 2, 256, P(q), P(d), 1, P(y)) == FL_EINVAL
    assert call((1 << 26) + 1, 256, 1) == FL_EINVAL and call(2, 256, (1 << 19) + 1) == FL_EINVAL and b"2^19" in L.fl_last_error(ctx.ctx)
    assert L.fl_kq_matvec_dev(ctx.ctx, FL_Q4K, P(w), 2, 256, P(q, 4), P(d), 1, P(y)) == FL_EINVAL and b"aligned" in L.fl_last_error(ctx.ctx)
    assert call(2, 256, 1, yp=P(y, 2)) == FL_EINVAL
    assert call(2, 256, 0) == FL_OK and call(2, 256, 2) == FL_OK
    ctx.sync()


# ---------------------------------------------------------------- as a format of the block
def random_matrix(fmt, R, K, seed):
    """device bytes of a matrix of the format, its scales small"""
    import torch
    from tests.test_gpu_kquant import KQ_BLOCK
    bs, od, om = {**KQ_BLOCK, orc.Q4K: (144, 0, 2)}[fmt]
    g = torch.Generator(device="cuda").manual_seed(seed)
    b = torch.randint(0, 256, (R * (K // 256), bs), dtype=torch.uint8, device="cuda", generator=g)
    for off in (od, om):
        if off is not None:
            v = torch.randint(0x0C00, 0x1C00, (b.shape[0],), dtype=torch.int32, device="cuda", generator=g).to(torch.int16)
            b[:, off:off + 2] = v.view(torch.uint8).view(-1, 2)
    return b.view(-1)


def test_layer_of_many_rows(ctx):
    """fl_moe_layer's shared Q4_K matrices on the tiled kernels (rows enough for them): the shared expert's part, formed by the
    products and Q8_K quantisation of their own, is what the block leaves in o's last rows, bit for bit; on the GEMM path and the
    per-pass one (second stream)"""
    import torch
    from loki_amd import FL_Q4K, MoeLayerWeights, lib
    from tests._helpers import make_x
    ne, n = 16, 300
    base = MoeLayerWeights.synthetic(ctx, 9190, n_exp=ne)
    sg, su, sd = (random_matrix(FL_Q4K, r, k, 9191 + i) for i, (r, k) in enumerate(((H, E), (H, E), (E, H))))
    layer = MoeLayerWeights(base.gate_inp, base.probs_b, base.gate, base.up, base.down, sg, su, sd, n_exp=ne)
    x = make_x(ctx, n, seed=9192)
    xq, xd = ctx.quant_q8k(x)
    gate, up = (ctx.kq_matvec(FL_Q4K, m, H, E, xq, xd) for m in (sg, su))
    ctx.sync()
    gate, up = gate.cpu().numpy(), up.cpu().numpy()
    ctx.set_routing(8, 4, 8, 2.5)
    ctx.set_layer_formats(4, orc.Q4K, orc.Q4K, orc.Q4K)
    try:
        ys = []
        for mfma in (1, 0):
            lib().fl_set_prefill_mfma(ctx.ctx, mfma)
            ys.append(ctx.moe_layer(layer, x))
            ctx.sync()
            h = ctx.d2h(ctx.debug().h, (n * KE + n, H), np.float32)[n * KE:]
            hq, hd = ctx.quant_q8k(torch.from_numpy(h).cuda())
            down = ctx.kq_matvec(FL_Q4K, sd, E, H, hq, hd)
            ctx.sync()
            o = ctx.d2h(ctx.debug().o, (n * KE + n, E), np.float32)[n * KE:]
            assert same(o, down.cpu().numpy())
            if mfma:
                first = h
            assert same(h, first)
            assert same(h[[0, 7, n - 1]], np.stack([orc.silu(gate[t]) * up[t] for t in (0, 7, n - 1)]))
    finally:
        lib().fl_set_prefill_mfma(ctx.ctx, 1)
        ctx.set_layer_formats()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fm", [(orc.Q4K, orc.Q4K, orc.Q4K, orc.Q4K), (orc.Q4K, orc.Q5K, orc.Q5K, orc.Q6K), (orc.Q2K, orc.Q4K, orc.Q5K, orc.Q4K),
                                (orc.Q4K, 4, 4, 4)], ids=["all", "down", "shared", "down_iq2_shared"])
def test_layer_formats(ctx, fm):
    """fl_moe_layer with Q4_K routed down and shared matrices at decode and prefill sizes: picks bit-identical, outputs within the
    K-quants' bar of the oracle, and each row's bits the same in a batch and alone (the per-pass kernels and the GEMMs)"""
    import torch
    from loki_amd import MoeLayerWeights
    from tests._helpers import host_matrix, make_x
    from tests.test_gpu_kquant import KQ_BLOCK, bar_close
    ne = 16
    block = {**KQ_BLOCK, orc.Q4K: (144, 0, 2)}

    def bytes_of(fmt, R, K, seed):
        bs, od, om = block[fmt]
        g = torch.Generator(device="cuda").manual_seed(seed)
        b = torch.randint(0, 256, (R * (K // 256), bs), dtype=torch.uint8, device="cuda", generator=g)
        for off in (od, om):
            if off is not None:
                v = torch.randint(0x0C00, 0x1C00, (b.shape[0],), dtype=torch.int32, device="cuda", generator=g).to(torch.int16)
                b[:, off:off + 2] = v.view(torch.uint8).view(-1, 2)
        return b.view(-1)

    base = MoeLayerWeights.synthetic(ctx, 9090, n_exp=ne)
    down = base.down if fm[0] == 4 else bytes_of(fm[0], ne * E, H, 9091)
    sh = [t if f == 4 else bytes_of(f, r, k, 9092 + i)
          for i, (f, (r, k), t) in enumerate(zip(fm[1:], ((H, E), (H, E), (E, H)), (base.sh_gate, base.sh_up, base.sh_down)))]
    layer = MoeLayerWeights(base.gate_inp, base.probs_b, base.gate, base.up, down, *sh, n_exp=ne)
    W, b = layer.gate_inp.cpu().numpy(), layer.probs_b.cpu().numpy()
    mb = E * (H // 256) * block[fm[0]][0]
    gate = {e: host_matrix(ctx, layer.expert_slice("gate", e), H, E) for e in range(ne)}
    up = {e: host_matrix(ctx, layer.expert_slice("up", e), H, E) for e in range(ne)}
    dn = {e: down[e * mb:(e + 1) * mb].cpu().numpy() for e in range(ne)}
    shh = [host_matrix(ctx, m, r, k) if f == 4 else m.cpu().numpy() for f, m, (r, k) in zip(fm[1:], sh, ((H, E), (H, E), (E, H)))]
    ctx.set_routing(8, 4, 8, 2.5)
    ctx.set_layer_formats(*fm)
    try:
        x = make_x(ctx, 40, seed=9100)
        xs = x.cpu().numpy()
        _, _, so, wo = orc.router(W, b, xs)
        want = orc.moe_experts(xs, so, wo, gate, up, dn, *shh, n_exp=ne, fmts=fm)["y"]
        for n in (1, 3, 8, 9, 40):
            print("q4_K layer %s n %d" % (fm, n), flush=True)
            y = ctx.moe_layer(layer, x[:n].contiguous())
            ctx.sync()
            assert np.array_equal(ctx.d2h(ctx.debug().sel, (n, KE), np.int32), so[:n])
            ok, err = bar_close(y.cpu().numpy(), want[:n])
            assert ok, (n, err)
    finally:
        ctx.set_layer_formats()
    torch.cuda.empty_cache()


def test_gguf_layer(ctx, tmp_path):
    """a layer of Q4_K routed down and shared matrices from a GGUF file: loaded tiled it runs through fl_moe_layer within the K-quants'
    bar of the oracle; the layout that fl_moe reads refuses the format"""
    import torch
    from loki_amd import FL_LAYOUT_GGML, FL_LAYOUT_TILED, Gguf, LokiError, lib
    from tests import _gguf
    from tests.golden import gen
    from tests.test_gpu_gguf import layer_tensors
    from tests.test_gpu_kquant import bar_close
    ne, n = 16, 20
    W, b, gate, up, _, _ = gen.layer(302, ne, E, H)
    down = [matrix(303 + e, E, H) for e in range(ne)]
    sh = (matrix(330, H, E), matrix(331, H, E), matrix(332, E, H))
    path = str(tmp_path / "q4.gguf")
    _gguf.write(path, layer_tensors(4, W, b, gate, up, down, sh, ["IQ2_XXS", "IQ2_XXS", "Q4_K", "Q4_K", "Q4_K", "Q4_K"]))
    g = Gguf(path)
    gl = ctx.load_gguf_layer(g, 4, FL_LAYOUT_TILED)
    try:
        fm = (gl.fmt_down, gl.fmt_sh_gate, gl.fmt_sh_up, gl.fmt_sh_down)
        assert fm == (orc.Q4K,) * 4
        ctx.set_experts(ne); ctx.set_routing(8, 4, 8, 2.5); ctx.set_layer_formats(*fm)
        x = gen.uniform(12, 304, (n, E), 2.0)
        xt = torch.from_numpy(x).cuda(); y = torch.empty_like(xt)
        ctx.check(lib().fl_moe_layer(ctx.ctx, ctypes.byref(gl.L), ctypes.c_void_p(xt.data_ptr()), n, ctypes.c_void_p(y.data_ptr())))
        ctx.sync()
        _, _, so, wo = orc.router(W, b, x, 8, 4, 8, 2.5)
        ok, err = bar_close(y.cpu().numpy(), orc.moe_experts(x, so, wo, gate, up, down, *sh, n_exp=ne, fmts=fm)["y"])
        assert ok, err
        with pytest.raises(LokiError, match="Q4_K"):
            ctx.load_gguf_layer(g, 4, FL_LAYOUT_GGML)
    finally:
        ctx.set_layer_formats(); ctx.set_experts()
        ctx.free_gguf_layer(gl)
        g.close()


# ---------------------------------------------------------------- graphs and streams
def test_captured_products_outlive_a_larger_scratch(ctx):
    """two captured products of one context (tiled: their scratch is the context's), an eager one that outgrows the scratch between
    their replays, and changed rows: every replay has the bits of its rows' eager product"""
    import torch
    from loki_amd import Context, lib
    R, K = 2049, 1024
    w = torch.from_numpy(matrix(61, R, K)).cuda()
    rows = [[torch.from_numpy(a).cuda() for a in q8k_rows(200, K, seed=62 + i)[:2]] for i in range(3)]
    big = [torch.from_numpy(a).cuda() for a in q8k_rows(3000, K, seed=66)[:2]]
    want = [ctx.kq_matvec(orc.Q4K, w, R, K, q, d).clone() for q, d in rows]
    want_big = ctx.kq_matvec(orc.Q4K, w, R, K, *big)
    ctx.sync()
    c = Context()
    try:
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        c.check(lib().fl_set_stream(c.ctx, side.cuda_stream))
        ins = [[t.clone() for t in rows[0]] for _ in range(2)]
        outs = [torch.empty((200, R), device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            c.kq_matvec(orc.Q4K, w, R, K, *ins[0], outs[0])   # (the scratch is allocated here, before the captures)
        torch.cuda.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for i, g in enumerate(graphs):
            with torch.cuda.graph(g, stream=side):
                c.kq_matvec(orc.Q4K, w, R, K, *ins[i], outs[i])
        for rep in range(3):
            for i, g in enumerate(graphs):
                pick = (rep + 2 * i) % 3
                for dst, src in zip(ins[i], rows[pick]):
                    dst.copy_(src)
                outs[i].fill_(-1.0)
                torch.cuda.synchronize()
                with torch.cuda.stream(side):
                    g.replay()
                    y = c.kq_matvec(orc.Q4K, w, R, K, *big)
                torch.cuda.synchronize()
                assert torch.equal(outs[i].view(torch.int32), want[pick].view(torch.int32)), (rep, i)
                assert torch.equal(y.view(torch.int32), want_big.view(torch.int32)), (rep, i)
        del graphs, g
    finally:
        torch.cuda.synchronize()
        c.close()


def test_two_contexts_at_once(ctx):
    """products on two contexts and streams in flight together, each with its own scratch: the bits that they have alone"""
    import torch
    from loki_amd import Context, lib
    R, K = 7168, 2048
    ws = [torch.from_numpy(matrix(71 + i, R, K)).cuda() for i in range(2)]
    rows = [[torch.from_numpy(a).cuda() for a in q8k_rows(300, K, seed=73 + i)[:2]] for i in range(2)]
    want = [ctx.kq_matvec(orc.Q4K, ws[i], R, K, *rows[i]) for i in range(2)]
    ctx.sync()
    cs, streams = [Context(), Context()], [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        for c, s in zip(cs, streams):
            c.check(lib().fl_set_stream(c.ctx, s.cuda_stream))
        outs = [[torch.full((300, R), -1.0, device="cuda") for _ in range(6)] for _ in range(2)]
        torch.cuda.synchronize()
        for k in range(6):
            for i in range(2):
                cs[i].kq_matvec(orc.Q4K, ws[i], R, K, *rows[i], outs[i][k])
        torch.cuda.synchronize()
        assert all(torch.equal(o.view(torch.int32), want[i].view(torch.int32)) for i in range(2) for o in outs[i])
    finally:
        torch.cuda.synchronize()
        for c in cs:
            c.close()
