"""GPU: fl_moe_layer's routed down in Q4_K with many slots an expert (several groups of a kernel's tokens, the last one not full) and with
one expert that every row picks: each expert's part of o has the bits of its matrix's product with its slots' Q8_K rows."""
import numpy as np
import pytest

from oracle import oracle as orc
from tests.test_gpu_q4k import E, H, KE, random_matrix, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,ne,hot", [(49, 16, None), (300, 32, [5]), (1101, 16, None), (1101, 64, [0, 63])])
def test_every_slot_of_an_expert(ctx, n, ne, hot):
    import torch
    from loki_amd import FL_Q4K, MoeLayerWeights, lib
    from tests._helpers import make_x
    base = MoeLayerWeights.synthetic(ctx, 9290, n_exp=ne, hot=hot, hot_bias=4.0)
    down = random_matrix(FL_Q4K, ne * E, H, 9291)
    layer = MoeLayerWeights(base.gate_inp, base.probs_b, base.gate, base.up, down, base.sh_gate, base.sh_up, base.sh_down, n_exp=ne)
    x = make_x(ctx, n, seed=9292)
    mb, P = E * (H // 256) * 144, n * KE
    ctx.set_routing(8, 4, KE, 2.5)
    ctx.set_layer_formats(orc.Q4K, 4, 4, 4)
    try:
        first = None
        for mfma in (1, 0):
            print("routed q4_K n %d ne %d mfma %d" % (n, ne, mfma), flush=True)
            lib().fl_set_prefill_mfma(ctx.ctx, mfma)
            y = ctx.moe_layer(layer, x)
            ctx.sync()
            g = ctx.debug()
            off = ctx.d2h(g.offsets, (ne + 1,), np.int32)
            sel = ctx.d2h(g.sel, (n, KE), np.int32)
            o = ctx.d2h(g.o, (P, E), np.float32)
            hq, hd = torch.from_numpy(ctx.d2h(g.hq, (P, H), np.int8)).cuda(), torch.from_numpy(ctx.d2h(g.hd, (P, H // 256), np.float32)).cuda()
            counts = np.bincount(sel.ravel(), minlength=ne)
            assert np.array_equal(np.diff(off), counts)
            assert hot is None or all(counts[e] == n for e in hot)
            for e in np.nonzero(counts)[0]:
                a, b = int(off[e]), int(off[e + 1])
                want = ctx.kq_matvec(FL_Q4K, down[e * mb:(e + 1) * mb], E, H, hq[a:b], hd[a:b])
                ctx.sync()
                assert same(o[a:b], want.cpu().numpy()), e
            y = y.cpu().numpy()
            if first is None:
                first = y
            assert same(y, first)
    finally:
        lib().fl_set_prefill_mfma(ctx.ctx, 1)
        ctx.set_layer_formats()
    torch.cuda.empty_cache()
