"""Three operators around the MoE layer, as cases that can be timed and checked.

  q4          Context.kq_matvec with FL_Q4K: y = W x for a matrix in 4-bit blocks with 6-bit group scales and mins, on Q8_K rows
  balance     Context.balance_loss (and balance_loss_grad): per-expert counts and the sequence-wise balance loss of routed rows
  route_grad  Context.route_grad: the router's backward pass, to the logits, the router weight and the rows

Q4_K: a block is 256 weights in 144 bytes = fp16 d, fp16 dmin, 12 bytes of 6-bit scales s_j and mins m_j (8 sub-blocks of 32),
128 bytes of quants; weight = d s_j q - dmin m_j. Q8_K rows: int8 q and an fp32 d per 256 values.
Balance: p = sigmoid(z) / sum sigmoid(z) per row, P_e the mean of p_e over the sequence's T rows, f_e = n_exp c_e / (topk T)
with c_e the picks of expert e, loss = alpha sum_e f_e P_e per sequence, the counts taken as constants in the gradient.
Router: w_k = scale s_k / max(sum_j s_j, 2^-14) over the row's picks, s = sigmoid(z), z = x W^T."""
import math

import torch

own = False

SCALE, CLAMP = 2.5, 2.0 ** -14   # of the routing weights
ALPHA = 1e-4                     # of the balance loss
E = 7168


def listed():
    return [
        # a token through the smallest matrix of a layer (7168 -> 2048), and through a vocabulary-sized one
        {"name": "q4_token", "op": "q4", "n": 1, "R": 2048, "K": 7168},
        {"name": "q4_token_head", "op": "q4", "n": 1, "R": 131072, "K": 7168},
        # a batch of six users or drafted tokens; a short question through a wide down projection
        {"name": "q4_batch_6", "op": "q4", "n": 6, "R": 7168, "K": 2048},
        {"name": "q4_prompt_37", "op": "q4", "n": 37, "R": 7168, "K": 16384},
        # prompt chunks, an odd one and a large one
        {"name": "q4_prompt_501", "op": "q4", "n": 501, "R": 7000, "K": 7168},
        {"name": "q4_prompt_2048", "op": "q4", "n": 2048, "R": 16384, "K": 7168},
        # a short sequence's loss alone; a padded batch of ragged sequences; a training batch, both with the gradient
        {"name": "balance_70", "op": "balance", "n": 70, "nseq": 1, "ne": 256, "topk": 8, "pad": 0, "grad": False},
        {"name": "balance_4100_ragged", "op": "balance", "n": 4100, "nseq": 7, "ne": 256, "topk": 8, "pad": 90, "grad": True},
        {"name": "balance_65536", "op": "balance", "n": 65536, "nseq": 16, "ne": 256, "topk": 8, "pad": 0, "grad": True},
        # the router's backward pass: a few rows, an odd batch over 64 experts, a training batch
        {"name": "route_grad_48", "op": "route_grad", "n": 48, "ne": 256, "topk": 8, "E": E},
        {"name": "route_grad_1001", "op": "route_grad", "n": 1001, "ne": 64, "topk": 6, "E": 2048},
        {"name": "route_grad_8192", "op": "route_grad", "n": 8192, "ne": 256, "topk": 8, "E": E},
    ]


def draw(rng):
    spread = lambda lo, hi: max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo - 0.49), math.log(hi + 0.49))))))  # noqa: E731
    op = rng.choice(["q4", "q4", "q4", "balance", "balance", "route_grad", "route_grad"])
    if op == "q4":
        n, K = spread(1, 2048), 256 * spread(1, 64)
        most = min(131072 * 7168 // K, 2048 * 16384 * 7168 // (n * K))
        return {"op": op, "n": n, "R": spread(64, max(64, min(131072, most))), "K": K}
    ne, topk = rng.choice([256, 256, 160, 64, rng.randint(16, 255)]), rng.choice([8, 8, 6, 2])
    if op == "balance":
        n = spread(8, 65536)
        return {"op": op, "n": n, "nseq": spread(1, min(64, n)), "ne": ne, "topk": topk, "pad": rng.choice([0, 0, n // 9]), "grad": rng.random() < 0.7}
    return {"op": op, "n": spread(1, 8192), "ne": ne, "topk": topk, "E": 1024 * rng.randint(1, 7)}


# ------------------------------------------------------------------------------------------------ inputs
def q4_inputs(case, g):
    """Random quants and scales, centred as a quantised weight's are; normal rows in Q8_K."""
    n, R, K = case["n"], case["R"], case["K"]
    nb = K // 256
    words = torch.randint(-(1 << 63), (1 << 63) - 1, (R * nb * 18,), dtype=torch.int64, device="cuda", generator=g)
    b = words.view(torch.uint8).view(R * nb, 144)
    d = 1.4e-4 * (0.5 + torch.rand(R * nb, device="cuda", generator=g))
    m = 7.5 * d * (0.8 + 0.4 * torch.rand(R * nb, device="cuda", generator=g))
    b[:, 0:2] = d.half().view(torch.uint8).view(-1, 2)
    b[:, 2:4] = m.half().view(torch.uint8).view(-1, 2)
    x = torch.randn((n, nb, 256), device="cuda", generator=g)
    xd = x.abs().amax(2) / 127
    q = torch.round(x / xd[:, :, None]).clamp_(-127, 127).to(torch.int8)
    return {"w": b.view(-1), "q": q.view(n, K), "d": xd.contiguous()}


def routed(case, g):
    """Logits of routed rows with experts of unequal favour, and their picks (top-k of the biased scores)."""
    n, ne = case["n"], case["ne"]
    z = 1.7 * torch.randn((n, ne), device="cuda", generator=g) + 0.5 * torch.randn(ne, device="cuda", generator=g)
    bias = 0.05 * torch.randn(ne, device="cuda", generator=g)
    sel = torch.topk(torch.sigmoid(z) + bias, case["topk"], dim=1).indices.to(torch.int32)
    return z, sel


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)
    if case["op"] == "q4":
        return {"case": case, **q4_inputs(case, g)}
    z, sel = routed(case, g)
    s = {"case": case, "z": z, "sel": sel}
    n, ne = case["n"], case["ne"]
    if case["op"] == "balance":
        rows = n - case["pad"]   # the batch's last rows belong to no sequence
        cuts = torch.sort(torch.randint(0, rows + 1, (case["nseq"] - 1,), device="cuda", generator=g)).values
        ends = torch.tensor([0, rows], device="cuda")
        s["seq"] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
        s["gloss"] = 0.5 + torch.rand(case["nseq"], device="cuda", generator=g)
        return s
    s["W"] = 0.02 * torch.randn((ne, case["E"]), device="cuda", generator=g)
    s["x"] = torch.randn((n, case["E"]), device="cuda", generator=g)
    s["dw"] = 1e-3 * torch.randn((n, case["topk"]), device="cuda", generator=g)
    s["dz"] = 1e-6 * torch.randn((n, ne), device="cuda", generator=g)   # a balance loss's gradient of the logits
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
_contexts = {}


def context(topk):
    """The program's context for this routing rule, on torch's current stream."""
    import loki_amd
    key = (topk, torch.cuda.current_stream().cuda_stream)
    if key not in _contexts:
        c = loki_amd.Context()
        c.set_routing(1, 1, topk, SCALE)
        _contexts[key] = c
    return _contexts[key]


def run_own(s):
    import loki_amd
    case = s["case"]
    c = context(case.get("topk", 8))
    if case["op"] == "q4":
        return c.kq_matvec(loki_amd.FL_Q4K, s["w"], case["R"], case["K"], s["q"], s["d"])
    if case["op"] == "balance":
        counts, loss = c.balance_loss(s["z"], s["sel"], ALPHA, seq=s["seq"])
        if not case["grad"]:
            return counts, loss
        return counts, loss, c.balance_loss_grad(s["z"], counts, case["topk"], ALPHA, seq=s["seq"], gloss=s["gloss"])
    return c.route_grad(s["W"], s["x"], s["z"], s["sel"], s["dw"], dz=s["dz"])


# ------------------------------------------------------------------------------------------------ plain forms
def q4_weights(w, R, K, dtype):
    """The matrix in `dtype`, dequantised."""
    b = w.view(-1, 144)
    d, m = b[:, 0:4].contiguous().view(torch.float16).to(dtype).unbind(1)
    s = b[:, 4:16]
    lo, mid, hi = s[:, 0:4], s[:, 4:8], s[:, 8:12]
    sc = torch.cat([lo & 63, (hi & 15) | ((lo >> 6) << 4)], 1).to(dtype) * d[:, None]
    mn = torch.cat([mid & 63, (hi >> 4) | ((mid >> 6) << 4)], 1).to(dtype) * m[:, None]
    qs = b[:, 16:].reshape(-1, 4, 32)
    q = torch.stack([qs & 15, qs >> 4], 2).view(-1, 8, 32)   # sub-block 2 j: the low nibbles of bytes 32 j .., 2 j + 1: the high ones
    return (q.to(dtype) * sc[:, :, None] - mn[:, :, None]).view(R, K)


def run_plain(s):
    case = s["case"]
    if case["op"] == "q4":
        n, R, K = case["n"], case["R"], case["K"]
        x = (s["q"].view(n, -1, 256).float() * s["d"][:, :, None]).view(n, K)
        return x @ q4_weights(s["w"], R, K, torch.float32).t()
    z, sel = s["z"], s["sel"].long()
    n, ne, topk = case["n"], case["ne"], case["topk"]
    sg = torch.sigmoid(z)
    if case["op"] == "balance":
        nseq = case["nseq"]
        row = torch.arange(n, device=z.device)
        at = torch.bucketize(row, s["seq"][1:].long(), right=True)   # the row's sequence; nseq: none
        T = (s["seq"][1:] - s["seq"][:-1]).float().clamp_(min=1)
        counts = torch.zeros((nseq + 1) * ne, dtype=torch.int32, device=z.device)
        ones = torch.ones(n * topk, dtype=torch.int32, device=z.device)
        counts = counts.scatter_add_(0, (at[:, None] * ne + sel).view(-1), ones).view(nseq + 1, ne)[:nseq].contiguous()
        p = sg / sg.sum(1, keepdim=True)
        P = torch.zeros((nseq + 1, ne), device=z.device).index_add_(0, at, p)[:nseq] / T[:, None]
        f = counts.float() * (ne / topk) / T[:, None]
        loss = ALPHA * (f * P).sum(1)
        if not case["grad"]:
            return counts, loss
        zero = torch.zeros((1, ne), device=z.device)
        fr = torch.cat([f, zero])[at]
        k = torch.cat([s["gloss"] * ALPHA / T, zero[0, :1]])[at][:, None]
        return counts, loss, k * p * (1 - sg) * (fr - (fr * p).sum(1, keepdim=True))
    sk = torch.gather(sg, 1, sel)
    S = sk.sum(1, keepdim=True)
    dw = s["dw"]
    ds = torch.where(S > CLAMP, SCALE / S * (dw - (dw * sk).sum(1, keepdim=True) / S), SCALE / CLAMP * dw)
    dz = s["dz"].scatter_add(1, sel, ds * sk * (1 - sk))
    return dz, dz.t() @ s["x"], dz @ s["W"]


def run(state):
    return run_own(state) if own else run_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n = case["n"]
    if case["op"] == "q4":
        R, K = case["R"], case["K"]
        return {"bytes": R * (K // 256) * 144 + n * K + 4 * n * (K // 256) + 4 * n * R, "flops": 2 * n * R * K}
    ne, topk = case["ne"], case["topk"]
    if case["op"] == "balance":
        nseq, rows = case["nseq"], n - case["pad"]
        read = 4 * rows * (ne + topk) + 4 * (nseq + 1)
        out = 4 * nseq * (ne + 1)
        more = 4 * n * ne + 4 * nseq if case["grad"] else 0
        return {"bytes": read + out + more, "flops": rows * ne * (14 if case["grad"] else 8)}
    e = case["E"]
    return {"bytes": 4 * (2 * n * e + 2 * ne * e + 3 * n * ne + 2 * n * topk), "flops": 4 * n * ne * e}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "q4":
        n, R, nb = case["n"], case["R"], case["K"] // 256
        x = s["q"].view(n, nb, 256).to(f8) * s["d"].to(f8)[:, :, None]
        y = torch.empty((n, R), dtype=f8, device="cuda")
        blocks = s["w"].view(R, nb, 144)
        for r in range(0, R, 8192):   # some rows at a time, for memory's sake
            b = blocks[r:r + 8192]
            dm = b[:, :, :4].contiguous().view(torch.float16).to(f8)
            sb = b[:, :, 4:16].to(torch.int32)
            acc = torch.zeros((n, b.shape[0]), dtype=f8, device="cuda")
            for j in range(8):   # sub-block j: 32 weights with one scale and one min
                if j < 4:
                    sc, mn = sb[:, :, j] & 63, sb[:, :, 4 + j] & 63
                else:
                    sc = (sb[:, :, 4 + j] & 15) + 16 * (sb[:, :, j - 4] >> 6)
                    mn = (sb[:, :, 4 + j] >> 4) + 16 * (sb[:, :, j] >> 6)
                by = b[:, :, 16 + 32 * (j // 2):48 + 32 * (j // 2)]
                q = (by >> 4 if j % 2 else by & 15).to(f8)
                w = (dm[:, :, 0] * sc)[:, :, None] * q - (dm[:, :, 1] * mn)[:, :, None]
                acc += x[:, :, 32 * j:32 * j + 32].reshape(n, -1) @ w.reshape(w.shape[0], -1).t()
            y[:, r:r + 8192] = acc
        return y
    z, sel = s["z"].to(f8), s["sel"].long()
    n, ne, topk = case["n"], case["ne"], case["topk"]
    sg = 1 / (1 + torch.exp(-z))
    if case["op"] == "balance":
        cuts = s["seq"].tolist()
        counts = torch.zeros((case["nseq"], ne), dtype=torch.int32, device="cuda")
        loss = torch.zeros(case["nseq"], dtype=f8, device="cuda")
        dz = torch.zeros((n, ne), dtype=f8, device="cuda")
        for i in range(case["nseq"]):
            a, b = cuts[i], cuts[i + 1]
            if a == b:
                continue
            counts[i] = torch.bincount(sel[a:b].reshape(-1), minlength=ne).to(torch.int32)
            f = counts[i].to(f8) * ne / (topk * (b - a))
            p = sg[a:b] / sg[a:b].sum(1, keepdim=True)
            loss[i] = ALPHA * torch.dot(f, p.mean(0))
            dz[a:b] = s["gloss"][i].to(f8) * ALPHA / (b - a) * p * (1 - sg[a:b]) * (f[None] - (p @ f)[:, None])
        return (counts, loss, dz) if case["grad"] else (counts, loss)
    sk = sg.gather(1, sel)
    S, dw = sk.sum(1, keepdim=True), s["dw"].to(f8)
    ds = (dw - (dw * sk / S).sum(1, keepdim=True)) * SCALE / S
    flat = S <= CLAMP
    ds = torch.where(flat, dw * SCALE / CLAMP, ds)
    dz = s["dz"].to(f8)
    for k in range(topk):
        dz = dz.scatter_add(1, sel[:, k:k + 1], (ds * sk * (1 - sk))[:, k:k + 1])
    return dz, dz.t() @ s["x"].to(f8), dz @ s["W"].to(f8)
