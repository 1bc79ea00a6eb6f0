"""Operators that train and run a layer's matrices in bfloat16 or float16, as cases that can be timed and checked.

  matmul        Context.matmul: y = act(x W^T + bias) + residual, or the gated form silu(x W^T) * (x U^T)
  matmul_grad   Context.act_grad and matmul_grad: its backward pass, to the pre-activations, the bias, the rows and the matrix
  experts       Context.expert_matmul: the same product grouped by expert, ragged, its rows picked through dispatch()'s order
  experts_grad  Context.act_grad and expert_matmul_grad: its backward pass, each expert's matrix from its own rows
  combine       Context.combine and combine_grad: a row's picks summed under the routing weights, and the gradients of both

Slots are (row, pick) pairs sorted by expert: expert e has slots offsets[e] .. offsets[e + 1] - 1, perm[slot] is its pair (row * topk +
pick) and inv the other way round; pairs that no expert takes have no slot, and the slots behind the last expert's stay as they were.
act: silu(z) = z s(z), gelu(z) = z s(2 sqrt(2 / pi) (z + 0.044715 z^3)), s(t) = 1 / (1 + e^-t)."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GELU = 2 * math.sqrt(2 / math.pi)
E, H = 7168, 2048


def listed():
    dense = {"type": "bf16", "act": "", "gated": False, "bias": False, "residual": False, "out32": False}
    moe = {"type": "bf16", "act": "", "gated": False, "keep": False, "drop": 0.0}
    return [
        # a token through the smallest matrix of a layer, added to the row; a ragged prompt through a gated dense layer; a batch through its widest matrix
        {"name": "matmul_token", "op": "matmul", "n": 1, "R": E, "K": H, **dense, "bias": True, "residual": True},
        {"name": "matmul_prompt_501", "op": "matmul", "n": 501, "R": 7000, "K": E, **dense, "type": "f16", "act": "silu", "gated": True},
        {"name": "matmul_8192", "op": "matmul", "n": 8192, "R": 16384, "K": E, **dense, "act": "gelu", "bias": True},
        # the shared expert's down projection on an odd batch, the sums in float32; a dense layer's training batch
        {"name": "matmul_grad_501", "op": "matmul_grad", "n": 501, "R": E, "K": H, **dense, "bias": True, "out32": True},
        {"name": "matmul_grad_8192", "op": "matmul_grad", "n": 8192, "R": 16384, "K": E, **dense, "act": "gelu", "bias": True},
        # one token's eight experts, gate and up; rows of 64 small experts, as a training step keeps them; a prompt's down products
        {"name": "experts_token", "op": "experts", "n": 1, "ne": 256, "topk": 8, "R": H, "K": E, **moe, "act": "silu", "gated": True},
        {"name": "experts_1001", "op": "experts", "n": 1001, "ne": 64, "topk": 6, "R": 1024, "K": 2048, **moe, "type": "f16", "act": "silu", "gated": True, "keep": True, "drop": 0.1},
        {"name": "experts_8192_down", "op": "experts", "n": 8192, "ne": 256, "topk": 8, "R": E, "K": H, **moe},
        # the backward pass of those small experts (both matrices), and of a training batch's down products
        {"name": "experts_grad_1001", "op": "experts_grad", "n": 1001, "ne": 64, "topk": 6, "R": 1024, "K": 2048, **moe, "type": "f16", "act": "silu", "gated": True, "drop": 0.1},
        {"name": "experts_grad_4096_down", "op": "experts_grad", "n": 4096, "ne": 256, "topk": 8, "R": E, "K": H, **moe},
        # a decode batch, and a training batch
        {"name": "combine_6", "op": "combine", "n": 6, "ne": 256, "topk": 8, "R": E, "type": "bf16", "residual": True, "drop": 0.0},
        {"name": "combine_8192", "op": "combine", "n": 8192, "ne": 256, "topk": 8, "R": E, "type": "bf16", "residual": True, "drop": 0.05},
    ]


def draw(rng):
    spread = lambda lo, hi: max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo - 0.49), math.log(hi + 0.49))))))  # noqa: E731
    op = rng.choice(["matmul", "matmul", "matmul_grad", "experts", "experts", "experts_grad", "combine"])
    kind, act = rng.choice(["bf16", "bf16", "f16"]), rng.choice(["", "silu", "gelu"])
    if op in ("matmul", "matmul_grad"):
        n, K = spread(1, 8192), 8 * spread(8, 2048)
        most = min((1 << 31) // K, 8192 * 16384 * 7168 // (n * K)) // 8
        gated = rng.random() < 0.3
        R = 8 * spread(8, max(8, min(16384, most // (2 if gated else 1))))
        return {"op": op, "n": n, "R": R, "K": K, "type": kind, "act": "silu" if gated else act, "gated": gated, "bias": not gated and rng.random() < 0.5,
                "residual": rng.random() < 0.3, "out32": rng.random() < 0.3 and (op == "matmul" or not (act or gated))}
    ne, topk = rng.choice([256, 160, 64, rng.randint(4, 255)]), rng.choice([8, 6, 2, 1])
    topk, drop = min(topk, ne), rng.choice([0.0, 0.0, 0.1])
    if op == "combine":
        return {"op": op, "n": spread(1, 8192), "ne": ne, "topk": topk, "R": 8 * spread(8, 896), "type": kind, "residual": rng.random() < 0.5, "drop": drop}
    gated = rng.random() < 0.5
    R, K = 8 * spread(16, 256), 8 * spread(16, 896)
    if not gated and rng.random() < 0.5:
        R, K = K, R
    return {"op": op, "n": spread(1, 4096), "ne": ne, "topk": topk, "R": R, "K": K, "type": kind, "act": "silu" if gated else act, "gated": gated,
            "keep": op == "experts" and rng.random() < 0.4, "drop": drop}


# ------------------------------------------------------------------------------------------------ inputs
def routed(case, g):
    """Picks of routed rows, experts of unequal favour, and their order by expert as a dispatch gives it."""
    n, ne, topk = case["n"], case["ne"], case["topk"]
    z = 1.7 * torch.randn((n, ne), device="cuda", generator=g) + 0.5 * torch.randn(ne, device="cuda", generator=g)
    sel = torch.topk(z, topk, dim=1).indices.to(torch.int32)
    if case["drop"]:   # picks over an expert's capacity go nowhere
        sel = torch.where(torch.rand((n, topk), device="cuda", generator=g) < case["drop"], -1, sel)
    key = torch.where(sel < 0, ne, sel).view(-1).long()
    perm = torch.sort(key, stable=True).indices
    inv = torch.empty_like(perm)
    inv[perm] = torch.arange(n * topk, device="cuda")
    counts = torch.bincount(key, minlength=ne + 1)[:ne]
    offsets = torch.zeros(ne + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(counts, 0)
    return {"sel": sel, "perm": perm.to(torch.int32), "inv": inv.to(torch.int32), "offsets": offsets, "cap": max(1, int(counts.max()))}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 31)
    t = TYPES[case["type"]]
    n, R = case["n"], case["R"]

    def normal(*shape, by=1.0, dtype=t):
        return torch.randn(shape, device="cuda", dtype=dtype, generator=g).mul_(by)

    s = {"case": case}
    if case["op"] == "combine":
        s.update(routed(case, g))
        s["o"], s["dy"] = normal(n * case["topk"], R, by=0.5), normal(n, R, by=1e-2)
        s["w"] = 0.05 + torch.rand((n, case["topk"]), device="cuda", generator=g)
        s["residual"] = normal(n, R) if case["residual"] else None
        s["do"] = torch.zeros_like(s["o"])   # the slots that no pair has stay 0
        return s
    K = case["K"]
    grouped = case["op"].startswith("experts")
    if grouped:
        s.update(routed(case, g))
    lead = (case["ne"],) if grouped else ()
    slots = n * case["topk"] if grouped else n
    s["gather"] = grouped and case["gated"]   # gate and up read the rows themselves, other products the slots' own
    s["x"] = normal(n if s["gather"] else slots, K)
    s["W"] = normal(*lead, R, K, by=K ** -0.5)
    s["W2"] = normal(*lead, R, K, by=K ** -0.5) if case["gated"] else None
    if case["op"].endswith("_grad"):
        s["dy"] = normal(slots, R, by=1e-2)
        s["z"] = normal(slots, R) if case["act"] else None
        s["z2"] = normal(slots, R) if case["gated"] else None
        if grouped:
            s["dx"] = torch.zeros((slots, K), dtype=t, device="cuda")
            s["dz"] = torch.zeros((slots, R), dtype=t, device="cuda") if case["act"] else None
            s["dz2"] = torch.zeros((slots, R), dtype=t, device="cuda") if case["gated"] else None
        return s
    s["bias"] = normal(R, dtype=torch.float32) if case.get("bias") else None
    s["residual"] = normal(slots, R) if case.get("residual") else None
    if grouped:
        s["y"] = torch.zeros((slots, R), dtype=t, device="cuda")
        s["z"] = torch.zeros((slots, R), dtype=t, device="cuda") if case["keep"] else None
        s["z2"] = torch.zeros((slots, R), dtype=t, device="cuda") if case["keep"] and case["gated"] else None
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
_contexts = {}


def context():
    """The program's context, on torch's current stream."""
    import loki_amd
    key = torch.cuda.current_stream().cuda_stream
    if key not in _contexts:
        _contexts[key] = loki_amd.Context()
    return _contexts[key]


def run_own(s):
    case, c = s["case"], context()
    op, act = case["op"], case.get("act") or None
    if op == "combine":
        y = c.combine(s["o"], s["inv"], s["w"], sel=s["sel"], n_exp=case["ne"], residual=s["residual"])
        return (y, *c.combine_grad(s["dy"], s["o"], s["inv"], s["w"], sel=s["sel"], n_exp=case["ne"], do=s["do"]))
    out = torch.float32 if case.get("out32") else None
    if op == "matmul":
        return c.matmul(s["x"], s["W"], up=s["W2"], bias=s["bias"], act=act, residual=s["residual"], dtype=out)
    if op == "matmul_grad":
        dz, dz2, db = c.act_grad(s["dy"], s["z"], act, z2=s["z2"], bias=case["bias"])
        return (dz, dz2, db, *c.matmul_grad(dz, s["x"], s["W"], dz2=dz2, up=s["W2"], dw_dtype=out))
    order = {"perm": s["perm"], "topk": case["topk"]} if s["gather"] else {}
    if op == "experts":
        return c.expert_matmul(s["x"], s["W"], s["offsets"], up=s["W2"], act=act, y=s["y"], z=s["z"], z2=s["z2"], **order)
    dz, dz2 = s["dy"], None
    if act:
        dz, dz2, _ = c.act_grad(s["dy"], s["z"], act, z2=s["z2"], offsets=s["offsets"], dz=s["dz"], dz2=s["dz2"])
    return (dz, dz2, *c.expert_matmul_grad(dz, s["x"], s["W"], s["offsets"], dz2=dz2, up=s["W2"], dx=s["dx"], **order))


# ------------------------------------------------------------------------------------------------ plain forms
def inner(z, act):
    return z if act == "silu" else GELU * (z + 0.044715 * z * z * z)


def activate(z, act):
    return z * torch.sigmoid(inner(z, act)) if act else z


def slope(z, act):
    s = torch.sigmoid(inner(z, act))
    return s + z * s * (1 - s) * (1.0 if act == "silu" else GELU * (1 + 3 * 0.044715 * z * z))


def act_back(s, t):
    """(dz, dz2, the bias's gradient) of the slots, in the type and the sums in 32 bits."""
    case = s["case"]
    dy = s["dy"].float()
    if not case["act"]:
        return s["dy"], None, dy.sum(0)
    z = s["z"].float()
    d = dy * slope(z, case["act"])
    if not case["gated"]:
        return d.to(t), None, d.sum(0)
    return (d * s["z2"].float()).to(t), (dy * activate(z, case["act"])).to(t), None


def places(s):
    """Every expert's slots side by side: (slot [ne][cap], whether there is one), and of each slot its expert and place, and whether it has one."""
    off, P = s["offsets"].long(), s["perm"].numel()
    j = torch.arange(s["cap"], device=off.device)
    there = j[None] < (off[1:] - off[:-1])[:, None]
    slot = (off[:-1, None] + j[None]).clamp_(max=P - 1)
    i = torch.arange(P, device=off.device)
    e = torch.bucketize(i, off[1:], right=True)
    held = e < off.numel() - 1
    e = e.clamp_(max=off.numel() - 2)
    return slot, there, e, (i - off[e]).clamp_(0, s["cap"] - 1), held


def rows_of(s):
    """The row of x that each slot reads."""
    P = s["perm"].numel()
    return s["perm"].long() // s["case"]["topk"] if s["gather"] else torch.arange(P, device=s["perm"].device)


def run_plain(s):
    case = s["case"]
    op, t = case["op"], TYPES[case["type"]]
    if op == "combine":
        n, k, R = case["n"], case["topk"], case["R"]
        ok = s["sel"] >= 0
        at = s["inv"].view(n, k).long()
        o, w = s["o"].float()[at], torch.where(ok, s["w"], 0.0)
        y = (o * w[:, :, None]).sum(1)
        if s["residual"] is not None:
            y = y + s["residual"].float()
        dy = s["dy"].float()[:, None]
        do = torch.zeros((n * k, R), dtype=t, device=o.device).index_copy_(0, at.view(-1), (dy * w[:, :, None]).to(t).view(-1, R))
        return y.to(t), do, torch.where(ok, (o * dy).sum(2), 0.0)
    out = torch.float32 if case.get("out32") else t
    if op == "matmul":
        x = s["x"].float()
        z = x @ s["W"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"]
        y = activate(z, case["act"])
        if case["gated"]:
            y = y * (x @ s["W2"].float().t())
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(out)
    if op == "matmul_grad":
        dz, dz2, db = act_back(s, t)
        d, x = dz.float(), s["x"].float()
        dx, dW = d @ s["W"].float(), d.t() @ x
        if not case["gated"]:
            return dz, dz2, db if case["bias"] else None, dx.to(t), dW.to(out)
        d2 = dz2.float()
        return dz, dz2, None, (dx + d2 @ s["W2"].float()).to(t), dW.to(out), (d2.t() @ x).to(out)
    slot, there, e, place, held = places(s)
    row, ne = rows_of(s), case["ne"]
    zero = torch.zeros((), device=row.device)
    xs = s["x"][row].float()   # of each slot
    few = row.numel() <= 64    # a matrix for each slot; else every expert's slots side by side
    side = lambda v: torch.where(there[:, :, None], v[slot], zero)  # noqa: E731
    if op == "experts":
        def product(W):
            if few:
                return torch.bmm(W[e].float(), xs[:, :, None])[:, :, 0]
            return torch.bmm(side(xs), W.float().transpose(1, 2).contiguous())[e, place]

        z = product(s["W"])
        y = activate(z, case["act"])
        both = [z]
        if case["gated"]:
            both.append(product(s["W2"]))
            y = y * both[1]
        res = [y, *both] if case["keep"] else [y]
        res = tuple(torch.where(held[:, None], v, zero).to(t) for v in res)
        return res if case["keep"] else res[0]
    dz, dz2, _ = act_back(s, t)
    if case["act"]:   # the slots of no expert stay 0
        dz = torch.where(held[:, None], dz, zero.to(t))
        dz2 = torch.where(held[:, None], dz2, zero.to(t)) if case["gated"] else None
    xp = side(xs)

    def back(d, W):
        dp = side(d.float())
        return torch.bmm(dp, W.float())[e, place], torch.bmm(dp.transpose(1, 2).contiguous(), xp).to(t)

    dx, dW = back(dz, s["W"])
    more = ()
    if case["gated"]:
        dx2, dW2 = back(dz2, s["W2"])
        dx, more = dx + dx2, (dW2,)
    return (dz, dz2, torch.where(held[:, None], dx, zero).to(t), dW, *more)


def run(state):
    return run_own(state) if own else run_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n, R = case["n"], case["R"]
    if case["op"] == "combine":
        P = n * case["topk"]
        # o, y, dy, do and the residual; the weights, their gradient, the picks and their slots
        return {"bytes": 2 * R * (2 * P + 2 * n + (n if case["residual"] else 0)) + 16 * P, "flops": 5 * P * R}
    K = case["K"]
    two = 2 if case["gated"] else 1
    grouped = case["op"].startswith("experts")
    slots = round(n * case["topk"] * (1 - case["drop"])) if grouped else n
    ne = case["ne"] if grouped else 1
    used = max(1, round(ne * (1 - (1 - 1 / ne) ** slots))) if grouped else 1   # experts with a slot
    xs = n if grouped and case["gated"] else slots
    out = 4 if case.get("out32") else 2
    if case["op"].endswith("_grad"):
        acts = 2 * slots * R * (1 + (1 + two if case["act"] else 0) + (1 if case["gated"] else 0))   # dy, z, dz
        return {"bytes": acts + 2 * (xs + slots) * K + two * R * K * (2 * used + out * ne), "flops": 4 * slots * R * K * two}
    kept = 1 + (two if case.get("keep") else 0) + (1 if case.get("residual") else 0)
    return {"bytes": 2 * xs * K + 2 * two * used * R * K + slots * R * (out + 2 * (kept - 1)) + (4 * R if case.get("bias") else 0), "flops": 2 * slots * R * K * two}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f8, n, R = torch.float64, case["n"], case["R"]
    up = lambda v: None if v is None else v.to(f8)  # noqa: E731

    def sigma(v):
        return 1 / (1 + torch.exp(-v))

    def arg(v):   # (what the sigmoid is taken of, its derivative)
        if case["act"] == "silu":
            return v, 1.0
        c = 2 * math.sqrt(2 / math.pi)
        return c * v + c * 0.044715 * v ** 3, c + 3 * c * 0.044715 * v ** 2

    def f(v):
        return v * sigma(arg(v)[0]) if case["act"] else v

    def df(v):
        a, da = arg(v)
        return sigma(a) + v * da * sigma(a) * sigma(-a)

    if case["op"] == "combine":
        k = case["topk"]
        y = up(s["residual"]) if s["residual"] is not None else torch.zeros((n, R), dtype=f8, device="cuda")
        do, dw = torch.zeros((n * k, R), dtype=f8, device="cuda"), torch.zeros((n, k), dtype=f8, device="cuda")
        inv, dy = s["inv"].view(n, k).long(), up(s["dy"])
        for j in range(k):
            on = (s["sel"][:, j] >= 0).nonzero()[:, 0]
            at, w = inv[on, j], up(s["w"][on, j])[:, None]
            o = up(s["o"][at])
            y[on] += w * o
            do[at] = w * dy[on]
            dw[on, j] = (o * dy[on]).sum(1)
        return y, do, dw
    if case["op"].endswith("_grad"):
        dy, t = up(s["dy"]), TYPES[case["type"]]
        dz, dz2, db = s["dy"], None, dy.sum(0) if case.get("bias") else None
        if case["gated"]:
            z = up(s["z"])
            dz, dz2 = dy * df(z) * up(s["z2"]), dy * f(z)
        elif case["act"]:
            dz = dy * df(up(s["z"]))
            db = dz.sum(0) if case.get("bias") else None
    if not case["op"].startswith("experts"):
        x, W, W2 = up(s["x"]), up(s["W"]), up(s["W2"])
        if case["op"] == "matmul":
            z = x @ W.t() + (up(s["bias"]) if s["bias"] is not None else 0.0)
            y = f(z) * (x @ W2.t()) if case["gated"] else f(z)
            return y + up(s["residual"]) if s["residual"] is not None else y
        d = up(dz.to(t))   # the products are of the gradients as they are kept
        if not case["gated"]:
            return dz, dz2, db, d @ W, d.t() @ x
        d2 = up(dz2.to(t))
        return dz, dz2, db, d @ W + d2 @ W2, d.t() @ x, d2.t() @ x
    cuts, P, K = s["offsets"].tolist(), n * case["topk"], case["K"]
    grad = case["op"] == "experts_grad"
    mats = [s["W"], s["W2"]] if case["gated"] else [s["W"]]
    if grad:
        ds = [v for v in (dz, dz2) if v is not None]
        if case["act"]:
            for v in ds:
                v[cuts[-1]:] = 0
        dx = torch.zeros((P, K), dtype=f8, device="cuda")
        dWs = [torch.zeros(W.shape, dtype=torch.float32, device="cuda") for W in mats]   # (rounded to 32 bits, for memory's sake)
    else:
        zs = [torch.zeros((P, R), dtype=f8, device="cuda") for _ in mats]
    for i in range(case["ne"]):
        a, b = cuts[i], cuts[i + 1]
        if a == b:
            continue
        x = up(s["x"][s["perm"][a:b].long() // case["topk"]] if s["gather"] else s["x"][a:b])
        for m, W in enumerate(mats):
            w = up(W[i])
            if grad:
                d = up(ds[m][a:b].to(t))
                dx[a:b] += d @ w
                dWs[m][i] = (d.t() @ x).float()
            else:
                zs[m][a:b] = x @ w.t()
    if grad:
        return (dz, dz2, dx, *dWs)
    y = f(zs[0]) * zs[1] if case["gated"] else f(zs[0])
    return (y, *zs) if case["keep"] else y
