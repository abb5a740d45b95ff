"""The workloads by which the mixture-of-experts and Muon operators are measured, through their public entry points.

``listed()`` names them, ``draw()`` gives more of the same ranges; ``prepare()`` builds what a program has in hand
before the call, ``run()`` is one pass (in plain torch operations, or through ``kan_amd`` where ``own`` is true),
``work()`` what a pass cannot do without and ``exact()`` the same results in 64 bits.
"""
import math

import torch

own = False

# The quintic Newton-Schulz iteration's coefficients and its count of steps.
NS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
# Muon's settings.
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
RENORM_EPS = 1e-20


def _route(name, rows, experts, top_k, score, dtype, groups=1, top_groups=1, bias=False, train=True):
    return {"name": name, "kind": "route", "rows": rows, "experts": experts, "top_k": top_k, "score": score,
            "dtype": dtype, "groups": groups, "top_groups": top_groups, "bias": bias, "train": train}


def _experts(name, rows, in_dim, out_dim, degree, experts, top_k, dtype, train, drop=0.0):
    return {"name": name, "kind": "experts", "rows": rows, "in": in_dim, "out": out_dim, "degree": degree,
            "experts": experts, "top_k": top_k, "dtype": dtype, "train": train, "drop": drop}


def _orth(name, batch, rows, cols, dtype):
    return {"name": name, "kind": "orthogonalize", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}


def _muon(name, experts, in_dim, out_dim, degree):
    return {"name": name, "kind": "muon", "experts": experts, "in": in_dim, "out": out_dim, "degree": degree}


def listed():
    return [
        # One request's row choosing two of eight experts: latency alone.
        _route("route_1", 1, 8, 2, "softmax", "fp32", train=False),
        # A training batch over many small experts: sigmoid scores, a balancing bias, groups; forward and backward.
        _route("route_16384_sigmoid_groups", 16384, 256, 8, "sigmoid", "fp32", 8, 4, True),
        # A ragged batch and an expert count that is no power of two, logits from a bf16 gate.
        _route("route_5000_softmax_bf16", 5000, 60, 6, "softmax", "bf16"),
        # Serving one request: the coefficients of the two experts that it goes to are the traffic.
        _experts("experts_1_bf16", 1, 2048, 2048, 8, 8, 2, "bf16", False),
        # A small batch of requests in the default precision.
        _experts("experts_48_fp32", 48, 512, 512, 8, 16, 2, "fp32", False),
        # The benchmark's layer width and batch as a mixture, forward and backward in bf16.
        _experts("experts_8192_bf16", 8192, 1024, 1024, 8, 8, 2, "bf16", True),
        # A mixture of the deep stack's width in the default precision, forward and backward.
        _experts("experts_8192_fp32", 8192, 512, 512, 8, 16, 2, "fp32", True),
        # Widths, degree and batch that are no powers of two, some slots dropped by a capacity limit.
        _experts("experts_3000_odd_fp32", 3000, 500, 300, 5, 6, 2, "fp32", True, 0.02),
        # The gradient of the small classifier's first layer: [out, in x (degree + 1)], launch-bound.
        _orth("orthogonalize_64x3920_fp32", 1, 64, 3920, "fp32"),
        # The gradient of the benchmark's layer.
        _orth("orthogonalize_1024x9216_bf16", 1, 1024, 9216, "bf16"),
        # A few tall matrices of odd sizes.
        _orth("orthogonalize_3x900x500_bf16", 3, 900, 500, "bf16"),
        # One whole optimizer step of a mixture's coefficients.
        _muon("muon_8_experts_fp32", 8, 512, 512, 8),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]; half of them as they fall, half multiples of 32 where that fits."""
    while True:
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        v = int(round(v / 32) * 32) if rng.random() < 0.5 and v > 48 else int(round(v))
        v = max(lo, min(hi, v))
        if v != 3 * 1024:
            return v


def draw(rng):
    kind = rng.choice(["route", "route", "infer", "infer", "train", "train", "train", "orth", "orth", "muon"])
    top = work(listed()[5])["flops"]
    while True:
        if kind == "route":
            groups = rng.choice([1, 1, 2, 4, 8])
            experts = groups * _size(rng, 4, 256 // groups)
            top_groups = rng.randint((groups + 1) // 2, groups)
            c = _route("", _size(rng, 1, 16384), experts, rng.randint(1, min(8, experts // groups * top_groups)),
                       rng.choice(["softmax", "sigmoid"]), rng.choice(["fp32", "bf16"]), groups, top_groups,
                       rng.random() < 0.5, rng.random() < 0.7)
        elif kind == "infer":
            experts = _size(rng, 2, 32)
            c = _experts("", _size(rng, 1, 512), _size(rng, 64, 2048), _size(rng, 32, 2048), rng.randint(2, 16),
                         experts, rng.randint(1, min(4, experts)), rng.choice(["bf16", "fp32"]), False)
        elif kind == "train":
            experts = _size(rng, 2, 32)
            c = _experts("", _size(rng, 128, 8192), _size(rng, 64, 1024), _size(rng, 32, 1024), rng.randint(2, 16),
                         experts, rng.randint(1, min(4, experts)), rng.choice(["bf16", "fp32"]), True,
                         rng.choice([0.0, 0.0, 0.05]))
        elif kind == "orth":
            c = _orth("", rng.randint(1, 8), _size(rng, 16, 1024), _size(rng, 16, 9216), rng.choice(["bf16", "fp32"]))
            if rng.random() < 0.3:
                c["rows"], c["cols"] = c["cols"], c["rows"]
        else:
            c = _muon("", rng.randint(1, 8), _size(rng, 16, 512), _size(rng, 16, 512), rng.randint(2, 8))
        # no more than the largest listed case: plain 32-bit products, and room for the coefficients
        w = work(c)
        scale = 4.0 if kind in ("orth", "muon") else 1.0
        if scale * w["flops"] <= top and w["bytes"] <= 2.5e9:
            del c["name"]
            return c


# ---- what a program has before the call --------------------------------------

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _gradient(gen, batch, rows, cols):
    """Matrices as gradients are: a few strong directions over a broad floor."""
    r = max(1, min(rows, cols) // 32)
    strong = torch.matmul(_randn(gen, batch, rows, r), _randn(gen, batch, r, cols)) / math.sqrt(r)
    return 1e-3 * (strong + 0.3 * _randn(gen, batch, rows, cols))


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "route":
        dtype = _DTYPES[case["dtype"]]
        # logits of a gate that has learned to prefer some experts
        popularity = 0.5 * _randn(gen, 1, case["experts"])
        s["logits"] = (1.5 * _randn(gen, case["rows"], case["experts"]) + popularity).to(dtype)
        # a balancing bias is moved in fixed small steps
        s["bias"] = torch.round(20 * _randn(gen, case["experts"])) * 0.001 if case["bias"] else None
        s["dw"] = _randn(gen, case["rows"], case["top_k"])
    elif case["kind"] == "experts":
        dtype = _DTYPES[case["dtype"]]
        rows, top_k, experts = case["rows"], case["top_k"], case["experts"]
        s["x"] = _randn(gen, rows, case["in"]).to(dtype)
        std = 1.0 / (case["in"] * (case["degree"] + 1))
        s["coeffs"] = (std * _randn(gen, experts, case["in"], case["out"], case["degree"] + 1)).to(dtype)
        # a router's choice: distinct experts in each row, some more popular than others
        scores = _randn(gen, rows, experts) + 0.5 * _randn(gen, 1, experts)
        best, idx = torch.topk(scores, top_k, dim=1)
        s["weights"] = torch.softmax(best, dim=1).to(dtype)
        if case["drop"]:
            gone = torch.rand(rows, top_k, device="cuda", generator=gen) < case["drop"]
            idx = torch.where(gone, -1, idx)
            s["weights"] = torch.where(gone, 0.0, s["weights"]).to(dtype)
        s["indices"] = idx
        # the rows that the plain form's padded products hold for each expert
        s["capacity"] = max(1, int(torch.bincount(idx[idx >= 0], minlength=1).max())) if bool((idx >= 0).any()) else 1
        s["dy"] = (_randn(gen, rows, case["out"]) / rows).to(dtype)
    elif case["kind"] == "orthogonalize":
        s["g"] = _gradient(gen, case["batch"], case["rows"], case["cols"]).to(_DTYPES[case["dtype"]])
    else:
        e, i, o, d = case["experts"], case["in"], case["out"], case["degree"] + 1
        s["p"] = _randn(gen, e, i, o, d) / (i * d)
        s["g"] = _gradient(gen, e, o, i * d).reshape(e, o, i, d).transpose(1, 2).contiguous()
        s["buf"] = 1e-3 * _randn(gen, e, i, o, d)
    return s


# ---- the plain forms ----------------------------------------------------------

def _plain_route(s):
    c = s["case"]
    x = s["logits"].float()
    open_ = x > -math.inf  # false for NaN too
    x = torch.where(open_, x, -math.inf)
    if c["score"] == "softmax":
        e = torch.exp(x - torch.clamp(x.amax(-1, keepdim=True), min=torch.finfo(torch.float32).min))
        total = e.double().sum(-1, keepdim=True).float()
        p = torch.where(total > 0, e / total, 0.0)
    else:
        p = 1.0 / (1.0 + torch.exp(-x))
    key = torch.where(open_, p if s["bias"] is None else p + s["bias"], -math.inf)
    if c["groups"] > 1:
        by = key.view(key.shape[0], c["groups"], -1)
        two = torch.sort(by, dim=-1, descending=True, stable=True).values[..., :2]
        value = two[..., 0] + (torch.where(two[..., 1] > -math.inf, two[..., 1], 0.0) if by.shape[-1] > 1 else 0.0)
        kept = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(keep[..., None], by, -math.inf).view_as(key)
    order = torch.sort(key, dim=-1, descending=True, stable=True)
    best, idx = order.values[:, :c["top_k"]], order.indices[:, :c["top_k"]]
    there = best > -math.inf
    chosen = torch.where(there, p.gather(1, idx), 0.0)
    total = chosen.sum(-1, keepdim=True) + RENORM_EPS
    w = chosen / total
    out = {"weights": w, "indices": torch.where(there, idx, -1)}
    if c["train"]:
        dchosen = torch.where(there, (s["dw"] - (s["dw"] * w).sum(-1, keepdim=True)) / total, 0.0)
        dp = torch.zeros_like(p).scatter_(1, idx, dchosen)
        if c["score"] == "softmax":
            dl = p * (dp - (p * dp).sum(-1, keepdim=True))
        else:
            dl = p * (1.0 - p) * dp
        out["dlogits"] = dl.to(s["logits"].dtype)
    return out


def _plain_basis(t, degree, slope):
    """T_0..T_degree of t, and with `slope` their derivatives, in a last dimension."""
    ts, us = [torch.ones_like(t), t], [torch.zeros_like(t), torch.ones_like(t)]
    for n in range(2, degree + 1):
        ts.append(2 * t * ts[-1] - ts[-2])
        if slope:  # T_n' = 2 T_{n-1} + 2 t T_{n-1}' - T_{n-2}'
            us.append(2 * ts[n - 1] + 2 * t * us[-1] - us[-2])
    return torch.stack(ts[:degree + 1], -1), torch.stack(us[:degree + 1], -1) if slope else None


def _plain_experts(s):
    c = s["case"]
    x, coeffs, idx, w = s["x"].float(), s["coeffs"].float(), s["indices"], s["weights"].float()
    rows, top_k, experts, cap = c["rows"], c["top_k"], c["experts"], s["capacity"]
    width, out, d = c["in"], c["out"], c["degree"] + 1
    # each kept slot's place in its expert's padded block
    slots = torch.where(idx >= 0, idx, experts).reshape(-1)
    order = torch.argsort(slots, stable=True)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=x.device).scatter_add_(0, slots, torch.ones_like(slots))
    place = torch.empty_like(slots)
    place[order] = torch.arange(slots.numel(), device=x.device) - (torch.cumsum(counts, 0) - counts)[slots[order]]
    kept = slots < experts
    at = torch.where(kept, slots * cap + place, experts * cap)
    token = torch.full((experts * cap + 1,), rows, dtype=torch.int64, device=x.device)
    token[at] = torch.arange(slots.numel(), device=x.device) // top_k
    token[-1] = rows
    token = token[:-1]
    t = torch.tanh(x)
    basis, slope = _plain_basis(t, c["degree"], c["train"])
    basis = torch.cat([basis.reshape(rows, -1), basis.new_zeros(1, width * d)])
    phi = basis[token].view(experts, cap, width * d)
    matrix = coeffs.permute(0, 1, 3, 2).reshape(experts, width * d, out).contiguous()
    z = torch.cat([torch.bmm(phi, matrix).view(-1, out), phi.new_zeros(1, out)])
    mine = z[at].view(rows, top_k, out)
    result = {"y": (mine * w[..., None]).sum(1).to(s["x"].dtype)}
    if c["train"]:
        dy = s["dy"].float()
        result["dweights"] = torch.where(idx >= 0, (mine * dy[:, None]).sum(-1), 0.0).to(s["weights"].dtype)
        dz = z.new_zeros(experts * cap + 1, out)
        dz[at] = (dy[:, None] * w[..., None]).view(-1, out)
        dz[-1] = 0
        dz = dz[:-1].view(experts, cap, out)
        dmatrix = torch.bmm(phi.transpose(1, 2), dz)
        result["dcoeffs"] = dmatrix.view(experts, width, d, out).transpose(2, 3).contiguous().to(s["coeffs"].dtype)
        dphi = torch.bmm(dz, matrix.transpose(1, 2)).view(-1, width * d)
        dphi = torch.cat([dphi, dphi.new_zeros(1, width * d)])
        dphi = dphi[at].view(rows, top_k, width, d).sum(1)
        result["dx"] = ((dphi * slope).sum(-1) * (1 - t * t)).to(s["x"].dtype)
    return result


def _plain_orthogonalize(g):
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + NS_EPS)
    a, b, c = NS
    for _ in range(NS_STEPS):
        gram = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-2, -1) if tall else x


def _plain_muon(s):
    p, g, buf = s["p"], s["g"], s["buf"]
    e, i, o, d = p.shape
    buf.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
    u = (1 - MOMENTUM) * g + MOMENTUM * buf
    update = _plain_orthogonalize(u.transpose(1, 2).reshape(e, o, i * d))
    update = update.reshape(e, o, i, d).transpose(1, 2)
    p.mul_(1 - LR * DECAY).add_(update, alpha=-LR * math.sqrt(max(1.0, o / (i * d))))
    return {"param": p, "momentum": buf}


# ---- one pass -----------------------------------------------------------------

def _own(s):
    from kan_amd import functional, optim
    c = s["case"]
    if c["kind"] == "route":
        logits = s["logits"].detach().requires_grad_(c["train"])
        w, idx = functional.route(logits, c["top_k"], score=c["score"], bias=s["bias"], groups=c["groups"],
                                  top_groups=c["top_groups"])
        out = {"weights": w.detach(), "indices": idx}
        if c["train"]:
            out["dlogits"], = torch.autograd.grad(w, logits, s["dw"])
        return out
    if c["kind"] == "experts":
        x, coeffs, w = s["x"], s["coeffs"], s["weights"]
        if not c["train"]:
            return {"y": functional.kan_experts(x, coeffs, s["indices"], w)}
        x, coeffs, w = (v.detach().requires_grad_() for v in (x, coeffs, w))
        y = functional.kan_experts(x, coeffs, s["indices"], w)
        dx, dcoeffs, dw = torch.autograd.grad(y, (x, coeffs, w), s["dy"])
        return {"y": y.detach(), "dx": dx, "dcoeffs": dcoeffs, "dweights": dw}
    if c["kind"] == "orthogonalize":
        return functional.orthogonalize(s["g"], steps=NS_STEPS, coefficients=NS, eps=NS_EPS)
    optim.muon_step_(s["p"], s["g"], s["buf"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, steps=NS_STEPS,
                     coefficients=NS, eps=NS_EPS)
    return {"param": s["p"], "momentum": s["buf"]}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "route":
        return _plain_route(state)
    if kind == "experts":
        return _plain_experts(state)
    if kind == "orthogonalize":
        return _plain_orthogonalize(state["g"]).to(state["g"].dtype)
    return _plain_muon(state)


def work(case):
    """Bytes: each input read once and each output written once. Flops: multiply-adds of the products, twice."""
    size = 2 if case.get("dtype") == "bf16" else 4
    if case["kind"] == "route":
        t, e, k = case["rows"], case["experts"], case["top_k"]
        nbytes = t * e * size + t * k * 12
        if case["train"]:  # dw read, dlogits written
            nbytes += t * k * 4 + t * e * size
        return {"bytes": nbytes, "flops": 4.0 * t * e}
    if case["kind"] == "experts":
        t, k = case["rows"], case["top_k"]
        slots = t * k * (1 - case["drop"])
        per = case["in"] * case["out"] * (case["degree"] + 1)
        # experts that at least one slot goes to, for the coefficients' bytes
        hit = case["experts"] * (1 - (1 - 1 / case["experts"]) ** slots)
        nbytes = per * hit * size + t * (case["in"] + case["out"]) * size + t * k * 12
        flops = 2.0 * slots * case["in"] * case["out"] * case["degree"]
        if case["train"]:
            nbytes += per * case["experts"] * size + t * (case["in"] + case["out"]) * size + t * k * 4
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["kind"] == "orthogonalize":
        n, rows, cols = case["batch"], case["rows"], case["cols"]
        moved = 2 * n * rows * cols * size
    else:
        n, rows, cols = case["experts"], case["out"], case["in"] * (case["degree"] + 1)
        moved = 5 * n * rows * cols * 4
    # every factor is a polynomial in X X^T: one such product, one product with X, and four symmetric ones a step
    # between them, each symmetric one at half its multiply-adds
    m, wide = min(rows, cols), max(rows, cols)
    return {"bytes": moved, "flops": n * (3.0 * m * m * wide + NS_STEPS * 4.0 * m ** 3)}


# ---- the same from the definitions, in 64 bits --------------------------------

def _exact_route(s):
    c = s["case"]
    l = s["logits"].double()
    p = torch.softmax(l, -1) if c["score"] == "softmax" else torch.sigmoid(l)
    key = p if s["bias"] is None else p + s["bias"].double()
    if c["groups"] > 1:
        by = key.view(key.shape[0], c["groups"], -1)
        value = by.topk(min(2, by.shape[-1]), -1).values.sum(-1)
        floor = value.topk(c["top_groups"], -1).values[:, -1:]
        key = torch.where((value >= floor)[..., None], by, -math.inf).view_as(key)
    idx = key.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_k"]]
    l = l.requires_grad_()
    p = torch.softmax(l, -1) if c["score"] == "softmax" else torch.sigmoid(l)
    chosen = p.gather(1, idx)
    w = chosen / (chosen.sum(-1, keepdim=True) + RENORM_EPS)
    out = {"weights": w.detach(), "indices": None}
    if c["train"]:
        out["dlogits"], = torch.autograd.grad(w, l, s["dw"].double())
    return out


def _exact_experts(s):
    c = s["case"]
    rows, top_k, degree = c["rows"], c["top_k"], c["degree"]
    x, idx, w = s["x"].double(), s["indices"], s["weights"].double()
    n = torch.arange(degree + 1, device=x.device, dtype=torch.float64)
    t = torch.tanh(x)
    y = x.new_zeros(rows, c["out"])
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    dcoeffs = []
    for e in range(c["experts"]):
        r, j = torch.nonzero(idx == e, as_tuple=True)
        m = s["coeffs"][e].double().transpose(1, 2).reshape(-1, c["out"])
        theta = torch.acos(t[r])[..., None]
        phi = torch.cos(n * theta).view(len(r), m.shape[0])
        z = phi @ m
        y.index_add_(0, r, z * w[r, j][:, None])
        if c["train"]:
            dy = s["dy"].double()[r]
            dw[r, j] = (z * dy).sum(-1)
            dz = dy * w[r, j][:, None]
            dcoeffs.append((phi.t() @ dz).view(c["in"], degree + 1, c["out"]).transpose(1, 2).to(torch.float64))
            dphi = (dz @ m.t()).view(len(r), c["in"], degree + 1)
            # d cos(n acos t) / dx = n sin(n theta) / sin(theta) (1 - t^2), and sin(theta)^2 = 1 - t^2
            dx.index_add_(0, r, (dphi * n * torch.sin(n * theta) * torch.sin(theta)).sum(-1))
    out = {"y": y}
    if c["train"]:
        out.update(dx=dx, dcoeffs=torch.stack(dcoeffs), dweights=dw)
    return out


def _exact_orthogonal(g):
    """The iteration on the singular values: X = V q(L) V^T X0 with X0 X0^T = V L V^T."""
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + NS_EPS)
    gram = torch.matmul(x, x.transpose(-2, -1).contiguous())
    values, vectors = torch.linalg.eigh(gram.cpu())
    squared, factor = values.clamp(min=0), torch.ones_like(values)
    for _ in range(NS_STEPS):
        step = NS[0] + NS[1] * squared + NS[2] * squared ** 2
        factor, squared = factor * step, squared * step ** 2
    q = torch.matmul(vectors * factor[..., None, :], vectors.transpose(-2, -1)).to(x.device)
    x = torch.matmul(q, x.contiguous())
    return x.transpose(-2, -1) if tall else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(s)
    if case["kind"] == "experts":
        return _exact_experts(s)
    if case["kind"] == "orthogonalize":
        return _exact_orthogonal(s["g"])
    p, g, buf = (s[k].double() for k in ("p", "g", "buf"))
    e, i, o, d = p.shape
    buf = MOMENTUM * buf + (1 - MOMENTUM) * g
    u = (1 - MOMENTUM) * g + MOMENTUM * buf
    update = _exact_orthogonal(u.transpose(1, 2).reshape(e, o, i * d)).reshape(e, o, i, d).transpose(1, 2)
    return {"param": p * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, o / (i * d))) * update, "momentum": buf}
