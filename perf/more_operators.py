"""The workloads by which the residual-block, dropout, log-probability and few-row mixture operators are measured,
through their public entry points.

``listed()`` names them, ``draw()`` gives more of the same ranges; ``prepare()`` builds what a program has in hand
before the call, ``run()`` is one pass (in plain torch operations, or through ``kan_amd`` where ``own`` is true),
``work()`` what a pass cannot do without and ``exact()`` the same results in 64 bits.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
# Added to the sum that the renormalised weights of a mixture are divided by.
RENORM_EPS = 1e-20


def _residual(name, rows, dim, stream, branch, norm="rms", params="fp32", post=True, bias=False, gate="dim",
              following=True, drop=0.0, train=True, first=False):
    return {"name": name, "kind": "residual", "rows": rows, "dim": dim, "stream": stream, "branch": branch,
            "norm": norm, "params": params, "post": post, "bias": bias, "gate": gate, "next": following,
            "drop": drop, "train": train, "first": first}


def _dropout(name, rows, dim, dtype, p, train):
    return {"name": name, "kind": "dropout", "rows": rows, "dim": dim, "dtype": dtype, "p": p, "train": train}


def _logprobs(name, rows, classes, dtype, top, train, masked=0.0):
    return {"name": name, "kind": "logprobs", "rows": rows, "classes": classes, "dtype": dtype, "top": top,
            "train": train, "masked": masked}


def _mixture(name, rows, in_dim, out_dim, degree, experts, top_k, dtype, coeffs, score="softmax", groups=1,
             top_groups=1, bias=False):
    return {"name": name, "kind": "mixture", "rows": rows, "in": in_dim, "out": out_dim, "degree": degree,
            "experts": experts, "top_k": top_k, "dtype": dtype, "coeffs": coeffs, "score": score, "groups": groups,
            "top_groups": top_groups, "bias": bias}


def listed():
    return [
        # One request's row after a layer of 2048 outputs: the norm of the branch, the sum and the next norm.
        _residual("residual_1_bf16", 1, 2048, "fp32", "bf16", train=False),
        # The norm before the first block of a batch, a width that is no power of two; forward and backward.
        _residual("norm_8192x1000_fp32", 8192, 1000, "fp32", "fp32", "layer", bias=True, first=True),
        # A residual block at the benchmark's layer width and batch in bf16, with dropout; forward and backward.
        _residual("residual_8192x1024_bf16", 8192, 1024, "bf16", "bf16", drop=0.1),
        # The deep stack's width and batch in the default precision, layer norms, a gate a row; forward and backward.
        _residual("residual_65536x512_fp32", 65536, 512, "fp32", "fp32", "layer", bias=True, gate="row"),
        # Dropout of a small classifier's input, launch-bound; forward and backward.
        _dropout("dropout_256x784_fp32", 256, 784, "fp32", 0.2, True),
        # Dropout of the deep stack's hidden rows; forward and backward.
        _dropout("dropout_65536x512_bf16", 65536, 512, "bf16", 0.1, True),
        # The small classifier's batch of logits: log probabilities and entropy, forward and backward.
        _logprobs("logprobs_256x10_fp32", 256, 10, "fp32", 0, True),
        # One request over many classes with its twenty likeliest: one long row.
        _logprobs("logprobs_1x131072_top20", 1, 131072, "fp32", 20, False),
        # A training batch over many classes, an odd number of them, some masked; forward and backward.
        _logprobs("logprobs_4000x50001_bf16", 4000, 50001, "bf16", 5, True, 0.05),
        # One request through a mixture of the wide layer: gate, choice and two of eight experts.
        _mixture("mixture_1_bf16", 1, 2048, 2048, 8, 8, 2, "bf16", "bf16"),
        # A few requests in the default precision, many small experts, sigmoid scores with a balancing bias.
        _mixture("mixture_6_fp32", 6, 512, 512, 8, 64, 4, "fp32", "fp32", "sigmoid", 8, 4, True),
        # A small batch, widths and degree that are no powers of two, coefficients held in bf16.
        _mixture("mixture_40_odd", 40, 500, 300, 5, 6, 2, "fp32", "bf16"),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]; half of them as they fall, half multiples of 32 where that fits."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    v = int(round(v / 32) * 32) if rng.random() < 0.5 and v > 48 else int(round(v))
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["residual", "residual", "residual", "dropout", "logprobs", "logprobs", "mixture", "mixture"])
    while True:
        two = ["fp32", "bf16"]
        if kind == "residual":
            first, gate = rng.random() < 0.2, rng.choice(["none", "dim", "dim", "row"])
            branch = rng.choice(two)
            c = _residual("", _size(rng, 1, 65536), _size(rng, 8, 16384), branch if first else rng.choice(two), branch,
                          rng.choice(["rms", "layer"]), rng.choice(["fp32", "fp32", "bf16"]), rng.random() < 0.8,
                          rng.random() < 0.4, gate, rng.random() < 0.8, rng.choice([0.0, 0.0, 0.1, 0.37]),
                          rng.random() < 0.7, first)
        elif kind == "dropout":
            c = _dropout("", _size(rng, 1, 65536), _size(rng, 8, 16384), rng.choice(two),
                         round(rng.uniform(0.01, 0.6), 3), rng.random() < 0.7)
        elif kind == "logprobs":
            classes = _size(rng, 2, 131072)
            c = _logprobs("", _size(rng, 1, 65536), classes, rng.choice(two),
                          rng.choice([0, 0, 1, min(5, classes), min(20, classes)]), rng.random() < 0.6,
                          rng.choice([0.0, 0.0, 0.05, 0.6]))
        else:
            groups = rng.choice([1, 1, 1, 2, 4])
            experts = groups * _size(rng, 4, 64 // groups)
            top_groups = rng.randint((groups + 1) // 2, groups)
            dtype = rng.choice(two)
            c = _mixture("", _size(rng, 1, 64), _size(rng, 16, 2048), _size(rng, 16, 2048), rng.randint(2, 16), experts,
                         rng.randint(1, min(4, experts // groups * top_groups)), dtype,
                         rng.choice(two) if dtype == "fp32" else "bf16", rng.choice(["softmax", "sigmoid"]), groups,
                         top_groups, rng.random() < 0.4)
            if c["experts"] * c["in"] * c["out"] * (c["degree"] + 1) > 3.2e8:
                continue
        if work(c)["bytes"] <= work(listed()[3])["bytes"]:
            del c["name"]
            return c


# ---- what a program has before the call --------------------------------------

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _dropout_state(gen):
    """(seed, offset) as a training program keeps them on the device."""
    return torch.randint(0, 2 ** 62, (2,), device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "residual":
        rows, dim = case["rows"], case["dim"]
        stream, branch, params = _DTYPES[case["stream"]], _DTYPES[case["branch"]], _DTYPES[case["params"]]
        # a residual stream has grown over the blocks before, some features more than others
        s["x"] = (2.0 * _randn(gen, rows, dim) * torch.exp(0.5 * _randn(gen, 1, dim))).to(stream)
        norms = (["next"] if case["next"] or case["first"] else []) + (["post"] if case["post"] and not case["first"] else [])
        for n in norms:
            s[n + "_weight"] = (1.0 + 0.2 * _randn(gen, dim)).to(params)
            s[n + "_bias"] = (0.1 * _randn(gen, dim)).to(params) if case["bias"] else None
        s["dh"] = (_randn(gen, rows, dim) / rows).to(branch)
        if not case["first"]:
            s["y"] = (0.3 * _randn(gen, rows, dim) + 0.1 * _randn(gen, 1, dim)).to(branch)
            s["gate"] = None
            if case["gate"] == "dim":  # a gate that has been learned from a small value on
                s["gate"] = (0.1 + 0.05 * _randn(gen, dim)).to(params)
            elif case["gate"] == "row":
                s["gate"] = (0.3 * _randn(gen, rows, dim)).to(branch)
            s["dout"] = (_randn(gen, rows, dim) / rows).to(stream)
        s["state"] = _dropout_state(gen)
    elif case["kind"] == "dropout":
        dtype = _DTYPES[case["dtype"]]
        s["x"] = _randn(gen, case["rows"], case["dim"]).to(dtype)
        s["dy"] = (_randn(gen, case["rows"], case["dim"]) / case["rows"]).to(dtype)
        s["state"] = _dropout_state(gen)
    elif case["kind"] == "logprobs":
        rows, classes, dtype = case["rows"], case["classes"], _DTYPES[case["dtype"]]
        # logits of a model that has learned something: a spread of their own, and some rows surer than others
        logits = _randn(gen, rows, classes) * (1.0 + 2.0 * torch.rand(rows, 1, device="cuda", generator=gen))
        targets = torch.randint(0, classes, (rows,), device="cuda", generator=gen)
        logits.scatter_add_(1, targets[:, None], 4.0 * torch.rand(rows, 1, device="cuda", generator=gen))
        if case["masked"]:  # classes that are not allowed here, never the target, and rows without a target
            gone = torch.rand(rows, classes, device="cuda", generator=gen) < case["masked"]
            logits.masked_fill_(gone.scatter_(1, targets[:, None], False), -math.inf)
            targets = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.05, -100, targets)
        s["logits"], s["targets"] = logits.to(dtype), targets
        s["dlogp"] = -torch.ones(rows, device="cuda") / rows
        s["dentropy"] = 0.01 * _randn(gen, rows) / rows
    else:
        rows, width, out, experts = case["rows"], case["in"], case["out"], case["experts"]
        s["x"] = _randn(gen, rows, width).to(_DTYPES[case["dtype"]])
        s["gate"] = 1.5 * _randn(gen, experts, width) / math.sqrt(width)
        std = 1.0 / (width * (case["degree"] + 1))
        s["coeffs"] = (std * _randn(gen, experts, width, out, case["degree"] + 1)).to(_DTYPES[case["coeffs"]])
        # a balancing bias is moved in fixed small steps
        s["bias"] = torch.round(20 * _randn(gen, experts)) * 0.001 if case["bias"] else None
    return s


# ---- the plain forms ----------------------------------------------------------

_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _plain_bits(state, rows, chunks, second):
    """16 random bits for each of 8 chunks' elements [rows, 8 chunks]: the ten rounds of Philox 4x32 (Salmon et al.,
    2011) on the counter (chunk, row, call), keyed by the seed; ``second`` selects the low halves' stream."""
    seed, call = state[0], state[1] & (2 ** 63 - 1)
    x0 = torch.arange(chunks, device=state.device).expand(rows, chunks)
    x1 = torch.arange(rows, device=state.device)[:, None].expand(rows, chunks)
    x2, x3 = (call & _LOW).expand(rows, chunks), ((call >> 32) + (2 ** 31 if second else 0)).expand(rows, chunks)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        # 64-bit products of 32-bit values: the low bits wrap as unsigned ones do, the shift's sign bits are masked off
        a, b = x0 * _M0, x2 * _M1
        x0, x1, x2, x3 = ((b >> 32) & _LOW) ^ x1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ x3 ^ k1, a & _LOW
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    words = torch.stack([x0, x1, x2, x3], -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, chunks * 8)


def _plain_keep(state, rows, dim, p):
    chunks = (dim + 7) // 8
    r = _plain_bits(state, rows, chunks, False) * 65536 + _plain_bits(state, rows, chunks, True)
    return r[:, :dim] >= round(p * 2 ** 32)


def _plain_stats(v, norm):
    """(v minus its mean where the norm takes it, 1 / its root mean square)."""
    if norm == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v, 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)


def _plain_norm_backward(g, weight, centred, r, norm):
    """Gradient of weight * centred * r in the values before it."""
    g, hat = g * weight, centred * r
    d = g - hat * (g * hat).mean(-1, keepdim=True)
    if norm == "layer":
        d = d - g.mean(-1, keepdim=True)
    return d * r


def _plain_residual(s):
    c, like = s["case"], lambda v, name: v.to(s[name].dtype)
    x, norm, out = s["x"].float(), c["norm"], {}
    grads = {}
    g = None if c["first"] or not c["train"] else s["dout"].float()
    if not c["first"]:
        u = s["y"].float()
        if c["post"]:
            centred, r = _plain_stats(u, norm)
            weight = s["post_weight"].float()
            u = centred * r * weight
            if c["bias"]:
                u = u + s["post_bias"].float()
        if c["drop"]:
            keep = _plain_keep(s["state"], c["rows"], c["dim"], c["drop"])
            u = torch.where(keep, u / (1.0 - c["drop"]), 0.0)
        gate = 1.0 if s["gate"] is None else s["gate"].float()
        x = x + 0.5 * gate * u
        out["out"] = x.to(s["x"].dtype)
    if c["next"] or c["first"]:
        next_centred, next_r = _plain_stats(x, norm)
        next_weight = s["next_weight"].float()
        h = next_centred * next_r * next_weight
        if c["bias"]:
            h = h + s["next_bias"].float()
        out["h"] = like(h, "dh")
        if c["train"]:
            dh = s["dh"].float()
            grads["next_weight"] = like((dh * next_centred * next_r).sum(0), "next_weight")
            if c["bias"]:
                grads["next_bias"] = like(dh.sum(0), "next_bias")
            dx = _plain_norm_backward(dh, next_weight, next_centred, next_r, norm)
            g = dx if g is None else g + dx
    if c["train"]:
        grads["x"] = like(g, "x")
        if not c["first"]:
            if s["gate"] is not None:
                dgate = 0.5 * g * u
                grads["gate"] = like(dgate.sum(0) if s["gate"].dim() == 1 else dgate, "gate")
            g = 0.5 * gate * g
            if c["drop"]:
                g = torch.where(keep, g / (1.0 - c["drop"]), 0.0)
            if c["post"]:
                grads["post_weight"] = like((g * centred * r).sum(0), "post_weight")
                if c["bias"]:
                    grads["post_bias"] = like(g.sum(0), "post_bias")
                g = _plain_norm_backward(g, weight, centred, r, norm)
            grads["y"] = like(g, "y")
        out.update(("d" + k, grads[k]) for k in sorted(grads))
    return out


def _plain_dropout(s):
    c = s["case"]
    keep = _plain_keep(s["state"], c["rows"], c["dim"], c["p"])
    out = {"y": torch.where(keep, s["x"].float() / (1.0 - c["p"]), 0.0).to(s["x"].dtype)}
    if c["train"]:
        out["dx"] = torch.where(keep, s["dy"].float() / (1.0 - c["p"]), 0.0).to(s["x"].dtype)
    return out


def _plain_logprobs(s):
    c, top = s["case"], s["case"]["top"]
    l = s["logits"].float()
    m = torch.clamp(l.amax(-1, keepdim=True), min=torch.finfo(torch.float32).min)
    e = torch.exp(l - m)
    # near 0 in rows that are sure: the sum in 64 bits
    lse = torch.log(e.double().sum(-1, keepdim=True)).float()
    logp = (l - m) - lse
    p = torch.exp(logp)
    ours = torch.where(p > 0, logp, 0.0)
    entropy = -(p * ours).double().sum(-1).float()
    has = (s["targets"] >= 0) & (s["targets"] < c["classes"])
    at = torch.where(has, s["targets"], 0)[:, None]
    out = {"logp": torch.where(has, logp.gather(1, at)[:, 0], 0.0), "entropy": entropy}
    if top:
        order = torch.sort(l, dim=-1, descending=True, stable=True)
        there = order.values[:, :top] > -math.inf
        out["top_logp"] = torch.where(there, (order.values[:, :top] - m) - lse, -math.inf)
        out["top_indices"] = torch.where(there, order.indices[:, :top], -1)
    if c["train"]:
        dlogp = torch.where(has, s["dlogp"], 0.0)[:, None]
        d = -p * (dlogp + s["dentropy"][:, None] * (ours + entropy[:, None]))
        d.scatter_add_(1, at, dlogp)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _plain_choice(s):
    """(weights, indices) of the rows' experts; the gate's sums in 64 bits, since choices hang on them."""
    c = s["case"]
    l = (s["x"].double()[:, None] * s["gate"].double()).sum(-1).float()
    if c["score"] == "softmax":
        e = torch.exp(l - l.amax(-1, keepdim=True))
        p = e / e.double().sum(-1, keepdim=True).float()
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    key = p if s["bias"] is None else p + s["bias"]
    if c["groups"] > 1:
        by = key.view(key.shape[0], c["groups"], -1)
        value = torch.sort(by, dim=-1, descending=True).values[..., :2].sum(-1)
        kept = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(keep[..., None], by, -math.inf).view_as(key)
    idx = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :c["top_k"]]
    chosen = p.gather(1, idx)
    return chosen / (chosen.sum(-1, keepdim=True) + RENORM_EPS), idx


def _plain_mixture(s):
    c = s["case"]
    w, idx = _plain_choice(s)
    t = torch.tanh(s["x"].float())
    basis = [torch.ones_like(t), t]
    while len(basis) <= c["degree"]:
        basis.append(2 * t * basis[-1] - basis[-2])
    phi = torch.stack(basis, -1)  # [rows, in, degree + 1]
    y = t.new_zeros(c["rows"], c["out"])
    for r in range(c["rows"]):
        for j in range(c["top_k"]):
            matrix = s["coeffs"].index_select(0, idx[r, j:j + 1])[0].float()  # [in, out, degree + 1]
            y[r] += w[r, j] * (matrix * phi[r][:, None]).sum((0, 2))
    return {"y": y.to(s["x"].dtype), "weights": w, "indices": idx}


# ---- one pass -----------------------------------------------------------------

def _own_residual(s):
    from kan_amd import functional
    c = s["case"]
    names = [k for k in ("x", "y", "gate", "post_weight", "post_bias", "next_weight", "next_bias")
             if s.get(k) is not None]
    v = {k: s[k].detach().requires_grad_() if c["train"] else s[k] for k in names}
    if c["first"]:
        results = (functional.row_norm(v["x"], v["next_weight"], v.get("next_bias"), norm=c["norm"], eps=EPS),)
        out, given = {"h": results[0].detach()}, (s["dh"],)
    else:
        results = functional.residual_norm(
            v["x"], v["y"], norm=c["norm"], eps=EPS, post_weight=v.get("post_weight"), post_bias=v.get("post_bias"),
            gate=v.get("gate"), scale=0.5, dropout=c["drop"], dropout_state=s["state"] if c["drop"] else None,
            next_weight=v.get("next_weight"), next_bias=v.get("next_bias"))
        if c["next"]:
            out, given = {"out": results[0].detach(), "h": results[1].detach()}, (s["dout"], s["dh"])
        else:
            out, given, results = {"out": results.detach()}, (s["dout"],), (results,)
    if c["train"]:
        grads = torch.autograd.grad(results, [v[k] for k in names], given)
        out.update(sorted(("d" + k, g) for k, g in zip(names, grads)))
    return out


def _own(s):
    from kan_amd import functional
    c = s["case"]
    if c["kind"] == "residual":
        return _own_residual(s)
    if c["kind"] == "dropout":
        x = s["x"].detach().requires_grad_(c["train"])
        y = functional.dropout(x, c["p"], s["state"])
        out = {"y": y.detach()}
        if c["train"]:
            out["dx"], = torch.autograd.grad(y, x, s["dy"])
        return out
    if c["kind"] == "logprobs":
        logits = s["logits"].detach().requires_grad_(c["train"])
        got = functional.log_probs(logits, s["targets"], top=c["top"])
        out = {"logp": got.logp.detach(), "entropy": got.entropy.detach()}
        if c["top"]:
            out.update(top_logp=got.top_logp, top_indices=got.top_indices)
        if c["train"]:
            out["dlogits"], = torch.autograd.grad((got.logp, got.entropy), logits, (s["dlogp"], s["dentropy"]))
        return out
    with torch.no_grad():
        y, w, idx = functional.kan_mixture(s["x"], s["gate"], s["coeffs"], c["top_k"], score=c["score"], bias=s["bias"],
                                           groups=c["groups"], top_groups=c["top_groups"])
    return {"y": y, "weights": w, "indices": idx}


def run(state):
    if own:
        return _own(state)
    return {"residual": _plain_residual, "dropout": _plain_dropout, "logprobs": _plain_logprobs,
            "mixture": _plain_mixture}[state["case"]["kind"]](state)


def work(case):
    """Bytes: each input read once and each output written once. Flops: additions and multiplications of the formulas."""
    size = {"fp32": 4, "bf16": 2}
    if case["kind"] == "residual":
        n, x, y = case["rows"] * case["dim"], size[case["stream"]], size[case["branch"]]
        following = case["next"] or case["first"]
        moved = x + (0 if case["first"] else x + y) + (y if following else 0)
        gate = y if case["gate"] == "row" and not case["first"] else 0
        moved += gate
        if case["train"]:  # the gradients of the outputs read, those of the inputs written
            moved += x + (0 if case["first"] else x + y) + (y if following else 0) + gate
        return {"bytes": n * moved, "flops": n * (30.0 if case["train"] else 12.0)}
    if case["kind"] == "dropout":
        n = case["rows"] * case["dim"]
        passes = 2 if case["train"] else 1
        return {"bytes": 2 * passes * n * size[case["dtype"]], "flops": 1.0 * passes * n}
    if case["kind"] == "logprobs":
        n = case["rows"] * case["classes"]
        nbytes = n * size[case["dtype"]] * (2 if case["train"] else 1) + case["rows"] * (16 + 12 * case["top"])
        return {"bytes": nbytes, "flops": n * (12.0 if case["train"] else 6.0)}
    rows, per = case["rows"], case["in"] * case["out"] * (case["degree"] + 1)
    slots = rows * case["top_k"]
    hit = case["experts"] * (1 - (1 - case["top_k"] / case["experts"]) ** rows)
    nbytes = per * hit * size[case["coeffs"]] + case["experts"] * case["in"] * 4
    nbytes += rows * (case["in"] + case["out"]) * size[case["dtype"]] + slots * 12
    return {"bytes": nbytes, "flops": 2.0 * slots * per + 2.0 * rows * case["experts"] * case["in"]}


# ---- the same from the definitions, in 64 bits --------------------------------

def _exact_keep(state, rows, dim, p):
    """The kept elements, by the generator's definition on unsigned 64-bit numbers of the host."""
    seed, call = (int(v) for v in state.tolist())
    u64, low = np.uint64, np.uint64(0xFFFFFFFF)
    chunks = -(-dim // 8)
    half = []
    for flag in (0, 1):
        c = [np.broadcast_to(np.arange(chunks, dtype=u64), (rows, chunks)),
             np.broadcast_to(np.arange(rows, dtype=u64)[:, None], (rows, chunks)),
             np.full((1, 1), call % 2 ** 32, dtype=u64), np.full((1, 1), (call >> 32) + flag * 2 ** 31, dtype=u64)]
        k = [seed % 2 ** 32, (seed >> 32) % 2 ** 32]
        for _ in range(10):
            p0, p1 = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
            c = [(p1 >> u64(32)) ^ c[1] ^ u64(k[0]), p1 & low, (p0 >> u64(32)) ^ c[3] ^ u64(k[1]), p0 & low]
            k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
        bits = np.empty((rows, chunks, 4, 2), dtype=np.uint32)
        for i in range(4):
            bits[:, :, i, 0] = c[i] & u64(0xFFFF)
            bits[:, :, i, 1] = c[i] >> u64(16)
        half.append(bits.reshape(rows, chunks * 8)[:, :dim])
    r = (half[0].astype(np.int64) << 16) | half[1]
    return torch.from_numpy(r >= round(p * 2 ** 32))


def _exact_residual(s):
    c = s["case"]
    v = {k: s[k].double().requires_grad_() for k in ("x", "y", "gate", "post_weight", "post_bias", "next_weight",
                                                    "next_bias") if s.get(k) is not None}

    def norm(u, which):
        if c["norm"] == "layer":
            u = u - u.mean(-1, keepdim=True)
        u = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + EPS) * v[which + "_weight"]
        return u + v[which + "_bias"] if which + "_bias" in v else u

    with torch.enable_grad():
        out, x = {}, v["x"]
        if not c["first"]:
            u = norm(v["y"], "post") if c["post"] else v["y"]
            if c["drop"]:
                u = u * (_exact_keep(s["state"], c["rows"], c["dim"], c["drop"]).to(u.device) / (1.0 - c["drop"]))
            x = x + 0.5 * u * v.get("gate", 1.0)
            out["out"] = x
        if c["next"] or c["first"]:
            out["h"] = norm(x, "next")
        given = [s["d" + k].double() for k in out]
        result = {k: t.detach() for k, t in out.items()}
        if c["train"]:
            grads = torch.autograd.grad(list(out.values()), list(v.values()), given)
            result.update(sorted(("d" + k, g) for k, g in zip(v, grads)))
    return result


def _exact_logprobs(s):
    c = s["case"]
    parts = []
    for r0 in range(0, c["rows"], max(1, 2 ** 27 // c["classes"])):
        rows = slice(r0, min(c["rows"], r0 + max(1, 2 ** 27 // c["classes"])))
        l, t = s["logits"][rows].double(), s["targets"][rows]
        lp = torch.log_softmax(l, -1)
        p = lp.exp()
        h = -torch.special.xlogy(p, p).sum(-1)
        has = t >= 0
        mine = lp.gather(1, t.clamp(min=0)[:, None])[:, 0]
        out = {"logp": torch.where(has, mine, 0.0), "entropy": h}
        if c["top"]:
            order = torch.argsort(l, dim=-1, descending=True, stable=True)[:, :c["top"]]
            value = lp.gather(1, order)
            out["top_logp"], out["top_indices"] = value, torch.where(value > -math.inf, order, -1)
        if c["train"]:
            g = torch.where(has, s["dlogp"][rows].double(), 0.0)
            d = -p * g[:, None] - s["dentropy"][rows].double()[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
            d[torch.arange(len(t), device=t.device), t.clamp(min=0)] += g
            out["dlogits"] = d
        parts.append(out)
    return {k: torch.cat([q[k] for q in parts]) for k in parts[0]}


def _exact_mixture(s):
    c = s["case"]
    x = s["x"].double()
    l = x @ s["gate"].double().t()
    p = torch.softmax(l, -1) if c["score"] == "softmax" else torch.sigmoid(l)
    key = p if s["bias"] is None else p + s["bias"].double()
    if c["groups"] > 1:
        by = key.view(key.shape[0], c["groups"], -1)
        value = by.topk(min(2, by.shape[-1]), -1).values.sum(-1)
        floor = value.topk(c["top_groups"], -1).values[:, -1:]
        key = torch.where((value >= floor)[..., None], by, -math.inf).view_as(key)
    idx = key.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = p.gather(1, idx)
    w = w / (w.sum(-1, keepdim=True) + RENORM_EPS)
    n = torch.arange(c["degree"] + 1, device=x.device, dtype=torch.float64)
    y = x.new_zeros(c["rows"], c["out"])
    for e in idx.unique().tolist():
        r, j = torch.nonzero(idx == e, as_tuple=True)
        phi = torch.cos(n * torch.acos(torch.tanh(x[r]))[..., None])
        z = torch.tensordot(phi, s["coeffs"][e].double().permute(0, 2, 1).contiguous(), dims=2)
        y.index_add_(0, r, z * w[r, j][:, None])
    return {"y": y, "weights": w, "indices": idx}


def exact(case, seed):
    if case.get("drop", case.get("p")) and case["rows"] * case["dim"] > 2 ** 27:
        return None  # the host's generator would take too long
    s = prepare(case, seed)
    if case["kind"] == "residual":
        return _exact_residual(s)
    if case["kind"] == "dropout":
        keep = _exact_keep(s["state"], case["rows"], case["dim"], case["p"]).cuda()
        factor = keep.double() / (1.0 - case["p"])
        out = {"y": s["x"].double() * factor}
        if case["train"]:
            out["dx"] = s["dy"].double() * factor
        return out
    return _exact_logprobs(s) if case["kind"] == "logprobs" else _exact_mixture(s)
