"""The operators around a deep KAN's layers in 64 bits (numpy), from their definitions: norms around a
residual block, dropout's mask, log probabilities.

``residual`` and ``log_probs`` return with each result the size that its roundings are relative to: the same
expression with every term's absolute value.
"""
from __future__ import annotations

import numpy as np


def keep_mask(seed, call, rows, dim, p):
    """The kept elements [rows, dim]: Philox 4x32-10 on (column / 8, row, call), two 16-bit halves an element."""
    low, u64 = np.uint64(0xFFFFFFFF), np.uint64
    chunks = -(-dim // 8)
    seed, call = int(seed) % 2 ** 64, int(call) % 2 ** 63
    halves = []
    for flag in (0, 1):
        c = [np.broadcast_to(np.arange(chunks, dtype=u64)[None], (rows, chunks)),
             np.broadcast_to(np.arange(rows, dtype=u64)[:, None], (rows, chunks)),
             np.full((rows, chunks), call & 0xFFFFFFFF, dtype=u64),
             np.full((rows, chunks), (call >> 32) | flag << 31, dtype=u64)]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
            c = [b >> u64(32) ^ c[1] ^ u64(k[0]), b & low, a >> u64(32) ^ c[3] ^ u64(k[1]), a & low]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        words = np.stack(c, -1)
        halves.append(np.stack([words & u64(0xFFFF), words >> u64(16)], -1).reshape(rows, chunks * 8)[:, :dim])
    number = (halves[0] << u64(16) | halves[1]).astype(np.int64)
    return number >= int(np.rint(p * 2.0 ** 32))


def _norm(v, mag, norm, eps):
    """(normalised rows, their size, 1 / root mean square)."""
    mean = v.mean(-1, keepdims=True) if norm == "layer" else 0.0
    size = mag + (mag.mean(-1, keepdims=True) if norm == "layer" else 0.0)
    r = 1.0 / np.sqrt(((v - mean) ** 2).mean(-1, keepdims=True) + eps)
    return (v - mean) * r, size * r, r


def _norm_backward(g, gmag, hat, hatmag, r, norm):
    d = g - hat * (g * hat).mean(-1, keepdims=True)
    mag = gmag + hatmag * (gmag * hatmag).mean(-1, keepdims=True)
    if norm == "layer":
        d, mag = d - g.mean(-1, keepdims=True), mag + gmag.mean(-1, keepdims=True)
    return r * d, r * mag


def residual(x, y=None, *, norm="rms", eps=1e-6, post_weight=None, post_bias=None, gate=None, scale=1.0, keep=None,
             p=0.0, next_weight=None, next_bias=None, dout=None, dh=None):
    """{name: (value, size)} of out, h and, where dout or dh is given, the gradients of all inputs."""
    res = {}
    o, omag = x, np.abs(x)
    if y is not None:
        u, umag = y, np.abs(y)
        if post_weight is not None:
            yhat, yhatmag, r1 = _norm(y, np.abs(y), norm, eps)
            u, umag = yhat * post_weight, yhatmag * np.abs(post_weight)
            if post_bias is not None:
                u, umag = u + post_bias, umag + np.abs(post_bias)
        factor = 1.0 if keep is None else np.where(keep, 1.0 / (1.0 - p) if p < 1 else 0.0, 0.0)
        u, umag = u * factor, umag * factor
        gt = scale * (1.0 if gate is None else gate)
        o, omag = x + gt * u, np.abs(x) + np.abs(gt) * umag
        res["out"] = o, omag
    if next_weight is not None:
        ohat, ohatmag, r2 = _norm(o, omag, norm, eps)
        h, hmag = ohat * next_weight, ohatmag * np.abs(next_weight)
        if next_bias is not None:
            h, hmag = h + next_bias, hmag + np.abs(next_bias)
        res["h"] = h, hmag
    if dout is None and dh is None:
        return res
    g = np.zeros_like(x) if dout is None else dout
    gmag = np.abs(g)
    if dh is not None and next_weight is not None:
        a = np.abs(dh)
        res["next_weight"] = (dh * ohat).sum(0), (a * ohatmag).sum(0)
        if next_bias is not None:
            res["next_bias"] = dh.sum(0), a.sum(0)
        d, dmag = _norm_backward(dh * next_weight, a * np.abs(next_weight), ohat, ohatmag, r2, norm)
        g, gmag = g + d, gmag + dmag
    res["x"] = g, gmag
    if y is not None:
        if gate is not None:
            dg, dgmag = scale * g * u, np.abs(scale) * gmag * umag
            res["gate"] = (dg.sum(0), dgmag.sum(0)) if gate.ndim == 1 else (dg, dgmag)
        g, gmag = gt * factor * g, np.abs(gt) * factor * gmag
        if post_weight is not None:
            res["post_weight"] = (g * yhat).sum(0), (gmag * yhatmag).sum(0)
            if post_bias is not None:
                res["post_bias"] = g.sum(0), gmag.sum(0)
            g, gmag = _norm_backward(g * post_weight, gmag * np.abs(post_weight), yhat, yhatmag, r1, norm)
        res["y"] = g, gmag
    return res


def log_probs(logits, targets, top=0):
    """(logp, entropy, top_logp, top_indices, log p): a row at a time."""
    rows, classes = logits.shape
    logp, entropy = np.zeros(rows), np.zeros(rows)
    top_logp, top_idx = np.full((rows, top), -np.inf), np.full((rows, top), -1, dtype=np.int64)
    every = np.full((rows, classes), -np.inf)
    for r in range(rows):
        l = logits[r]
        there = ~(l == -np.inf)
        t = int(targets[r])
        has = 0 <= t < classes
        if not there.any():
            logp[r] = -np.inf if has else 0.0
            continue
        if np.isnan(l).any() or (l == np.inf).any():
            every[r], entropy[r], logp[r] = np.nan, np.nan, np.nan if has else 0.0
        else:
            m = int(np.argmax(l))
            e = np.exp(l - l[m])
            e[m] = 0.0
            lp = (l - l[m]) - np.log1p(e.sum())
            every[r] = lp
            logp[r] = lp[t] if has else 0.0
            entropy[r] = -(np.exp(lp[there]) * lp[there]).sum()
        order = sorted((c for c in range(classes) if l[c] > -np.inf), key=lambda c: (-l[c], c))[:top]
        top_idx[r, :len(order)] = order
        top_logp[r, :len(order)] = every[r, order]
    return logp, entropy, top_logp, top_idx, every


def log_probs_backward(logits, targets, dlogp, dentropy):
    """(dlogits, size)."""
    rows, classes = logits.shape
    _, entropy, _, _, lp = log_probs(logits, targets)
    p = np.exp(lp)
    finite = np.where(p > 0, lp, 0.0)
    has = (targets >= 0) & (targets < classes) & (lp > -np.inf).any(1)
    g = np.where(has, dlogp, 0.0)[:, None]
    dH = np.asarray(dentropy)[:, None]
    d = -p * (g + dH * (finite + entropy[:, None]))
    size = p * (np.abs(g) + np.abs(dH) * (np.abs(finite) + entropy[:, None]))
    at = np.arange(rows), np.where(has, targets, 0)
    m = np.where(has, -np.expm1(lp[at]), 0.0)  # 1 - p of the target
    d[at] = np.where(has, g[:, 0] * m - p[at] * dH[:, 0] * (finite[at] + entropy), d[at])
    size[at] = np.where(has, np.abs(g[:, 0]) * m + p[at] * np.abs(dH[:, 0]) * (np.abs(finite[at]) + entropy), size[at])
    return d, size
