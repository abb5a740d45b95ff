"""Mixture-of-experts operators and the orthogonalised update, in 64 bits (numpy), from their definitions."""
from __future__ import annotations

import numpy as np

ROUTE_EPS = 1e-20


def route_scores(logits, score):
    """Scores [rows, experts]; an ineligible expert (-inf or NaN) scores 0."""
    l = np.asarray(logits, dtype=np.float64)
    open_ = l > -np.inf
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return np.where(open_, 1.0 / (1.0 + np.exp(-np.where(open_, l, 0.0))), 0.0), open_
    top = np.max(np.where(open_, l, -np.inf), axis=1, keepdims=True, initial=-np.inf)
    e = np.where(open_, np.exp(np.where(open_, l, 0.0) - np.where(np.isfinite(top), top, 0.0)), 0.0)
    total = e.sum(1, keepdims=True)
    return np.divide(e, total, out=np.zeros_like(e), where=total > 0), open_


def route(logits, top_k, score="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    """(weights, indices), one row at a time by sorting (key falling, index rising)."""
    s, open_ = route_scores(logits, score)
    rows, experts = s.shape
    key = np.where(open_, s if bias is None else s + np.asarray(bias, dtype=np.float64), -np.inf)
    idx = np.full((rows, top_k), -1, dtype=np.int64)
    size = experts // groups
    for r in range(rows):
        allowed = set(range(experts))
        if groups > 1:
            values = []
            for g in range(groups):
                k = np.sort(key[r, g * size:(g + 1) * size])[::-1]
                second = k[1] if size > 1 and np.isfinite(k[1]) else 0.0
                values.append((-(k[0] + second), g))
            kept = [g for _, g in sorted(values)[:top_groups]]
            allowed = {e for g in kept for e in range(g * size, (g + 1) * size)}
        order = sorted((e for e in allowed if key[r, e] > -np.inf), key=lambda e: (-key[r, e], e))
        idx[r, :min(top_k, len(order))] = order[:top_k]
    return route_weights(s, idx, renormalize, scale), idx


def route_weights(s, idx, renormalize=True, scale=1.0):
    chosen = np.where(idx >= 0, np.take_along_axis(s, np.maximum(idx, 0), 1), 0.0)
    if renormalize:
        chosen = chosen / (chosen.sum(1, keepdims=True) + ROUTE_EPS)
    return scale * chosen


def route_backward(logits, idx, dw, score="softmax", renormalize=True, scale=1.0):
    """dlogits for the choice ``idx`` held fixed."""
    s, open_ = route_scores(logits, score)
    c = np.where(idx >= 0, np.take_along_axis(s, np.maximum(idx, 0), 1), 0.0)
    dw = np.where(idx >= 0, np.asarray(dw, dtype=np.float64), 0.0) * scale
    if renormalize:
        total = c.sum(1, keepdims=True) + ROUTE_EPS
        dc = dw / total - (dw * c).sum(1, keepdims=True) / total ** 2
    else:
        dc = dw
    ds = np.zeros_like(s)
    for r, j in zip(*np.nonzero(idx >= 0)):
        ds[r, idx[r, j]] += dc[r, j]
    if score == "sigmoid":
        return ds * s * (1 - s)
    return s * (ds - (s * ds).sum(1, keepdims=True))


def orthogonalize(g, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """Newton-Schulz by its definition on one matrix [rows, cols]."""
    a, b, c = coefficients
    x = np.asarray(g, dtype=np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (np.sqrt((x * x).sum()) + eps)
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.T if tall else x


def coeff_matrix(c):
    """[in, out, D] coefficients as [out, in D]."""
    c = np.asarray(c)
    return c.transpose(1, 0, 2).reshape(c.shape[1], -1)


def muon_step(p, g, buf, lr, momentum=0.95, nesterov=True, weight_decay=0.0, **kw):
    """(p, buf) after a step; p a matrix [rows, cols] or coefficients [in, out, D]."""
    p, g, buf = (np.asarray(v, dtype=np.float64) for v in (p, g, buf))
    buf = momentum * buf + (1 - momentum) * g
    u = (1 - momentum) * g + momentum * buf if nesterov else buf
    if p.ndim == 3:
        i, o, d = p.shape
        up = orthogonalize(coeff_matrix(u), **kw).reshape(o, i, d).transpose(1, 0, 2)
        ratio = o / (i * d)
    else:
        up = orthogonalize(u, **kw)
        ratio = p.shape[0] / p.shape[1]
    return p * (1 - lr * weight_decay) - lr * np.sqrt(max(1.0, ratio)) * up, buf


def cheb(t, degree):
    """T_0..T_degree and their derivatives in t, in a last dimension (t away from +-1)."""
    theta = np.arccos(t)[..., None]
    n = np.arange(degree + 1)
    return np.cos(n * theta), n * np.sin(n * theta) / np.sin(theta)


def kan_experts(x, coeffs, indices, weights, dy=None):
    """y, and with dy also (dx, dcoeffs, dweights), one slot at a time."""
    x, coeffs, weights = (np.asarray(v, dtype=np.float64) for v in (x, coeffs, weights))
    experts, _, out, dd = coeffs.shape
    t = np.tanh(x)
    basis, slope = cheb(t, dd - 1)
    y = np.zeros((x.shape[0], out))
    dx, dc, dw = np.zeros_like(x), np.zeros_like(coeffs), np.zeros_like(weights)
    for (r, j), e in np.ndenumerate(np.asarray(indices)):
        if not 0 <= e < experts:
            continue
        z = np.einsum("id,iod->o", basis[r], coeffs[e])
        y[r] += weights[r, j] * z
        if dy is not None:
            dw[r, j] = z @ dy[r]
            g = weights[r, j] * np.asarray(dy[r], dtype=np.float64)
            dc[e] += basis[r][:, None, :] * g[None, :, None]
            dx[r] += np.einsum("iod,o,id->i", coeffs[e], g, slope[r]) * (1 - t[r] ** 2)
    return y if dy is None else (y, dx, dc, dw)
