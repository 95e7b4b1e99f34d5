"""float64 restatements of the operators around the retention core: rotary
positions, the residual-norm seam with its gradients, and the filtered draw.

Written from the definitions (see each function) without the library's code.
``seam64`` also returns, for every output, the sum of the absolute values of
the terms it is made of: what an fp32 evaluation's rounding errors are
relative to.
"""
from __future__ import annotations

import math

import numpy as np


def rotary64(x, inv_freq, positions, layout="interleaved", scale=1.0, inverse=False):
    """x [..., T, heads, dim] turned by position * inv_freq; positions broadcast
    against x.shape[:-2]."""
    x = np.asarray(x, np.float64)
    f = np.asarray(inv_freq, np.float64)
    half = f.size
    th = np.broadcast_to(np.asarray(positions, np.float64), x.shape[:-2])[..., None, None] * f
    if inverse:
        th = -th
    a_at = slice(0, 2 * half, 2) if layout == "interleaved" else slice(0, half)
    b_at = slice(1, 2 * half, 2) if layout == "interleaved" else slice(half, 2 * half)
    out = x.copy()
    a, b = x[..., a_at], x[..., b_at]
    out[..., a_at] = scale * (a * np.cos(th) - b * np.sin(th))
    out[..., b_at] = scale * (a * np.sin(th) + b * np.cos(th))
    return out


def swish64(g):
    g = np.asarray(g, np.float64)
    with np.errstate(over="ignore"):
        return np.where(np.isneginf(g), 0.0, np.where(np.isneginf(g), 0.0, g) / (1.0 + np.exp(-g)))


def seam64(x, h, gate=None, post_w=None, scale=None, pre_w=None, alpha=1.0, eps=1e-6, dz=None, dy=None,
           grads=False):
    """n = RMSNorm(h) post_w; z = alpha x + scale swish(gate) n; y = RMSNorm(z)
    pre_w, and with `grads` the gradients for dz, dy (None: zero).  Returns
    (values, magnitudes), dicts by name."""
    f = lambda v: None if v is None else np.asarray(v, np.float64)  # noqa: E731
    x, h, gate, post_w, scale, pre_w, dz, dy = (f(v) for v in (x, h, gate, post_w, scale, pre_w, dz, dy))
    d = x.shape[-1]
    r1 = 1.0 / np.sqrt((h * h).sum(-1, keepdims=True) / d + eps)
    hh = h * r1
    n = h if post_w is None else hh * post_w
    sw = 1.0 if gate is None else swish64(gate)
    s = 1.0 if scale is None else scale
    m = s * sw * n
    z = alpha * x + m
    zmag = np.abs(alpha * x) + np.abs(m)
    v, mag = {"z": z}, {"z": zmag}
    r2 = 1.0 / np.sqrt((z * z).sum(-1, keepdims=True) / d + eps)
    if pre_w is not None:
        v["y"], mag["y"] = z * r2 * pre_w, zmag * r2 * np.abs(pre_w)
    if not grads:
        return v, mag
    mean = lambda t: t.sum(-1, keepdims=True) / d  # noqa: E731
    dz = np.zeros_like(z) if dz is None else dz
    Z, Zm = dz, np.abs(dz)
    if pre_w is not None:
        dy = np.zeros_like(z) if dy is None else dy
        zh, zhm = z * r2, zmag * r2
        t = dy * pre_w
        Z = dz + r2 * (t - zh * mean(t * zh))
        Zm = np.abs(dz) + r2 * (np.abs(t) + zhm * mean(np.abs(t) * zhm))
        v["pre_w"], mag["pre_w"] = (dy * zh).sum(0), (np.abs(dy) * zhm).sum(0)
    v["x"], mag["x"] = alpha * Z, abs(alpha) * Zm
    if scale is not None:
        v["scale"], mag["scale"] = (Z * sw * n).sum(0), (Zm * np.abs(sw * n)).sum(0)
    if gate is not None:
        sg = 1.0 / (1.0 + np.exp(-gate))
        slope = sg * (1.0 + gate * (1.0 - sg))
        v["gate"] = Z * s * n * slope
        mag["gate"] = Zm * np.abs(s * n) * (sg * (1.0 + np.abs(gate) * (1.0 - sg)))
    N, Nm = Z * s * sw, Zm * np.abs(s * sw)
    if post_w is None:
        v["h"], mag["h"] = N, Nm
    else:
        v["post_w"], mag["post_w"] = (N * hh).sum(0), (Nm * np.abs(hh)).sum(0)
        t = N * post_w
        v["h"] = r1 * (t - hh * mean(t * hh))
        tm = Nm * np.abs(post_w)
        mag["h"] = r1 * (tm + np.abs(hh) * mean(tm * np.abs(hh)))
    return v, mag


def sample64(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, penalty=1.0, context=()):
    """(token, log-probability, margin) of one row of logits: the order is by
    logit (largest first, equal ones by index), top-k the first k, top-p
    through the first place whose running share exceeds it, min-p those at
    least min_p times the likeliest, then the first place whose running share
    of the kept mass reaches u.  The margin is how far, in shares, the nearest
    border that decides is."""
    row = np.asarray(row, np.float32).copy()
    V = row.size
    seen = sorted({int(t) for t in context if 0 <= int(t) < V})
    if seen and penalty != 1.0:
        pen = np.float32(penalty)
        row[seen] = np.where(row[seen] > 0, row[seen] / pen, row[seen] * pen)
    row[np.isnan(row)] = -np.inf
    live = np.flatnonzero(row > -np.inf)
    if live.size == 0:
        return -1, -math.inf, 1.0
    order = live[np.lexsort((live, -row[live].astype(np.float64)))]
    if not temperature > 1e-4:
        return int(order[0]), 0.0, 1.0
    if top_k > 0:
        order = order[:top_k]
    top = float(row[order[0]])
    if math.isinf(top):
        w = (row[order] == np.inf).astype(np.float64)
        order, w = order[w > 0], w[w > 0]
    else:
        w = np.exp((row[order].astype(np.float64) - top) / float(np.float32(temperature)))
    margin = 1.0
    run = np.cumsum(w)
    z = run[-1]
    keep = w.size
    p = float(np.float32(top_p))
    if not p >= 1.0:
        p = max(p, 0.0) if p == p else 0.0
        keep = min(keep, 1 + int(np.searchsorted(run, p * z, side="right")))
        if p > 0:
            margin = min(margin, float(np.min(np.abs(run / z - p))))
    mp = float(np.float32(min_p))
    if mp > 0:
        mp = min(mp, 1.0)
        n = int((w >= mp).sum())
        if mp < 1.0:
            margin = min(margin, float(np.min(np.abs(w / mp - 1.0))))
        keep = min(keep, n)
    mass = run[keep - 1]
    share = run[:keep] / mass
    u = min(max(float(np.float32(u)), 0.0), 1.0 - 2.0 ** -24)
    i = min(int(np.searchsorted(share, u, side="left")), keep - 1)
    if u > 0 and keep > 1:
        margin = min(margin, float(np.min(np.abs(share[:-1] - u))))
    return int(order[i]), math.log(w[i]) - math.log(mass), margin
