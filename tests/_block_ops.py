"""Definitions in 64 bits of the routing and the block seams, for their tests.

Each gradient comes with the sums of the magnitudes that its terms have, which
is what the rounding errors of its f32 evaluation are proportional to.
"""
from __future__ import annotations

import numpy as np
import torch

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
# f16's smallest step is 2^-24 (subnormals), the others' far below every value here
TINY = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}
F32 = 2.0 ** -24
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- routing -------------------------------------------------------------------

def scores(row, scoring):
    s = np.zeros(row.size)
    live = row > -np.inf
    if scoring == "sigmoid":
        s[live] = 1.0 / (1.0 + np.exp(-row[live]))
    elif live.any():
        e = np.exp(row[live] - row[live].max())
        s[live] = e / e.sum()
    return s


def route(logits, k, scoring="softmax", bias=None, groups=1, top_groups=None, group_top=2,
          renormalize=True, scale=1.0, eps=1e-9):
    """(idx, w, counts) of (T, E) f64 logits."""
    T, E = logits.shape
    per = E // groups
    idx, w = np.full((T, k), -1), np.zeros((T, k))
    for r in range(T):
        l = logits[r]
        s = scores(l, scoring)
        rank = s + bias if bias is not None else s if groups > 1 else l
        rank = np.where(np.isnan(rank), np.inf, rank)
        cand = [e for e in range(E) if l[e] != -np.inf and rank[e] != -np.inf]
        if groups > 1:
            worth = []
            for g in range(groups):
                best = sorted((rank[e] for e in cand if e // per == g), reverse=True)[:group_top]
                worth.append((-sum(best) if best else np.inf, g))
            kept = {g for _, g in sorted(worth)[:top_groups or groups]}
            cand = [e for e in cand if e // per in kept]
        sel = sorted(sorted(cand, key=lambda e: (-rank[e], e))[:k])
        idx[r, :len(sel)] = sel
        v = s[sel]
        w[r, :len(sel)] = scale * (v / (v.sum() + eps) if renormalize else v)
    return idx, w, np.bincount(idx[idx >= 0], minlength=E)


def route_grad(logits, idx, dw, scoring="softmax", renormalize=True, scale=1.0, eps=1e-9):
    """(dlogits, the sums of the magnitudes of its terms) by the formulas."""
    T, E = logits.shape
    dl, mag = np.zeros((T, E)), np.zeros((T, E))
    for r in range(T):
        s = scores(logits[r], scoring)
        ds, m = np.zeros(E), np.zeros(E)
        sel = [(e, dw[r, t]) for t, e in enumerate(idx[r]) if 0 <= e < E]
        total = sum(s[e] for e, _ in sel) + eps
        dot = sum(s[e] * d for e, d in sel)
        adot = sum(s[e] * abs(d) for e, d in sel)
        for e, d in sel:
            ds[e] += scale * ((d - dot / total) / total if renormalize else d)
            m[e] += abs(scale) * ((abs(d) + adot / total) / total if renormalize else abs(d))
        if scoring == "sigmoid":
            dl[r], mag[r] = ds * s * (1 - s), m * s * (1 - s)
        else:
            dl[r], mag[r] = s * (ds - (s * ds).sum()), s * (m + (s * m).sum())
    return dl, mag


def spread(logits, scoring):
    """What an exponential's argument can reach: its relative error is that many half steps."""
    with np.errstate(invalid="ignore"):
        a = np.abs(logits - logits.max(-1, keepdims=True)) if scoring == "softmax" else np.abs(logits)
    a = a[np.isfinite(a)]
    return float(a.max()) if a.size else 0.0


# ---- block seams ----------------------------------------------------------------

def rms(v, eps):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)


def ones(p, like, D):
    return torch.ones(D, dtype=like.dtype) if p is None else p


def seam(x, y, gate, shift, scale, post_norm, post_w, norm_w, alpha, eps):
    """(out, h) of f64 tensors (B, S, D); parameters (B, D) and (D,) or None."""
    D = y.shape[-1]
    n = rms(y, eps) * ones(post_w, y, D) if post_norm else y
    out = alpha * x + (n if gate is None else n * gate[:, None])
    h = rms(out, eps) * ones(norm_w, y, D)
    if scale is not None:
        h = h * (1.0 + scale[:, None])
    return out, h if shift is None else h + shift[:, None]


def seam_errors(x, y, gate, shift, scale, post_norm, post_w, norm_w, alpha, eps, dtype):
    """Bounds on the errors of (out, h): half a step of the output's type, and f32
    roundings: 6 products and sums and the mean's (a tree of at most 24 levels, halved by the
    root) come to 24 half steps of the terms' magnitudes in out; h carries out's errors, its
    mean's and 6 more."""
    D = y.shape[-1]
    out, h = seam(x, y, gate, shift, scale, post_norm, post_w, norm_w, alpha, eps)
    n = rms(y, eps) * ones(post_w, y, D) if post_norm else y
    eo = 24 * F32 * (abs(alpha * x) + abs(n if gate is None else n * gate[:, None]))
    r = torch.rsqrt(out.square().mean(-1, keepdim=True) + eps)
    f = ones(norm_w, y, D) * (1.0 if scale is None else 1.0 + scale[:, None])
    # the mean of squares moves with every element of out
    er = r ** 3 * (out.abs() * eo).mean(-1, keepdim=True) + 24 * F32 * r
    eh = (f * r).abs() * eo + (f * out).abs() * er + 6 * F32 * h.abs()
    if shift is not None:
        eh = eh + 2 * F32 * shift.abs()[:, None]
    return (out, eo + HALF[dtype] * (out.abs() + eo) + TINY[dtype],
            h, eh + HALF[dtype] * (h.abs() + eh) + TINY[dtype])


def seam_grad(dout, dh, out, y, gate, scale, post_norm, post_w, norm_w, alpha, eps):
    """The gradients by the formulas (f64), and for each the magnitudes of its terms."""
    some = dout if dout is not None else dh
    B, S, D = some.shape
    zero = torch.zeros_like(some)
    d, m = (zero, zero) if dout is None else (dout, dout.abs())
    got, mag = {}, {}
    if dh is not None:
        w = ones(norm_w, some, D)
        r = torch.rsqrt(out.square().mean(-1, keepdim=True) + eps)
        unit = out * r
        f = w if scale is None else w * (1.0 + scale[:, None])
        g = dh * f
        d = d + r * (g - unit * (g * unit).mean(-1, keepdim=True))
        m = m + r * (g.abs() + unit.abs() * (g * unit).abs().mean(-1, keepdim=True))
        q, mq = (dh * unit).sum(1), (dh * unit).abs().sum(1)
        got["dshift"], mag["dshift"] = dh.sum(1), dh.abs().sum(1)
        got["dscale"], mag["dscale"] = q * w, mq * w.abs()
        f1 = 1.0 if scale is None else 1.0 + scale
        got["dnorm_w"], mag["dnorm_w"] = (q * f1).sum(0), (mq * abs(f1)).sum(0)
    got["dx"], mag["dx"] = alpha * d, abs(alpha) * m
    if y is not None:
        gt = torch.ones(B, D, dtype=some.dtype) if gate is None else gate
        dn, mn = d * gt[:, None], m * gt.abs()[:, None]
        w = ones(post_w if post_norm else None, some, D)
        if post_norm:
            ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
            yn = y * ry
            gy, my = dn * w, mn * w.abs()
            got["dy"] = ry * (gy - yn * (gy * yn).mean(-1, keepdim=True))
            mag["dy"] = ry * (my + yn.abs() * (my * yn.abs()).mean(-1, keepdim=True))
        else:
            yn = y
            got["dy"], mag["dy"] = dn, mn
        p, mp = (d * yn).sum(1), (m * yn.abs()).sum(1)
        got["dgate"], mag["dgate"] = p * w, mp * w.abs()
        if post_norm:
            got["dpost_w"], mag["dpost_w"] = (p * gt).sum(0), (mp * gt.abs()).sum(0)
    return got, mag


def seam_grad_bound(name, want, mag, rows, dtype):
    """dx and dy: two means (24 levels each, one inside the other) and about 20 roundings
    besides, 96 half steps of f32 of the terms' magnitudes, then half a step of the type.
    The parameters' gradients: as many per term, and one per row summed."""
    if name in ("dx", "dy"):
        e = 96 * F32 * mag
        return e + HALF[dtype] * (want.abs() + e) + TINY[dtype]
    return (96 + rows) * F32 * mag
