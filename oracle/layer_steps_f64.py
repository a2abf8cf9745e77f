"""float64 definitions of the softmax-attention layer's steps around the rule (test infrastructure): the residual RMS norm
with its 8-bit form, rotary positions, and causal attention with a sliding window and first tokens that stay visible.
Plain loops and matrices; gradients by the formulas (the tests also check them against differences)."""
from __future__ import annotations

import math

import torch


def rms_norm(x, residual, w, eps=1e-6, zero_centered=False):
    """(y, s): s = x + residual rounded to x's dtype, y in float64 from that s."""
    s = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    s64 = s.double()
    y = s64 / torch.sqrt((s64 * s64).mean(-1, keepdim=True) + eps) * (w.double() + (1.0 if zero_centered else 0.0))
    return y, s


def rms_norm_backward(s, w, dy, ds, eps=1e-6, zero_centered=False):
    """(dx, dw, |terms of dx|, |terms of dw|): the last two bound what cancels."""
    s, w, dy, ds = s.double(), w.double() + (1.0 if zero_centered else 0.0), dy.double(), ds.double()
    r = 1.0 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    xh, h = s * r, dy * w
    m = (h * xh).mean(-1, keepdim=True)
    dx = ds + r * (h - xh * m)
    big = ds.abs() + r * (h.abs() + xh.abs() * (h * xh).abs().mean(-1, keepdim=True))
    rows = tuple(range(s.dim() - 1))
    return dx, (dy * xh).sum(rows), big, (dy * xh).abs().sum(rows)


def fp8_scales(y, group):
    """(scale [..., ceil(D / group)], y / its scale) in float64."""
    D = y.shape[-1]
    g = group or D
    tops = torch.stack([c.abs().amax(-1) for c in y.split(g, -1)], -1)
    scale = torch.where(tops > 0, tops / 448.0, torch.ones_like(tops))
    return scale, y / scale.repeat_interleave(g, -1)[..., :D]


def rotary(x, table, positions, interleaved=False, inverse=False):
    """x [B, T, H, D] turned in float64; positions [T] or [B, T]."""
    n = table.shape[1]
    t = table.double()[positions.clamp(0, table.shape[0] - 1).long()]
    t = t.expand(x.shape[0], *t.shape[-3:]) if t.dim() == 3 else t
    c, s = t[..., 0][:, :, None], t[..., 1][:, :, None] * (-1.0 if inverse else 1.0)
    y = x.double().clone()
    ia, ib = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def visible(Tq, Tk, window=None, sinks=0, device=None):
    """[Tq, Tk] bool: query i stands at position i + Tk - Tq."""
    p = (torch.arange(Tq, device=device) + Tk - Tq)[:, None]
    j = torch.arange(Tk, device=device)[None]
    seen = j <= p
    if window is not None:
        seen &= (j > p - window) | (j < sinks)
    return seen


def attention(q, k, v, window=None, sinks=0, scale=None, do=None):
    """q [B, Tq, H, D], k, v [B, Tk, HK, D]: o, or (o, dq, dk, dv) with a cotangent, in float64. A query without a visible
    key gets zeros."""
    B, Tq, H, D = q.shape
    Tk, HK = k.shape[1:3]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    seen = visible(Tq, Tk, window, sinks, q.device)
    Q = q.double().transpose(1, 2)                                                     # [B, H, Tq, D]
    K, V = (t.double().transpose(1, 2).repeat_interleave(H // HK, 1) for t in (k, v))
    e = torch.exp((Q @ K.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf).sub_(
        (Q @ K.transpose(-1, -2) * scale).masked_fill(~seen, -1e300).amax(-1, keepdim=True) if Tk else 0.0))
    z = e.sum(-1, keepdim=True)
    P = e / torch.where(z > 0, z, torch.ones_like(z))
    o = (P @ V).transpose(1, 2)
    if do is not None:
        G = do.double().transpose(1, 2)
        dP = G @ V.transpose(-1, -2)
        dS = P * (dP - (P * dP).sum(-1, keepdim=True)) * scale
        dq = (dS @ K).transpose(1, 2)
        dk, dv = ((t.transpose(-1, -2) @ x).unflatten(1, (HK, H // HK)).sum(2).transpose(1, 2) for t, x in ((dS, Q), (P, G)))
    return o if do is None else (o, dq, dk, dv)


def attention_step(q, k, v, k_cache, v_cache, lengths, window=None, sinks=0, scale=None):
    """(o [B, 1, H, D], k_cache, v_cache) in float64 after one token for each request (copies: nothing in place)."""
    B, _, H, D = q.shape
    S, HK = k_cache.shape[1:3]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    kc, vc = k_cache.double().clone(), v_cache.double().clone()
    o = torch.zeros(B, 1, H, D, dtype=torch.float64, device=q.device)
    first = min(sinks, S - 1)
    ring = S - first
    for b, p in enumerate(lengths.tolist()):
        if p < 0:
            continue

        def slot(j):
            return j if j < S else first + (j - first) % ring
        kc[b, slot(p)], vc[b, slot(p)] = k[b, 0].double(), v[b, 0].double()
        w = p + 1 if window is None else window
        if p >= S:
            w = min(w, ring)
        since = max(0, p - w + 1)
        at = torch.tensor([slot(j) for j in list(range(min(first, since))) + list(range(since, p + 1))], device=q.device)
        K, V = kc[b, at].repeat_interleave(H // HK, 1), vc[b, at].repeat_interleave(H // HK, 1)   # [n, H, D]
        P = torch.softmax((K * q[b, 0].double()).sum(-1) * scale, 0)
        o[b, 0] = (P[..., None] * V).sum(0)
    return o, kc, vc
