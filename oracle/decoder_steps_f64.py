"""float64 definitions of the operators around a hybrid decoder's mixers (test infrastructure): the rule's recurrent form, the
gated feed-forward block, the cross entropy of a vocabulary projection. Plain loops and matrices; gradients by the formulas
(the tests also check them against differences). Each comes with bounds of what rounding may do, by first-order error
propagation: `eps` arguments are half steps (torch.finfo(t).eps / 2)."""
from __future__ import annotations

import math

import torch

E32 = 2.0 ** -24


def rule_step(q, k, v, g, beta, s0, l2norm=False):
    """(o, S, bound of o, bound of S) of the recurrence over [B, T, heads, D] inputs from s0 [B, H, DK, DV], in float64; the
    bounds are those of the same recurrence in float32 arithmetic (sums in any order), before o's own rounding."""
    B, T, HK, DK = q.shape
    H = v.shape[2]
    heads = torch.arange(H, device=q.device) // (H // HK)
    q, k, v, g, beta, S = (t.double() for t in (q, k, v, g, beta, s0))
    if l2norm:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    q, k = q[:, :, heads] / math.sqrt(DK), k[:, :, heads]
    # a normalised element: the squares' sum (DK + 2 roundings, halved by the root), rsqrt and the query's scale (2 ulp = 4
    # half steps each), two products
    ev = (DK / 2 + 1 + 8 + 2) * E32 if l2norm else 5 * E32
    dot = (DK + 1) * E32                        # a sum of DK products
    E = torch.zeros_like(S)                     # bound of |S computed - S|
    o, eo = [], []
    for t in range(T):
        a = torch.exp(g[:, t])[..., None, None]
        ea = (g[:, t].abs()[..., None, None] * 0 + 4 * E32) * a          # expf: 2 ulp
        kt, qt = k[:, t, :, :, None], q[:, t, :, :, None]
        Sa = S * a
        Ea = E * a + S.abs() * ea + Sa.abs() * E32
        u = (kt * Sa).sum(-2)
        eu = (kt.abs() * Ea).sum(-2) + (kt.abs() * Sa.abs()).sum(-2) * (dot + ev)
        b = beta[:, t, :, None]
        d = b * (v[:, t] - u)
        ed = b.abs() * eu + 3 * E32 * b.abs() * (v[:, t].abs() + u.abs())
        S = Sa + kt * d[:, :, None]
        E = Ea + kt.abs() * (ed + d.abs() * ev)[:, :, None] + 3 * E32 * (Sa.abs() + kt.abs() * d.abs()[:, :, None])
        o.append((qt * S).sum(-2))
        # o = a (S q) + (q k) d: every term's magnitude, with both dots' errors
        mag = (qt.abs() * (Sa.abs() + kt.abs() * d.abs()[:, :, None])).sum(-2)
        eo.append((qt.abs() * (Ea + kt.abs() * ed[:, :, None])).sum(-2) + mag * (dot + 2 * ev + 4 * E32))
    if not T:
        z = torch.zeros(B, 0, H, v.shape[3], dtype=torch.float64, device=q.device)
        return z, S, z, E
    return torch.stack(o, 1), S, torch.stack(eo, 1), E


# ---- products of 16-bit operands with float32 sums. A sum of n products is off by at most n times 2^-23 of the sum of their
# magnitudes: the adder may cut instead of rounding (one step, not half), in any order.
def _gamma(n):
    return (n + 32) * 2.0 ** -23


FAST = 2.0 ** -19    # of the few fast float32 operations (exp2, division) an elementwise value passes through


def _halves(dt):
    """(half a step of the type, relative; half a step of its subnormal numbers)"""
    return torch.finfo(dt).eps / 2, {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dt]


def feed_forward(x, wg, wu, wd, dy=None):
    """The block's outputs in float64 with the bounds of what the kernels' roundings may do to them before their own output
    rounding: {"y": (value, bound), ...}; with dy also dx, dw_gate, dw_up, dw_down. x [n, D]."""
    dt = x.dtype
    eps, tiny = _halves(dt)
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    D, F = x.shape[1], wg.shape[0]
    g, u = x @ wg.T, x @ wu.T
    eg, eu = _gamma(D) * (x.abs() @ wg.abs().T), _gamma(D) * (x.abs() @ wu.abs().T)
    s = torch.sigmoid(g)
    a, da = g * s, s * (1 + g * (1 - s))
    h = a * u

    def of_h(eg, eu):
        return u.abs() * (1.1 * eg + FAST * a.abs()) + (a.abs() + 1.1 * eg) * eu + FAST * h.abs()
    eh = of_h(eg, eu)
    eh = eh + eps * (h.abs() + eh) + tiny      # rounded: the second product's operand
    out = {"y": (h @ wd.T, eh @ wd.abs().T + _gamma(F) * ((h.abs() + eh) @ wd.abs().T))}
    if dy is None:
        return out
    dy = dy.double()
    n, O = dy.shape
    dh = dy @ wd
    edh = _gamma(O) * (dy.abs() @ wd.abs())
    kg, ku = eg + 2.0 ** -15 * g.abs(), eu + 2.0 ** -15 * u.abs()     # as kept: 24 of 32 bits
    kh = of_h(kg, ku)
    kh = kh + eps * (h.abs() + kh) + tiny
    du, dg = dh * a, dh * u * da
    edu = edh * a.abs() + (dh.abs() + edh) * (1.1 * kg + FAST * a.abs())
    edg = (edh * u.abs() + (dh.abs() + edh) * ku) * (da.abs() + 0.6 * kg) + dh.abs() * u.abs() * (0.6 * kg) + FAST * dg.abs() \
        + FAST * (dh * u).abs()
    # float16: both carry a power of two that brings their bound to 2^14 .. 2^15
    low = 0.0
    if dt == torch.float16:
        most = dy.abs().sum(1).max() * wd.abs().max() * torch.maximum(g.abs().max(), 1.1 * u.abs().max())
        low = float(most) * 2.0 ** -25 / 2.0 ** 13
    edu, edg = edu + eps * (du.abs() + edu) + low, edg + eps * (dg.abs() + edg) + low
    dga, dua = dg.abs() + edg, du.abs() + edu
    out["dx"] = (dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + _gamma(2 * F) * (dga @ wg.abs() + dua @ wu.abs()))
    out["dw_gate"] = (dg.T @ x, edg.T @ x.abs() + _gamma(n) * (dga.T @ x.abs()))
    out["dw_up"] = (du.T @ x, edu.T @ x.abs() + _gamma(n) * (dua.T @ x.abs()))
    out["dw_down"] = (dy.T @ h, dy.abs().T @ kh + _gamma(n) * (dy.abs().T @ (h.abs() + kh)))
    return out


def cross_entropy(x, w, labels, ignore=-100, g=None):
    """Each row's loss in float64 (0 where ignored) and its bound; with g [n], the rows' gradients of the loss, also dx and
    dweight with theirs: {"loss": (value, bound), ...}."""
    dt = x.dtype
    eps, tiny = _halves(dt)
    x, w = x.double(), w.double()
    n, D = x.shape
    V = w.shape[0]
    kept = labels != ignore
    at = torch.where(kept, labels, torch.zeros_like(labels)).long()[:, None]
    l = x @ w.T
    el = _gamma(D) * (x.abs() @ w.abs().T)
    lse = torch.logsumexp(l, -1, keepdim=True)
    p = torch.exp(l - lse)
    # the logits' errors weighted as they enter the sum; a sum of V exponentials; the logarithm in units of log2
    else_ = (p * el).sum(-1, keepdim=True) * 1.1 + FAST + _gamma(8) * lse.abs()
    loss = torch.where(kept, (lse - l.gather(-1, at))[:, 0], torch.zeros_like(lse[:, 0]))
    eloss = torch.where(kept, (else_ + el.gather(-1, at) + _gamma(8) * l.gather(-1, at).abs())[:, 0], torch.zeros_like(lse[:, 0]))
    out = {"loss": (loss, eloss)}
    if g is None:
        return out
    gr = torch.where(kept, g.double(), torch.zeros_like(g.double()))[:, None]
    # (a probability below the smallest normal number 2^-126 may come out as 0: ex2.approx.ftz gives no subnormal numbers)
    ep = p * (el + else_ + _gamma(8) * l.abs()) * 1.1 + FAST * p + 2.0 ** -126
    d = p.clone()
    d.scatter_add_(-1, at, -torch.ones_like(at, dtype=torch.float64))
    top = float(gr.abs().max()) if n else 0.0
    low = top * (2.0 ** -25 / 2.0 ** 15 if dt == torch.float16 else 0.0)
    ed = gr.abs() * (ep + eps * (d.abs() + ep) + 2.0 ** -22 * d.abs()) + low * kept[:, None]
    d = d * gr
    da = d.abs() + ed
    out["dx"] = (d @ w, ed @ w.abs() + _gamma(V) * (da @ w.abs()))
    out["dweight"] = (d.T @ x, ed.T @ x.abs() + _gamma(n) * (da.T @ x.abs()))
    return out


def outside(got, want, bound, dt):
    """The largest excess of |got - want| over the bound and the output's own rounding to dt (at most 0 where it holds)."""
    if not want.numel():
        return 0.0
    eps, tiny = (2.0 ** -24, 0.0) if dt == torch.float32 else _halves(dt)
    return float(((got.double() - want).abs() - (bound + eps * (want.abs() + bound) + tiny)).max())
