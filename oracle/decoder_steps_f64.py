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
