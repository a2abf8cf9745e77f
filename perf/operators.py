"""The operators around the gated delta rule in a hybrid decoder's layers, measured: the residual addition with its RMS
norm (also with an 8-bit output), rotary positions, and causal attention with a sliding window and first tokens that stay
visible (training, prefill, and the single-token step over a cache).

`own` picks what run() calls: the plain forms below (32-bit torch operations, rounded once at the end) or this
repository's kernels."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-ai-engineering_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from macai_b200 import norm, rotary, window_attention
    return norm, rotary, window_attention


# ---- the cases

def listed():
    return [
        # one decoding step of a few requests: only latency counts
        {"name": "norm-token", "op": "norm", "rows": 4, "D": 2048, "dtype": "bf16", "wtype": "bf16",
         "zero_centered": False, "train": False},
        # a prefill whose projections take 8-bit inputs, a scale for every 128 channels
        {"name": "norm-fp8-prefill", "op": "norm8", "rows": 16384, "D": 4096, "dtype": "bf16", "wtype": "bf16",
         "zero_centered": False, "group": 128},
        # a training step's norm, an odd number of rows (packed tokens), the weight kept in float32 as 1 + w
        {"name": "norm-train", "op": "norm", "rows": 32771, "D": 2048, "dtype": "bf16", "wtype": "fp32",
         "zero_centered": True, "train": True},
        # decoding: one token of eight requests, a quarter of a wide head rotated
        {"name": "rotary-token", "op": "rotary", "B": 8, "T": 1, "H": 16, "HK": 2, "D": 256, "rot": 64,
         "interleaved": False, "factor": 1.0, "fused": True, "dtype": "bf16", "train": False},
        # a training step: q and k are views of one fused projection, a quarter of the head rotated
        {"name": "rotary-train", "op": "rotary", "B": 4, "T": 4096, "H": 16, "HK": 4, "D": 128, "rot": 32,
         "interleaved": False, "factor": 1.0, "fused": True, "dtype": "bf16", "train": True},
        # the benchmark's batch of the rule, as the attention layer between its layers sees it
        {"name": "attention-train", "op": "attention", "B": 4, "Tq": 1024, "Tk": 1024, "H": 16, "HK": 4, "D": 128,
         "window": 256, "sinks": 4, "dtype": "bf16", "train": True, "packed": 0},
        # long rows, the window well inside them
        {"name": "attention-train-long", "op": "attention", "B": 1, "Tq": 8192, "Tk": 8192, "H": 16, "HK": 4, "D": 128,
         "window": 2048, "sinks": 16, "dtype": "bf16", "train": True, "packed": 0},
        # 256-wide heads without a window
        {"name": "attention-train-wide", "op": "attention", "B": 2, "Tq": 2048, "Tk": 2048, "H": 8, "HK": 2, "D": 256,
         "window": 0, "sinks": 0, "dtype": "bf16", "train": True, "packed": 0},
        # packed rows of odd lengths, a head width that fills no tile, fp16
        {"name": "attention-train-packed", "op": "attention", "B": 1, "Tq": 4093, "Tk": 4093, "H": 12, "HK": 3, "D": 96,
         "window": 512, "sinks": 0, "dtype": "fp16", "train": True, "packed": 7},
        # a long prompt, narrow heads
        {"name": "attention-prefill", "op": "attention", "B": 1, "Tq": 16384, "Tk": 16384, "H": 16, "HK": 2, "D": 64,
         "window": 4096, "sinks": 4, "dtype": "bf16", "train": False, "packed": 0},
        # one request, a short cache: latency
        {"name": "step-token", "op": "step", "B": 1, "S": 1024, "low": 777, "high": 777, "idle": 0, "H": 16, "HK": 2,
         "D": 256, "window": 0, "sinks": 0, "dtype": "bf16"},
        # serving: rolling caches of requests of all ages, two slots idle
        {"name": "step-serving", "op": "step", "B": 64, "S": 4160, "low": 100, "high": 60000, "idle": 2, "H": 32, "HK": 4,
         "D": 128, "window": 4096, "sinks": 64, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm8", "rotary", "attention", "attention", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("norm", "norm8"):
        D = rng.choice([_log(rng, 64, 8192), 8 * _log(rng, 16, 1024), rng.choice([1024, 2048, 4096, 5120])])
        if op == "norm":
            dtype = rng.choice(["bf16", "fp16", "fp32"])
        rows = _log(rng, 1, min(32768, (1 << (25 if dtype == "fp32" else 26)) // D))
        if op == "norm":
            return {"op": op, "rows": rows, "D": D, "dtype": dtype, "wtype": rng.choice([dtype, "fp32"]),
                    "zero_centered": rng.random() < 0.5, "train": rng.random() < 0.6}
        return {"op": op, "rows": rows, "D": D, "dtype": dtype, "wtype": rng.choice([dtype, "fp32"]),
                "zero_centered": rng.random() < 0.5, "group": rng.choice([0, 32, 64, 128])}
    if op == "rotary":
        HK = rng.choice([1, 2, 4, 8])
        H, D = HK * rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 256])
        B = rng.choice([1, 2, 4, 8])
        T = _log(rng, 1, min(16384, (1 << 26) // (B * (H + HK) * D)))
        return {"op": op, "B": B, "T": T, "H": H, "HK": HK, "D": D, "rot": rng.choice([D, D // 2, D // 4]),
                "interleaved": rng.random() < 0.5, "factor": rng.choice([1.0, 4.0, 8.0]), "fused": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "train": rng.random() < 0.5}
    HK, D = rng.choice([1, 2, 4]), rng.choice([64, 72, 96, 128, 128, 256])
    if op == "attention":
        H, B = HK * rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4])
        train = rng.random() < 0.7
        most = 8 * 4096 * 4096 if train else 16 * 8192 * 8192
        Tk = _log(rng, 1, min(8192, int(math.sqrt(most / (B * H)))))
        packed = rng.choice([0, 0, 2, 5]) if Tk >= 16 else 0
        if packed:
            B = 1
        Tq = Tk if packed or train or rng.random() < 0.5 else _log(rng, 1, Tk)
        return {"op": op, "B": B, "Tq": Tq, "Tk": Tk, "H": H, "HK": HK, "D": D, "window": rng.choice([0, 1, _log(rng, 2, 4096), 512]),
                "sinks": rng.choice([0, 1, 4, 130]), "dtype": dtype, "train": train, "packed": packed}
    B, H = _log(rng, 1, 64), HK * rng.choice([1, 2, 4, 8])
    sinks = rng.choice([0, 4, 64])
    window = rng.choice([0, _log(rng, 16, 4096)])
    S = _log(rng, 64, min(32768, (1 << 27) // (B * HK * D))) if not window else sinks + window + rng.choice([0, 1, 60])
    high = S - 1 if not window else _log(rng, 2, 100000)
    return {"op": op, "B": B, "S": S, "low": rng.randint(0, high), "high": high, "idle": rng.choice([0, 0, 1]) if B > 1 else 0,
            "H": H, "HK": HK, "D": D, "window": window, "sinks": sinks, "dtype": dtype}


# ---- what the cases' plain values stand for

def _splits(case):
    """The packed rows' boundaries: `packed` sequences of uneven, mostly odd lengths (one of them may be empty)."""
    r, T, n = random.Random(case["packed"] * 1000003 + case["Tq"]), case["Tq"], case["packed"]
    return [0] + sorted(r.randint(0, T) for _ in range(n - 1)) + [T]


def _lengths(case):
    """Tokens in each request's cache before the step: evenly spread, the last `idle` slots without a request (-1)."""
    B, low, high = case["B"], case["low"], case["high"]
    n = [low + (high - low) * i // max(1, B - 1) for i in range(B)]
    return n[:B - case["idle"]] + [-1] * case["idle"]


def _pairs(Tq, Tk, window, sinks):
    """Visible (query, key) pairs of one head of one row."""
    p = np.arange(Tq, dtype=np.int64) + Tk - Tq
    p = p[p >= 0]
    w = window or 1 << 40
    return int((np.minimum(p + 1, w) + np.minimum(sinks, np.maximum(0, p + 1 - w))).sum())


def _visible(case, lengths):
    """Positions a step reads, over all requests."""
    w = min(case["window"] or 1 << 40, case["S"] - case["sinks"]) if max(lengths) >= case["S"] else case["window"] or 1 << 40
    return sum(min(n + 1, w) + min(case["sinks"], max(0, n + 1 - w)) for n in lengths if n >= 0)


def work(case):
    e = SIZES[case["dtype"]]
    if case["op"] in ("norm", "norm8"):
        n = case["rows"] * case["D"]
        if case["op"] == "norm8":
            groups = -(-case["D"] // (case["group"] or case["D"]))
            return {"bytes": 3 * n * e + n + 4 * case["rows"] * groups, "flops": 8 * n}
        return {"bytes": (8 if case["train"] else 4) * n * e, "flops": (20 if case["train"] else 6) * n}
    if case["op"] == "rotary":
        tokens = case["B"] * case["T"]
        n = tokens * (case["H"] + case["HK"]) * case["D"]
        ways = 2 if case["train"] else 1
        return {"bytes": ways * (2 * n * e + 4 * tokens * case["rot"]), "flops": ways * 3 * n * case["rot"] // case["D"]}
    if case["op"] == "step":
        lengths = _lengths(case)
        seen = _visible(case, lengths)
        return {"bytes": 2 * e * case["D"] * (case["HK"] * seen + case["B"] * (case["H"] + 2 * case["HK"])),
                "flops": 4 * case["D"] * case["H"] * seen}
    if case["packed"]:
        cu = _splits(case)
        pairs = sum(_pairs(b - a, b - a, case["window"], case["sinks"]) for a, b in zip(cu, cu[1:]))
    else:
        pairs = case["B"] * _pairs(case["Tq"], case["Tk"], case["window"], case["sinks"])
    qo, kv = case["B"] * case["Tq"] * case["H"] * case["D"], case["B"] * case["Tk"] * case["HK"] * case["D"]
    return {"bytes": e * ((4 * qo + 4 * kv) if case["train"] else (2 * qo + 2 * kv)),
            "flops": (14 if case["train"] else 4) * case["D"] * case["H"] * pairs}


# ---- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    st = {"case": case}
    if case["op"] in ("norm", "norm8"):
        rows, D, wt = case["rows"], case["D"], DTYPES[case["wtype"]]
        st["x"], st["res"] = rand(rows, D, scale=0.5), rand(rows, D, scale=2.0)
        st["w"] = rand(D, scale=0.1, dtype=wt) if case["zero_centered"] else (1 + rand(D, scale=0.1, dtype=torch.float32)).to(wt)
        if case.get("train"):
            st["dy"], st["ds"] = rand(rows, D), rand(rows, D)
            for n in ("x", "res", "w"):
                st[n].requires_grad_(True)
        return st
    H, HK, D, B = case["H"], case["HK"], case["D"], case["B"]
    if case["op"] == "rotary":
        T, R = case["T"], case["rot"]
        if case["fused"]:  # views of one projection's output: q, k, v side by side
            qkv = rand(B, T, (H + 2 * HK) * D)
            st["q"] = qkv[..., :H * D].view(B, T, H, D)
            st["k"] = qkv[..., H * D:(H + HK) * D].view(B, T, HK, D)
        else:
            st["q"], st["k"] = rand(B, T, H, D), rand(B, T, HK, D)
        rows = 32768  # positions of the table
        freq = (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)) / case["factor"]
        angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
        st["table"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()  # [positions, rot / 2, 2]
        first = torch.randint(0, rows - T, (B, 1), generator=gen, device="cuda")
        st["positions"] = first + torch.arange(T, device="cuda")
        if case["train"]:
            st["dq"], st["dk"] = rand(B, T, H, D), rand(B, T, HK, D)
            for n in ("q", "k"):
                st[n] = st[n].detach().requires_grad_(True)
        return st
    st["window"] = case["window"] or None
    if case["op"] == "step":
        n = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        st["lengths"] = n[torch.randperm(B, generator=gen, device="cuda")].contiguous()
        st["q"], st["k"], st["v"] = rand(B, 1, H, D, scale=1.5), rand(B, 1, HK, D), rand(B, 1, HK, D)
        st["k_cache"], st["v_cache"] = rand(B, case["S"], HK, D), rand(B, case["S"], HK, D)
        return st
    st["q"] = rand(B, case["Tq"], H, D, scale=1.5)
    st["k"], st["v"] = rand(B, case["Tk"], HK, D), rand(B, case["Tk"], HK, D)
    st["cu"] = torch.tensor(_splits(case), dtype=torch.int32, device="cuda") if case["packed"] else None
    if case["train"]:
        st["do"] = rand(B, case["Tq"], H, D)
        for n in ("q", "k", "v"):
            st[n].requires_grad_(True)
    return st


# ---- the plain forms

def _plain_norm(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    w = st["w"].float() + (1.0 if case["zero_centered"] else 0.0)
    s = (st["x"].float() + st["res"].float()).to(dt)  # the residual stream, an output of its own: y is the norm of it
    sf = s.float()
    r = (sf.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh = sf * r
    y = xh * w
    if case["op"] == "norm8":
        rows, D = y.shape
        g = case["group"] or D
        pad = -D % g
        blocks = torch.cat([y, y.new_zeros(rows, pad)], -1).view(rows, -1, g) if pad else y.view(rows, -1, g)
        top = blocks.abs().amax(-1)
        scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
        q = (blocks / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        return {"q": q.view(rows, -1)[:, :D].contiguous(), "scale": scale, "s": s}
    out = {"y": y.to(dt), "s": s}
    if case["train"]:
        dy, ds = st["dy"].float(), st["ds"].float()
        h = dy * w
        d = (ds + r * (h - xh * (h * xh).mean(-1, keepdim=True))).to(dt)
        out.update(dx=d, dres=d, dw=(dy * xh).sum(0).to(st["w"].dtype))
    return out


def _turn(x, cos, sin, interleaved):
    """x [B, T, heads, D] in float32, its first 2 * cos.shape[-1] channels rotated in pairs."""
    n = cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_rotary(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    cos, sin = st["table"][st["positions"]].unbind(-1)
    il = case["interleaved"]
    with torch.no_grad():
        out = {"q": _turn(st["q"].float(), cos, sin, il).to(dt), "k": _turn(st["k"].float(), cos, sin, il).to(dt)}
        if case["train"]:
            out["dq"] = _turn(st["dq"].float(), cos, -sin, il).to(dt)
            out["dk"] = _turn(st["dk"].float(), cos, -sin, il).to(dt)
    return out


def _mask(case, cu, device):
    """[Tq, Tk]: what each query sees."""
    Tq, Tk, w = case["Tq"], case["Tk"], case["window"] or 1 << 40
    j = torch.arange(Tk, device=device)
    if case["packed"]:
        seq = torch.searchsorted(cu[1:].long(), j, right=True)
        p = j - cu.long()[seq]
        same = seq[:, None] == seq[None, :]
        return same & (p[None, :] <= p[:, None]) & ((p[None, :] > p[:, None] - w) | (p[None, :] < case["sinks"]))
    p = (torch.arange(Tq, device=device) + Tk - Tq)[:, None]
    return (j <= p) & ((j > p - w) | (j < case["sinks"]))


def _plain_attention(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    B, Tq, Tk, H, HK, D = (case[n] for n in ("B", "Tq", "Tk", "H", "HK", "D"))
    G, scale = H // HK, D ** -0.5
    with torch.no_grad():
        q = st["q"].float().view(B, Tq, HK, G, D).permute(0, 2, 3, 1, 4)           # [B, HK, G, Tq, D]
        k, v = (st[n].float().permute(0, 2, 1, 3).unsqueeze(2) for n in ("k", "v"))  # [B, HK, 1, Tk, D]
        seen = _mask(case, st["cu"], q.device)
        s = (torch.matmul(q, k.transpose(-1, -2)).mul_(scale)).masked_fill_(~seen, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = s.sub_(torch.where(m.isinf(), torch.zeros_like(m), m)).exp_()
        p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
        o = torch.matmul(p, v)
        back = lambda x, n: x.permute(0, 3, 1, 2, 4).reshape(B, -1, n, D).to(dt)  # noqa: E731
        out = {"o": back(o, H)}
        if case["train"]:
            do = st["do"].float().view(B, Tq, HK, G, D).permute(0, 2, 3, 1, 4)
            dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
            dp = torch.matmul(do, v.transpose(-1, -2))
            ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            out["dq"] = back(torch.matmul(ds, k), H)
            out["dk"] = back(torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True), HK)
            out["dv"] = back(dv, HK)
    return out


def _slots(case, lengths):
    """(slot of the new token, [B, S] positions that the slots hold after it, -1 where none)."""
    S, sinks = case["S"], case["sinks"]
    j = torch.arange(S, device=lengths.device)
    p = lengths.long()[:, None]
    ring = S - sinks
    slot = torch.where(p < S, p, sinks + (p - sinks).clamp_min(0) % ring)
    # the newest position congruent to the slot; slots below `sinks` keep the first tokens
    last = p - (p - j) % ring
    held = torch.where((p < S) | (j < sinks), j.expand_as(last), last)
    return slot, torch.where(held <= p, held, -torch.ones_like(held))


def _plain_step(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    B, S, H, HK, D = (case[n] for n in ("B", "S", "H", "HK", "D"))
    live = st["lengths"] >= 0
    slot, held = _slots(case, st["lengths"])
    rows, at = torch.arange(B, device=slot.device), slot[:, 0].clamp(0, S - 1)
    for c, x in (("k_cache", "k"), ("v_cache", "v")):
        st[c][rows, at] = torch.where(live[:, None, None], st[x][:, 0], st[c][rows, at])
    w = case["window"] or 1 << 40
    p = st["lengths"].long()[:, None]
    seen = (held >= 0) & ((held > p - w) | (held < case["sinks"])) & live[:, None]
    q = st["q"].float().view(B, HK, H // HK, D)
    s = torch.einsum("bhgd,bshd->bhgs", q, st["k_cache"].float()) * D ** -0.5
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = (s - torch.where(m.isinf(), torch.zeros_like(m), m)).exp()
    e = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.einsum("bhgs,bshd->bhgd", e, st["v_cache"].float())
    return {"o": o.reshape(B, 1, H, D).to(dt), "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _plain(st):
    op = st["case"]["op"]
    with torch.no_grad():
        return {"norm": _plain_norm, "norm8": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention,
                "step": _plain_step}[op](st)


# ---- one pass

def run(st):
    if not own:
        return _plain(st)
    norm, rot, attn = _package()
    case = st["case"]
    if case["op"] == "norm":
        y, s = norm.add_rms_norm(st["x"], st["res"], st["w"], EPS, zero_centered=case["zero_centered"])
        out = {"y": y, "s": s}
        if case["train"]:
            dx, dres, dw = torch.autograd.grad([y, s], [st["x"], st["res"], st["w"]], [st["dy"], st["ds"]])
            out = {"y": y.detach(), "s": s.detach(), "dx": dx, "dres": dres, "dw": dw}
        return out
    if case["op"] == "norm8":
        q, scale, s = norm.add_rms_norm_fp8(st["x"], st["res"], st["w"], EPS, group=case["group"] or None,
                                            zero_centered=case["zero_centered"])
        return {"q": q, "scale": scale, "s": s}
    if case["op"] == "rotary":
        q, k = rot.rotary(st["q"], st["k"], st["table"], st["positions"], interleaved=case["interleaved"])
        out = {"q": q, "k": k}
        if case["train"]:
            dq, dk = torch.autograd.grad([q, k], [st["q"], st["k"]], [st["dq"], st["dk"]])
            out = {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
        return out
    if case["op"] == "step":
        o = attn.window_attention_step(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["lengths"],
                                       window=st["window"], sinks=case["sinks"])
        return {"o": o, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    o = attn.window_attention(st["q"], st["k"], st["v"], window=st["window"], sinks=case["sinks"], cu_seqlens=st["cu"])
    if not case["train"]:
        return {"o": o}
    dq, dk, dv = torch.autograd.grad(o, [st["q"], st["k"], st["v"]], st["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


# ---- the definitions in 64 bits, row by row and head by head

def _exact_norm(st):
    case = st["case"]
    s = (st["x"].double() + st["res"].double()).to(DTYPES[case["dtype"]])
    x, w = s.double(), st["w"].double()
    if case["zero_centered"]:
        w = 1.0 + w
    rms = torch.sqrt((x * x).sum(-1, keepdim=True) / case["D"] + EPS)
    y = x / rms * w
    if case["op"] == "norm8":
        g = case["group"] or case["D"]
        tops = torch.stack([c.abs().amax(-1) for c in y.split(g, -1)], -1)
        scale = torch.where(tops > 0, tops / E4M3_MAX, torch.ones_like(tops))
        return {"q": y / scale.repeat_interleave(g, -1)[:, :case["D"]], "scale": scale, "s": s.double()}
    out = {"y": y, "s": s.double()}
    if case["train"]:
        g = st["dy"].double() * w
        d = st["ds"].double() + g / rms - x * (g * x).sum(-1, keepdim=True) / (case["D"] * rms ** 3)
        out.update(dx=d, dres=d, dw=(st["dy"].double() * x / rms).sum(0))
    return out


def _exact_rotary(st):
    case = st["case"]
    n = case["rot"] // 2
    t = st["table"].double()[st["positions"]]
    unit = torch.complex(t[..., 0], t[..., 1])[:, :, None]

    def turn(x, u):
        y = x.double().clone()
        at = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if case["interleaved"] else (slice(0, n), slice(n, 2 * n))
        z = torch.complex(y[..., at[0]].contiguous(), y[..., at[1]].contiguous()) * u
        y[..., at[0]], y[..., at[1]] = z.real, z.imag
        return y

    out = {x: turn(st[x], unit) for x in ("q", "k")}
    if case["train"]:
        out.update({x: turn(st[x], unit.conj()) for x in ("dq", "dk")})
    return out


def _exact_attention(st):
    case = st["case"]
    B, Tq, Tk, H, HK, D, W, sinks = (case[n] for n in ("B", "Tq", "Tk", "H", "HK", "D", "window", "sinks"))
    if case["packed"]:
        cu = _splits(case)
        parts = [(0, slice(a, b), slice(a, b)) for a, b in zip(cu, cu[1:]) if b > a]
    else:
        parts = [(b, slice(0, Tq), slice(0, Tk)) for b in range(B)]
    out = {"o": torch.zeros(B, Tq, H, D, dtype=torch.float64, device="cuda")}
    if case["train"]:
        out.update(dq=torch.zeros_like(out["o"]), dk=torch.zeros(B, Tk, HK, D, dtype=torch.float64, device="cuda"),
                   dv=torch.zeros(B, Tk, HK, D, dtype=torch.float64, device="cuda"))
    for b, rq, rk in parts:
        at = torch.arange(rk.stop - rk.start, device="cuda")
        behind = at[rk.stop - rk.start - (rq.stop - rq.start):][:, None] - at if rq.stop - rq.start <= rk.stop - rk.start else \
            torch.arange(rk.stop - rk.start - (rq.stop - rq.start), rk.stop - rk.start, device="cuda")[:, None] - at
        hidden = behind < 0
        if W:
            hidden |= (behind >= W) & (at >= sinks)
        for h in range(H):
            q, k, v = st["q"][b, rq, h].double(), st["k"][b, rk, h * HK // H].double(), st["v"][b, rk, h * HK // H].double()
            x = q @ k.T / math.sqrt(D)
            x[hidden] = -math.inf
            top = x.max(-1, keepdim=True).values
            e = torch.exp(x - torch.nan_to_num(top, neginf=0.0))
            total = e.sum(-1, keepdim=True)
            p = e / torch.where(total > 0, total, torch.ones_like(total))
            out["o"][b, rq, h] = p @ v
            if case["train"]:
                g = st["do"][b, rq, h].double()
                out["dv"][b, rk, h * HK // H] += p.T @ g
                dp = g @ v.T
                dx = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                out["dq"][b, rq, h] = dx @ k
                out["dk"][b, rk, h * HK // H] += dx.T @ q
    return out


def _exact_step(st):
    case = st["case"]
    S, sinks, H, HK, D = (case[n] for n in ("S", "sinks", "H", "HK", "D"))
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    o = torch.zeros(case["B"], 1, H, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lengths"].tolist()):
        if n < 0:
            continue
        place = lambda p: p if p < sinks or n < S else sinks + (p - sinks) % (S - sinks)  # noqa: E731
        kc[b, place(n)], vc[b, place(n)] = st["k"][b, 0].double(), st["v"][b, 0].double()
        from_ = max(0, n + 1 - case["window"]) if case["window"] else 0
        seen = torch.tensor([place(p) for p in list(range(min(sinks, from_))) + list(range(from_, n + 1))], device="cuda")
        k, v = kc[b, seen], vc[b, seen]
        for h in range(HK):
            g = slice(h * H // HK, (h + 1) * H // HK)
            p = torch.softmax(st["q"][b, 0, g].double() @ k[:, h].T / math.sqrt(D), -1)
            o[b, 0, g] = p @ v[:, h]
    return {"o": o, "k_cache": kc, "v_cache": vc}


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "norm8": _exact_norm, "rotary": _exact_rotary, "attention": _exact_attention,
                "step": _exact_step}[case["op"]](st)
