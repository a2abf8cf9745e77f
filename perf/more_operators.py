"""The operators that a hybrid decoder needs around its mixers, measured: the gated feed-forward block (trained, prefilled,
and for the few tokens of a decoding step), the softmax cross entropy of a vocabulary projection that never keeps the
logits (scored and trained), and the gated delta rule's recurrent form over a pool of states (single tokens and short runs).

`own` picks what run() calls: the plain forms below (32-bit torch operations, rounded once at the end) or this
repository's kernels."""
import math
import os
import sys

import torch

own = False

L2_EPS = 1e-6
IGNORED = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-ai-engineering_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from macai_b200 import feed_forward, gated_delta, loss
    return feed_forward, loss, gated_delta


# ---- the cases

def listed():
    return [
        # one decoding step of a few requests
        {"name": "ff-token", "op": "ff", "rows": 4, "D": 2048, "F": 6144, "dtype": "bf16", "train": False},
        # a decoding step of a full server
        {"name": "ff-serving", "op": "ff", "rows": 64, "D": 4096, "F": 12288, "dtype": "bf16", "train": False},
        # a prompt, its length no multiple of a tile
        {"name": "ff-prefill", "op": "ff", "rows": 2050, "D": 4096, "F": 12288, "dtype": "fp16", "train": False},
        # a training step's batch, 8 x 2,048 tokens
        {"name": "ff-train", "op": "ff", "rows": 16384, "D": 2048, "F": 6144, "dtype": "bf16", "train": True},
        # packed rows of a small model, widths that fill no tile
        {"name": "ff-train-ragged", "op": "ff", "rows": 4093, "D": 1000, "F": 2728, "dtype": "fp16", "train": True},
        # scoring a text: the loss of every token, no gradient, a vocabulary of odd size
        {"name": "loss-score", "op": "loss", "rows": 777, "D": 2048, "V": 50257, "dtype": "bf16", "train": False,
         "reduction": "none", "ignored": 0.0},
        # a training step's batch over a large vocabulary, some of it padding
        {"name": "loss-train", "op": "loss", "rows": 8192, "D": 2048, "V": 128000, "dtype": "bf16", "train": True,
         "reduction": "mean", "ignored": 0.1},
        # a small model's fine-tuning step: prompts are ignored, every token has a weight of its own
        {"name": "loss-train-weighted", "op": "loss", "rows": 1500, "D": 768, "V": 32003, "dtype": "fp16", "train": True,
         "reduction": "none", "ignored": 0.5},
        # one request's token: latency
        {"name": "rule-token", "op": "rule", "B": 1, "T": 1, "HK": 16, "H": 32, "DK": 128, "DV": 128, "dtype": "bf16",
         "vtype": "bf16", "spare": 3, "idle": 0},
        # serving: one token of each request, some slots idle, the convolution path's float32 values
        {"name": "rule-serving", "op": "rule", "B": 128, "T": 1, "HK": 16, "H": 32, "DK": 128, "DV": 128,
         "dtype": "bf16", "vtype": "fp32", "spare": 5, "idle": 3},
        # drafted tokens run from the kept states into spare slots
        {"name": "rule-drafts", "op": "rule", "B": 24, "T": 6, "HK": 16, "H": 16, "DK": 128, "DV": 128, "dtype": "fp16",
         "vtype": "fp16", "spare": 0, "idle": 1},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ff", "ff", "loss", "loss", "rule"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "ff":
        D, F = 8 * _log(rng, 8, 512), 8 * _log(rng, 16, 1536)
        train = rng.random() < 0.5
        rows = _log(rng, 1, min(16384, 16384 * 2048 * 6144 // (D * F)))
        return {"op": op, "rows": rows, "D": D, "F": F, "dtype": dtype, "train": train}
    if op == "loss":
        D, V = 8 * _log(rng, 8, 512), _log(rng, 2, 131072)
        train = rng.random() < 0.7
        rows = _log(rng, 1, min(16384, 8192 * 128000 // V, 8192 * 2048 * 128000 // (V * D)))
        return {"op": op, "rows": rows, "D": D, "V": V, "dtype": dtype, "train": train,
                "reduction": rng.choice(["mean", "sum", "none"]), "ignored": rng.choice([0.0, 0.1, 0.6])}
    HK = rng.choice([1, 2, 4, 8, 16])
    H, DK, DV = HK * rng.choice([1, 2, 4]), rng.choice([32, 64, 96, 128, 128, 128]), rng.choice([64, 96, 128, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    B = _log(rng, 1, min(256, (1 << 26) // (H * DK * DV)))
    T = rng.choice([1, 1, 1, _log(rng, 2, 16)])
    return {"op": op, "B": B, "T": T, "HK": HK, "H": H, "DK": DK, "DV": DV, "dtype": dtype,
            "vtype": rng.choice([dtype, "fp32"]), "spare": rng.choice([0, 1, 7]), "idle": rng.choice([0, 0, 1]) if B > 1 else 0}


def work(case):
    e = SIZES[case["dtype"]]
    if case["op"] == "ff":
        n, f = case["rows"], case["D"] * case["F"]
        if case["train"]:  # x, y and their gradients, the weights and theirs
            return {"bytes": e * (4 * n * case["D"] + 6 * f), "flops": 18 * n * f}
        return {"bytes": e * (2 * n * case["D"] + 3 * f), "flops": 6 * n * f}
    if case["op"] == "loss":
        n, wide = case["rows"], case["D"] * case["V"]
        ways = 2 if case["train"] else 1
        losses = n if case["reduction"] == "none" else 1
        return {"bytes": ways * e * (n * case["D"] + wide) + 8 * n + 4 * losses * ways,
                "flops": (6 if case["train"] else 2) * n * wide}
    live, T = case["B"] - case["idle"], case["T"]
    rows = 2 * case["HK"] * case["DK"] * e + case["H"] * case["DV"] * (e + SIZES[case["vtype"]]) + 8 * case["H"]
    state = case["H"] * case["DK"] * case["DV"]
    return {"bytes": live * (8 * state + T * rows), "flops": 7 * live * T * state}


# ---- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    st = {"case": case}
    if case["op"] == "ff":
        n, D, F = case["rows"], case["D"], case["F"]
        st["x"] = rand(n, D)  # a norm's output
        st["w_gate"], st["w_up"] = rand(F, D, scale=D ** -0.5), rand(F, D, scale=D ** -0.5)
        st["w_down"] = rand(D, F, scale=F ** -0.5)
        if case["train"]:
            st["dy"] = rand(n, D, scale=0.05)
            for name in ("x", "w_gate", "w_up", "w_down"):
                st[name].requires_grad_(True)
        return st
    if case["op"] == "loss":
        n, D, V = case["rows"], case["D"], case["V"]
        st["weight"] = rand(V, D, scale=1.5 * D ** -0.5)
        labels = torch.randint(0, V, (n,), generator=gen, device="cuda")
        # from rows that know nothing of their label to rows that are nearly sure of it
        sure = 4.0 * torch.rand(n, 1, generator=gen, device="cuda")
        st["x"] = (torch.randn(n, D, generator=gen, device="cuda") + sure * st["weight"][labels].float()).to(dt)
        drop = torch.rand(n, generator=gen, device="cuda") < case["ignored"]
        st["labels"] = torch.where(drop, torch.full_like(labels, IGNORED), labels)
        if case["train"]:
            scale = 1.0 if case["dtype"] == "bf16" else 4096.0  # float16 trains with a scaled loss
            if case["reduction"] == "none":
                st["g"] = scale / n * (0.25 + torch.rand(n, generator=gen, device="cuda"))
            else:
                st["g"] = torch.tensor(scale if case["reduction"] == "mean" else scale / n, device="cuda")
            st["x"].requires_grad_(True)
            st["weight"].requires_grad_(True)
        return st
    B, T, HK, H, DK, DV = (case[n] for n in ("B", "T", "HK", "H", "DK", "DV"))
    st["q"], st["k"], st["v"] = rand(B, T, HK, DK), rand(B, T, HK, DK), rand(B, T, H, DV, dtype=DTYPES[case["vtype"]])
    st["beta"] = torch.sigmoid(rand(B, T, H, dtype=torch.float32))
    rate = torch.exp(torch.rand(H, generator=gen, device="cuda") * math.log(16.0))
    st["g"] = -rate * torch.nn.functional.softplus(rand(B, T, H, dtype=torch.float32) - 4.0)
    slots = 2 * B + case["spare"]
    st["state"] = rand(slots, H, DK, DV, scale=0.1, dtype=torch.float32)
    # each live request has a slot that it reads and a spare one that it writes, so that the state before the tokens stays
    order = torch.randperm(slots, generator=gen, device="cuda").to(torch.int32)
    live = torch.randperm(B, generator=gen, device="cuda") >= case["idle"]
    none = torch.full((B,), -1, dtype=torch.int32, device="cuda")
    st["slots"] = torch.where(live, order[:B], none).contiguous()
    st["out_slots"] = torch.where(live, order[B:2 * B], none).contiguous()
    st["live"] = live.nonzero()[:, 0]  # a server knows which of its requests these are
    return st


# ---- the plain forms

def _plain_ff(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    x, wg, wu, wd = (st[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    gate, up = x @ wg.T, x @ wu.T
    s = torch.sigmoid(gate)
    a = gate * s
    h = a * up
    out = {"y": (h @ wd.T).to(dt)}
    if case["train"]:
        dy = st["dy"].float()
        out["dw_down"] = (dy.T @ h).to(dt)
        dh = dy @ wd
        dup = dh * a
        dgate = dh * up * (s * (1.0 + gate * (1.0 - s)))
        out["dx"] = (dgate @ wg + dup @ wu).to(dt)
        out["dw_gate"], out["dw_up"] = (dgate.T @ x).to(dt), (dup.T @ x).to(dt)
    return out


def _plain_loss(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    x, w, labels = st["x"].float(), st["weight"].float(), st["labels"]
    kept = labels != IGNORED
    at = torch.where(kept, labels, torch.zeros_like(labels))[:, None]
    logits = x @ w.T
    top = logits.amax(-1, keepdim=True)
    target = logits.gather(-1, at) - top
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    losses = torch.where(kept, (total.log() - target)[:, 0], torch.zeros_like(total[:, 0]))
    count = kept.sum()
    out = {"loss": losses if case["reduction"] == "none" else losses.sum() / (count if case["reduction"] == "mean" else 1)}
    if case["train"]:
        g = st["g"] / count if case["reduction"] == "mean" else st["g"]
        g = torch.where(kept, g.expand(case["rows"]), torch.zeros_like(losses))[:, None]
        d = p.mul_(g / total)
        d.scatter_add_(-1, at, -g)
        out["dx"], out["dweight"] = (d @ w).to(dt), (d.T @ x).to(dt)
    return out


def _plain_rule(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    T, rep, DK = case["T"], case["H"] // case["HK"], case["DK"]
    live = st["live"]
    q, k, v, beta = (st[n][live].float() for n in ("q", "k", "v", "beta"))
    q = (q * (q.square().sum(-1, keepdim=True) + L2_EPS).rsqrt() * DK ** -0.5).repeat_interleave(rep, 2)
    k = (k * (k.square().sum(-1, keepdim=True) + L2_EPS).rsqrt()).repeat_interleave(rep, 2)
    a = st["g"][live].exp()[..., None, None]
    s = st["state"][st["slots"][live]]
    o = torch.zeros(case["B"], T, case["H"], case["DV"], dtype=dt, device=s.device)
    for t in range(T):  # a recurrence: each token needs the state that the one before left
        s = s * a[:, t]
        d = beta[:, t, :, None] * (v[:, t] - torch.matmul(k[:, t, :, None], s)[:, :, 0])
        s = s + k[:, t, :, :, None] * d[:, :, None]
        o[live, t] = torch.matmul(q[:, t, :, None], s)[:, :, 0].to(dt)
    st["state"][st["out_slots"][live]] = s
    return {"o": o, "state": st["state"]}


def _plain(st):
    with torch.no_grad():
        return {"ff": _plain_ff, "loss": _plain_loss, "rule": _plain_rule}[st["case"]["op"]](st)


# ---- one pass

def run(st):
    if not own:
        return _plain(st)
    feed_forward, loss, gated_delta = _package()
    case = st["case"]
    if case["op"] == "ff":
        y = feed_forward.gated_feed_forward(st["x"], st["w_gate"], st["w_up"], st["w_down"])
        if not case["train"]:
            return {"y": y}
        dx, dwg, dwu, dwd = torch.autograd.grad(y, [st["x"], st["w_gate"], st["w_up"], st["w_down"]], st["dy"])
        return {"y": y.detach(), "dw_down": dwd, "dx": dx, "dw_gate": dwg, "dw_up": dwu}
    if case["op"] == "loss":
        value = loss.linear_cross_entropy(st["x"], st["weight"], st["labels"], ignore_index=IGNORED,
                                          reduction=case["reduction"])
        if not case["train"]:
            return {"loss": value}
        dx, dw = torch.autograd.grad(value, [st["x"], st["weight"]], st["g"])
        return {"loss": value.detach(), "dx": dx, "dweight": dw}
    o = gated_delta.gated_delta_step(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"], st["slots"],
                                     st["out_slots"], use_qk_l2norm_in_kernel=True)
    return {"o": o, "state": st["state"]}


# ---- the definitions in 64 bits

def _exact_ff(st):
    case = st["case"]
    x, wg, wu, wd = (st[n].detach().double() for n in ("x", "w_gate", "w_up", "w_down"))
    out = {"y": torch.empty_like(x)}
    if case["train"]:
        out.update(dw_down=torch.zeros_like(wd), dx=torch.empty_like(x), dw_gate=torch.zeros_like(wg),
                   dw_up=torch.zeros_like(wu))
    for at in torch.arange(case["rows"], device=x.device).split(4096):  # tokens are independent
        g, u = torch.nn.functional.linear(x[at], wg), torch.nn.functional.linear(x[at], wu)
        h = torch.nn.functional.silu(g) * u
        out["y"][at] = torch.nn.functional.linear(h, wd)
        if case["train"]:
            dy = st["dy"][at].double()
            dh, e = torch.mm(dy, wd), torch.exp(-g)
            dg = dh * u * (1 + e + g * e) / (1 + e) ** 2  # d/dg of g / (1 + exp(-g))
            du = dh * g / (1 + e)
            out["dw_down"] += torch.mm(dy.t(), h)
            out["dw_gate"] += torch.mm(dg.t(), x[at])
            out["dw_up"] += torch.mm(du.t(), x[at])
            out["dx"][at] = torch.mm(dg, wg) + torch.mm(du, wu)
    return out


def _exact_loss(st):
    case = st["case"]
    x, w, labels = st["x"].detach().double(), st["weight"].detach().double(), st["labels"]
    n = case["rows"]
    losses = torch.zeros(n, dtype=torch.float64, device=x.device)
    valid = int((labels >= 0).sum())
    out = {}
    if case["train"]:
        out.update(dx=torch.zeros_like(x), dweight=torch.zeros_like(w))
        each = {"none": lambda: st["g"].double(), "sum": lambda: st["g"].double().repeat(n),
                "mean": lambda: st["g"].double().repeat(n) / valid}[case["reduction"]]()
    for at in (labels >= 0).nonzero()[:, 0].split(1024):
        logp = torch.log_softmax(torch.mm(x[at], w.t()), -1)
        here = torch.arange(len(at), device=x.device)
        losses[at] = -logp[here, labels[at]]
        if case["train"]:
            d = logp.exp_()
            d[here, labels[at]] -= 1.0
            d *= each[at][:, None]
            out["dx"][at] = torch.mm(d, w)
            out["dweight"].addmm_(d.t(), x[at])
    total = {"none": lambda: losses, "sum": losses.sum, "mean": lambda: losses.sum() / valid if valid else losses.sum() / 0.0}
    return {"loss": total[case["reduction"]](), **out}


def _exact_rule(st):
    case = st["case"]
    pool = st["state"].double()
    o = torch.zeros(case["B"], case["T"], case["H"], case["DV"], dtype=torch.float64, device=pool.device)
    live = (st["slots"] >= 0).nonzero()[:, 0]
    s = pool[st["slots"][live].long()]
    heads = torch.arange(case["H"], device=pool.device) * case["HK"] // case["H"]
    unit = lambda x: x / torch.sqrt((x * x).sum(-1, keepdim=True) + L2_EPS)  # noqa: E731
    for t in range(case["T"]):
        q, k = (unit(st[n][live, t].double())[:, heads] for n in ("q", "k"))
        s = s * torch.exp(st["g"][live, t].double())[..., None, None]
        wrong = st["v"][live, t].double() - torch.einsum("bhk,bhkv->bhv", k, s)
        s = s + torch.einsum("bhk,bhv->bhkv", k, wrong * st["beta"][live, t].double()[..., None])
        o[live, t] = torch.einsum("bhk,bhkv->bhv", q, s) / math.sqrt(case["DK"])
    pool[st["out_slots"][live].long()] = s
    return {"o": o, "state": pool}


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"ff": _exact_ff, "loss": _exact_loss, "rule": _exact_rule}[case["op"]](st)
