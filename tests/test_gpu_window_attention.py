"""Sliding-window attention with first tokens that stay visible (macai_b200.window_attention) against its float64 formulas.

Tolerances. u is the unit roundoff of the inputs' type (2^-8 bf16, 2^-11 fp16): P and dS are rounded to it once, as the
operands of the matrix instruction, and each result once more. So, per element, with A the sum of the absolute values of the
terms that a result adds up (formed in float64):
    o   within u |o| + (u + f) sum_j P |v|         dv  within u |dv| + (u + f) sum_i P |do|
    dq  within u |dq| + scale sum_j |k| ((u + f) |dS| + P (u C + f B)),   dk likewise with |q| and sums over i,
B_i = sum_d |do_id| max_j |v_jd| bounding dP, and u C_i = u sum_j P |dP| what the rounding of P in o makes of
delta = rowsum(do o). f = 6e-5 covers what is fp32: scores (sums of D products, so
256 * 2^-24 of at most 16 in size, as a relative error of P), exp2 (2^-22), the running sums, delta from o as a pair of
16-bit values (2^-16)."""
import pytest
import torch

from oracle import layer_steps_f64 as ref

gpu = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, HF: 2.0 ** -11}
ETA = {BF: 1e-30, HF: 2.0 ** -25}   # half the spacing of fp16's subnormals
F = 6e-5
DEV = "cuda"


def _inputs(B, Tq, Tk, H, HK, D, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (1.5 * torch.randn(B, Tq, H, D, generator=g)).to(dt).to(DEV)
    k, v = (torch.randn(B, Tk, HK, D, generator=g).to(dt).to(DEV) for _ in range(2))
    return q, k, v, torch.randn(B, Tq, H, D, generator=g).to(dt).to(DEV)


def _bounds(q, k, v, do, window, sinks, scale):
    """(results, tolerances) of o, dq, dk, dv."""
    B, Tq, H, D = q.shape
    Tk, HK = k.shape[1:3]
    u, eta = U[q.dtype], ETA[q.dtype]
    res = ref.attention(q, k, v, window, sinks, scale, do)
    tol = [u * r.abs() + eta for r in res]
    seen = ref.visible(Tq, Tk, window, sinks, q.device)
    for b in range(B):
        for h in range(H):
            c = h * HK // H
            Q, K, V, G = q[b, :, h].double(), k[b, :, c].double(), v[b, :, c].double(), do[b, :, h].double()
            P = torch.softmax((Q @ K.T * scale).masked_fill(~seen, -1e300), -1) * seen
            dP = G @ V.T
            dS = (P * (dP - (P * dP).sum(-1, keepdim=True))).abs()
            Bi = G.abs() @ V.abs().amax(0)[:, None] if Tk else G.new_zeros(Tq, 1)
            Ci = (P * dP.abs()).sum(-1, keepdim=True)
            E = scale * ((u + F) * dS + P * (u * Ci + F * Bi))
            tol[0][b, :, h] += (u + F) * (P @ V.abs())
            tol[1][b, :, h] += E @ K.abs()
            tol[2][b, :, c] += E.T @ Q.abs()
            tol[3][b, :, c] += (u + F) * (P.T @ G.abs())
    return res, tol


def _check(got, res, tol, what):
    for name, x, r, t in zip(("o", "dq", "dk", "dv"), got, res, tol):
        err = (x.double() - r).abs()
        assert torch.isfinite(x).all(), (what, name)
        assert (err <= t).all(), (what, name, (err / t).max().item())


def _run(q, k, v, do, **kw):
    from macai_b200.window_attention import window_attention
    xs = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = window_attention(*xs, **kw)
    return (o.detach(), *torch.autograd.grad(o, xs, do))


SHAPES = [  # B, Tq, Tk, H, HK, D, window, sinks
    (1, 1, 1, 1, 1, 8, None, 0), (1, 2, 2, 2, 1, 64, 1, 0), (2, 128, 128, 2, 2, 128, None, 0),
    (1, 129, 129, 3, 1, 128, 100, 0), (2, 257, 257, 4, 2, 64, 64, 4), (1, 300, 300, 2, 1, 256, None, 0),
    (1, 300, 300, 2, 1, 256, 50, 130), (1, 640, 640, 2, 1, 96, 128, 1), (1, 65, 500, 4, 2, 72, 200, 3),
    (1, 1, 777, 2, 1, 128, 300, 0), (2, 130, 50, 2, 1, 80, None, 0), (1, 400, 390, 1, 1, 136, 33, 300),
    (1, 900, 900, 8, 1, 64, 256, 200), (1, 513, 513, 1, 1, 248, 129, 0), (1, 1500, 1500, 2, 1, 128, 300, 5),
    (1, 600, 600, 2, 2, 128, 10 ** 9, 7), (1, 384, 384, 2, 1, 40, 128, 10 ** 9)]


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, dt):
    B, Tq, Tk, H, HK, D, w, s = shape
    q, k, v, do = _inputs(B, Tq, Tk, H, HK, D, dt, Tq + Tk + D)
    got = _run(q, k, v, do, window=w, sinks=s)
    res, tol = _bounds(q, k, v, do, w, s, D ** -0.5)
    _check(got, res, tol, shape)
    again = _run(q, k, v, do, window=w, sinks=s)
    assert all(torch.equal(a, b) for a, b in zip(got, again))        # the same bits every run
    from macai_b200.window_attention import window_attention
    assert torch.equal(window_attention(q, k, v, window=w, sinks=s), got[0])


@gpu
def test_queries_without_a_visible_key():
    """More queries than keys: the first T_q - T_k see nothing and give zeros, with zero gradients."""
    q, k, v, do = _inputs(1, 300, 40, 2, 1, 64, BF)
    o, dq, dk, dv = _run(q, k, v, do, window=16)
    assert (o[:, :260] == 0).all() and (dq[:, :260] == 0).all()
    _check((o, dq, dk, dv), *_bounds(q, k, v, do, 16, 0, 0.125), "late keys")
    o, dq, dk, dv = _run(q[:, :, :, :], k[:, :0], v[:, :0], do)
    assert (o == 0).all() and (dq == 0).all() and dk.shape == (1, 0, 1, 64)
    o, dq, dk, dv = _run(q[:, :0], k, v, do[:, :0])
    assert o.shape == (1, 0, 2, 64) and (dk == 0).all() and (dv == 0).all()


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("cu,D,w,s", [([0, 100, 100, 357, 900, 1000], 128, 150, 3), ([0, 1, 2, 130, 131], 64, None, 0),
                                      ([0, 128, 256, 700], 256, 64, 130), (list(range(0, 301, 7)) + [301], 96, 5, 1)])
def test_packed_rows(cu, D, w, s, dt):
    """Every sequence on its own: the results of separate calls, to the same tolerance, and near a neighbour's values."""
    T = cu[-1]
    q, k, v, do = _inputs(1, T, T, 4, 2, D, dt, T)
    got = _run(q, k, v, do, window=w, sinks=s, cu_seqlens=torch.tensor(cu, dtype=torch.int32))
    for a, b in zip(cu, cu[1:]):
        if b > a:
            part = [t[:, a:b] for t in (q, k, v, do)]
            _check([t[:, a:b] for t in got], *_bounds(*part, w, s, D ** -0.5), (a, b))
    wild = torch.tensor([0, T + 50, -3, T], dtype=torch.int64, device=DEV)   # clamped on the device: in bounds, any result
    _run(q, k, v, do, window=w, sinks=s, cu_seqlens=wild)
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_packed_sequences_do_not_reach_each_other(D):
    """Infinities and NaN of a sequence stay in it, in tiles that hold rows of both too."""
    cu, T = [0, 150, 300, 427, 700], 700
    seqs = torch.tensor(cu, dtype=torch.int32)
    q, k, v, do = _inputs(1, T, T, 4, 2, D, BF, 11)
    want = _run(q, k, v, do, window=90, sinks=3, cu_seqlens=seqs)
    for bad in (float("nan"), float("inf"), float("-inf")):
        w = [t.clone() for t in (q, k, v, do)]
        for t in w:
            t[:, 150:300] = bad
            t[:, 427:430] = bad
        got = _run(*w, window=90, sinks=3, cu_seqlens=seqs)
        for a, b in ((0, 150), (300, 427)):
            assert all(torch.equal(x[:, a:b], y[:, a:b]) for x, y in zip(want, got)), (bad, a)


@gpu
def test_many_packed_sequences():
    """More sequences than a warp's scan step holds (256)."""
    lens = [(7 * i) % 5 for i in range(700)]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    T = cu[-1]
    q, k, v, do = _inputs(1, T, T, 2, 1, 64, BF, 5)
    got = _run(q, k, v, do, window=3, cu_seqlens=torch.tensor(cu))
    for i in (0, 1, 255, 256, 257, 511, 512, 698, 699):
        a, b = cu[i], cu[i + 1]
        if b > a:
            part = [t[:, a:b] for t in (q, k, v, do)]
            _check([t[:, a:b] for t in got], *_bounds(*part, 3, 0, 0.125), i)


@gpu
def test_strided_views_scale_and_streams():
    B, T, H, HK, D = 2, 200, 4, 2, 64
    qkv = torch.randn(B, T, (H + 2 * HK) * D, device=DEV).to(BF)
    q = qkv[..., :H * D].unflatten(-1, (H, D))
    k = qkv[..., H * D:(H + HK) * D].unflatten(-1, (HK, D))
    v = qkv[..., (H + HK) * D:].unflatten(-1, (HK, D))
    do = torch.randn(B, H, T, D, device=DEV).to(BF).transpose(1, 2)
    got = _run(q, k, v, do, window=70, sinks=2, scale=0.3)
    _check(got, *_bounds(q, k, v, do, 70, 2, 0.3), "views")
    odd = torch.randn(B, T, H, D + 1, device=DEV).to(BF)[..., 1:]            # rows that TMA cannot read: copied
    got = _run(odd, k, v, do, window=70)
    _check(got, *_bounds(odd, k, v, do, 70, 0, 0.125), "unaligned")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = _run(q, k, v, do, window=70, sinks=2, scale=0.3)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, _run(q, k, v, do, window=70, sinks=2, scale=0.3)))


@gpu
def test_large_scores_and_masked_infinities():
    """Scores of some hundreds (a maximum that moves in every tile), and keys of infinities and NaN where no query looks:
    they reach neither o nor dq."""
    q, k, v, do = _inputs(1, 520, 520, 1, 1, 64, BF, 3)
    k = (k * torch.linspace(0.1, 12, 520, device=DEV)[None, :, None, None]).to(BF)
    from macai_b200.window_attention import window_attention
    o = window_attention(q, k, v, window=200)
    r = ref.attention(q, k, v, 200, 0)
    A = ref.attention(q, k, v.abs(), 200, 0)
    # scores to 450: their fp32 error is up to 64 * 2^-24 * 450 * 1.44 of P
    assert ((o.double() - r).abs() <= U[BF] * r.abs() + (U[BF] + 3e-3) * A).all()
    q, k, v, _ = _inputs(1, 400, 400, 1, 1, 64, BF, 4)
    clean = window_attention(q, k, v, window=100)
    k[:, 300:] = float("nan")
    k[:, 350:] = float("inf")
    assert torch.equal(window_attention(q, k, v, window=100)[:, :300], clean[:, :300])
    assert window_attention(q, k, v, window=100)[:, 300:].isnan().all()       # and a NaN that is seen stays one


@gpu
def test_tiny_gradients_in_float16():
    """dS is scaled before its rounding: gradients of 1e-6 lose nothing to float16's range."""
    q, k, v, do = _inputs(1, 600, 600, 2, 1, 64, HF, 6)
    big = _run(q, k, v, do, window=500)
    small = _run(q, k, v, (do * 2.0 ** -6), window=500)
    for a, b in zip(big[1:], small[1:]):
        err = (b.double() * 2.0 ** 6 - a.double()).abs()
        # each rounds once: 2^-11 of its size, or half a subnormal step, scaled up
        assert (err <= 2 * 2.0 ** -11 * a.double().abs() + 2.0 ** -25 * 2.0 ** 6 + 1e-6).all()


@gpu
def test_gradient_against_differences():
    """Directional differences of the float64 attention at the kernels' (16-bit) inputs; h = 1e-3: error O(h^2) and the
    kernels' own roundings, u of the sum of the terms' sizes."""
    from macai_b200.window_attention import window_attention
    q, k, v, do = _inputs(1, 150, 150, 2, 1, 32, BF, 9)
    _, dq, dk, dv = _run(q, k, v, do, window=40, sinks=3)
    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate((dq, dk, dv)):
        x = (q, k, v)[i]
        e = torch.randn(x.shape, generator=g).double().to(DEV)
        vals = []
        for sign in (1, -1):
            ys = [t.double() for t in (q, k, v)]
            ys[i] = ys[i] + sign * 1e-3 * e
            vals.append(float((ref.attention(*ys, 40, 3) * do.double()).sum()))
        d = (vals[0] - vals[1]) / 2e-3
        # each element of the gradient is off by a few u of its size, at random: 4 u of the root of the sum of squares
        size = float((grad.double() * e).square().sum().sqrt())
        assert abs(d - float((grad.double() * e).sum())) <= 4 * U[BF] * size + 1e-3 * abs(d)


@gpu
def test_refusals():
    from macai_b200.window_attention import window_attention
    q, k, v, _ = _inputs(1, 8, 8, 4, 2, 64, BF)
    with pytest.raises(TypeError):
        window_attention(q.float(), k.float(), v.float())
    for bad in ((q, k.half(), v), (q, k[:, :4], v), (q[0], k, v), (q[:, :, :3], k, v), (q[..., :32], k, v)):
        with pytest.raises((ValueError, TypeError)):
            window_attention(*bad)
    with pytest.raises(NotImplementedError):
        window_attention(q[..., :12], k[..., :12], v[..., :12])
    with pytest.raises(RuntimeError, match="CPU"):
        window_attention(q.cpu(), k.cpu(), v.cpu())
    for kw in ({"window": 0}, {"window": -4}, {"window": 1.5}, {"sinks": -1}, {"sinks": 2.0}):
        with pytest.raises(ValueError):
            window_attention(q, k, v, **kw)
    for cu in ([0, 4], [1, 8], [0, 5, 3, 8]):
        with pytest.raises(ValueError):
            window_attention(q, k, v, cu_seqlens=torch.tensor(cu))
    with pytest.raises(ValueError):
        window_attention(q.expand(2, 8, 4, 64), k.expand(2, 8, 2, 64), v.expand(2, 8, 2, 64), cu_seqlens=torch.tensor([0, 8]))


# ---- the single-token form

STEPS = [  # S, H, HK, D, window, sinks, lengths
    (64, 1, 1, 128, None, 0, [0, 40, 63]), (1024, 16, 2, 256, None, 0, [777, -1, 0, 1023]),
    (68, 8, 4, 96, 32, 4, [10, 67, 68, 1000]), (4160, 32, 4, 128, 4096, 64, [60000, 4000, 100]),
    (20000, 34, 2, 64, None, 0, [19999, 5]), (300, 3, 1, 8, 100, 7, [299, 5000]), (64, 2, 1, 64, None, 64, [63, 30]),
    (40, 4, 1, 72, 8, 4, [2 ** 31 - 1, 39, 40]), (130, 20, 1, 128, 1, 0, [0, 129, 4000])]


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("case", STEPS)
def test_step(case, dt):
    """Tolerance as the forward's: P rounded to the inputs' type, u |o| + (u + f) sum_j P |v|; the caches bit for bit."""
    from macai_b200.window_attention import window_attention_step
    S, H, HK, D, w, s, lens = case
    B = len(lens)
    g = torch.Generator().manual_seed(S)
    q = (1.5 * torch.randn(B, 1, H, D, generator=g)).to(dt).to(DEV)
    k, v = (torch.randn(B, 1, HK, D, generator=g).to(dt).to(DEV) for _ in range(2))
    kc, vc = (torch.randn(B, S, HK, D, generator=g).to(dt).to(DEV) for _ in range(2))
    for b, n in enumerate(lens):      # what no token has written yet may hold anything
        if n < S:
            kc[b, max(n, 0):], vc[b, max(n, 0):] = float("nan"), float("inf")
    L = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ro, rk, rv = ref.attention_step(q, k, v, kc, vc, L, w, s)
    A, _, _ = ref.attention_step(q, k, v.abs(), kc, vc.abs(), L, w, s)
    o = window_attention_step(q, k, v, kc, vc, L, w, s)
    assert torch.isfinite(o).all()
    assert ((o.double() - ro).abs() <= U[dt] * ro.abs() + (U[dt] + F) * A + ETA[dt]).all()
    same = lambda x, y: torch.equal(x.double().nan_to_num(7.0, 8.0), y.nan_to_num(7.0, 8.0))  # noqa: E731
    assert same(kc, rk) and same(vc, rv)
    assert torch.equal(window_attention_step(q, k, v, kc, vc, L, w, s), o)   # storing the same token again changes nothing


@gpu
def test_step_follows_the_prefill():
    """Tokens fed one by one through a rolling cache give what window_attention gives for the whole row."""
    from macai_b200.window_attention import window_attention, window_attention_step
    B, T, H, HK, D, w, s = 2, 90, 4, 2, 64, 20, 3
    q, k, v, _ = _inputs(B, T, T, H, HK, D, BF, 2)
    whole = window_attention(q, k, v, window=w, sinks=s)
    kc, vc = (torch.empty(B, s + w, HK, D, dtype=BF, device=DEV).fill_(float("nan")) for _ in range(2))
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    A = ref.attention(q, k, v.abs(), w, s)
    for t in range(T):
        o = window_attention_step(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], kc, vc, lengths, w, s)
        lengths += 1
        # both within u |o| + (u + f) A of the same value
        assert ((o.double() - whole[:, t:t + 1].double()).abs() <= 2 * (2 * U[BF] + F) * A[:, t:t + 1]).all(), t


@gpu
def test_step_strided_caches_and_long_offsets():
    """Caches as views of one buffer with heads outside the slots; a cache whose offsets pass 32 bits."""
    from macai_b200.window_attention import window_attention_step
    B, S, H, HK, D = 2, 100, 4, 2, 64
    kv = torch.randn(2, B, HK, S, D, device=DEV).to(BF)
    kc, vc = kv[0].transpose(1, 2), kv[1].transpose(1, 2)
    q, k, v, _ = _inputs(B, 1, 1, H, HK, D, BF, 8)
    L = torch.tensor([50, 99], dtype=torch.int32, device=DEV)
    ro, rk, rv = ref.attention_step(q, k, v, kc, vc, L, 30, 2)
    o = window_attention_step(q, k, v, kc, vc, L, 30, 2)
    assert torch.equal(kc.double(), rk) and torch.equal(vc.double(), rv)
    assert ((o.double() - ro).abs() <= (2 * U[BF] + F) * ref.attention_step(q, k, v.abs(), kc, vc.abs(), L, 30, 2)[0] + 1e-6).all()
    S = 2 ** 21 + 64                                     # 2^21 slots of 2048 elements: past 2^32
    kc, vc = (torch.zeros(1, S, 16, 128, dtype=BF, device=DEV) for _ in range(2))
    q, k, v, _ = _inputs(1, 1, 1, 16, 16, 128, BF, 9)
    near = torch.randn(1, 64, 16, 128, device=DEV).to(BF)
    kc[:, S - 64:], vc[:, S - 64:] = near, near.flip(1)
    L = torch.tensor([S - 1], dtype=torch.int32, device=DEV)
    o = window_attention_step(q, k, v, kc, vc, L, 60, 0)
    want, _, _ = ref.attention_step(q, k, v, near, near.flip(1), torch.tensor([63], device=DEV), 60, 0)
    A, _, _ = ref.attention_step(q, k, v.abs(), near, near.flip(1).abs(), torch.tensor([63], device=DEV), 60, 0)
    assert ((o.double() - want).abs() <= (2 * U[BF] + F) * A).all()
    assert torch.equal(kc[:, S - 1], k[:, 0]) and torch.equal(vc[:, S - 1], v[:, 0])


@gpu
def test_step_refusals():
    from macai_b200.window_attention import window_attention_step
    q, k, v, _ = _inputs(2, 1, 1, 4, 2, 64, BF)
    kc, vc = (torch.zeros(2, 32, 2, 64, dtype=BF, device=DEV) for _ in range(2))
    L = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in ((q.expand(2, 3, 4, 64), k, v, kc, vc, L), (q, k, v, kc.half(), vc, L), (q, k, v, kc[:1], vc, L),
                (q, k, v, kc[:, :0], vc[:, :0], L), (q, k, v, kc, vc, L.long()), (q, k, v, kc, vc, L[:1]),
                (q, k, v, kc, vc, L.cpu()), (q, k, v, kc, vc[:, :16], L),
                (q, k, v, torch.zeros(2, 32, 2, 65, dtype=BF, device=DEV)[..., :64], vc, L)):
        with pytest.raises(ValueError):
            window_attention_step(*bad)
    with pytest.raises(RuntimeError, match="no gradient"):
        window_attention_step(q.requires_grad_(True), k, v, kc, vc, L)
