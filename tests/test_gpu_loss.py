"""The cross entropy of a vocabulary projection against its float64 definition with bounds from the kernels' roundings:
vocabularies of any size, ignored and impossible labels, reductions, pieces, float16's range, graphs."""
import math

import pytest
import torch

from macai_b200.loss import linear_cross_entropy
from oracle import decoder_steps_f64 as steps

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def _inputs(n, D, V, dt, seed=0, ignored=0.2, sharp=1.5):
    gen = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=gen) * sharp * D ** -0.5).to(dt)
    lab = torch.randint(0, V, (n,), generator=gen)
    x = (torch.randn(n, D, generator=gen) + 4 * torch.rand(n, 1, generator=gen) * w[lab].float()).to(dt)
    lab[torch.rand(n, generator=gen) < ignored] = -100
    return x.cuda(), w.cuda(), lab.cuda()


def _rows(g, lab, reduction, ignore=-100):
    """The rows' gradients of the reduced loss."""
    if reduction == "none":
        return g
    n = int((lab != ignore).sum()) if reduction == "mean" else 1
    return (g / n).expand(lab.shape)


def _run(x, w, lab, reduction, g, **kw):
    leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
    loss = linear_cross_entropy(*leaves, lab, reduction=reduction, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, leaves, g))


def _check(got, want, dt):
    for v, k in zip(got, ("loss", "dx", "dweight")):
        assert steps.outside(v, *want[k], torch.float32 if k == "loss" else dt) <= 0, k


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("n,D,V", [(1, 8, 1), (1, 8, 2), (2, 64, 63), (5, 200, 64), (130, 72, 65), (257, 136, 255), (300, 64, 257),
                                   (33, 512, 1001), (700, 128, 513), (512, 264, 4099)])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_loss_and_gradients(n, D, V, dt, reduction):
    x, w, lab = _inputs(n, D, V, dt, seed=n + V, ignored=0.2 if n > 2 else 0.0)
    gen = torch.Generator().manual_seed(1)
    size = 4096.0 if dt == F16 else 1.0
    g = (size * (torch.rand(n, generator=gen) - 0.3) if reduction == "none" else torch.tensor(size * 0.37)).cuda()
    loss, dx, dw = _run(x, w, lab, reduction, g)
    want = steps.cross_entropy(x, w, lab, g=_rows(g, lab, reduction))
    v, e = want["loss"]
    if reduction != "none":   # a sum of n float32 values in some order, then a division
        k = float((lab >= 0).sum()) if reduction == "mean" else 1.0
        v, e = v.sum() / k, (e.sum() + n * 2.0 ** -24 * v.abs().sum()) / k + 2.0 ** -23 * (v.abs().sum() / k)
    assert loss.dtype == torch.float32 and loss.shape == (lab.shape if reduction == "none" else ())
    _check((loss, dx, dw), {**want, "loss": (v, e)}, dt)
    # without a gradient: the same loss; labels of 32 bits: the same everything
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, lab, reduction=reduction), loss)
    again = _run(x, w, lab.int(), reduction, g)
    assert all(torch.equal(a, b) for a, b in zip(again, (loss, dx, dw)))


def test_pieces():
    """A vocabulary whose logits' gradients come in several pieces (256 MiB each), the last one ragged; labels at their
    borders; the row factors vary."""
    n, D, V = 8192, 64, 50001
    x, w, lab = _inputs(n, D, V, BF, seed=3)
    for i, v in enumerate((16383, 16384, 16639, 16640, 16641, 33279, 33280, 49919, 49920, 50000, 0)):
        lab[i] = v
    g = torch.rand(n, generator=torch.Generator().manual_seed(2)).cuda()
    got = _run(x, w, lab, "none", g)
    rows = torch.arange(0, n, 2048).tolist()
    for a in rows:   # in parts: the definition holds n V values in float64
        at = slice(a, a + 256)
        want = steps.cross_entropy(x[at], w, lab[at], g=g[at])
        _check((got[0][at], got[1][at]), want, BF)
    leaves = [t.detach().float().requires_grad_(True) for t in (x, w)]
    loss = torch.nn.functional.cross_entropy(leaves[0] @ leaves[1].T, lab, reduction="none")
    want = torch.autograd.grad(loss, leaves, g)
    for a, b in zip(got[1:], want):   # D and the result are each rounded by at most 2^-8: 2^-7 of the norm bounds both
        assert float((a.float() - b).norm() / b.norm()) < 2.0 ** -7
    for v in (16383, 16384, 33279, 33280, 49919, 49920, 50000):
        assert float((got[2][v].float() - want[1][v]).norm() / want[1][v].norm()) < 2.0 ** -6
    again = _run(x, w, lab, "none", g)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


def test_a_mean_shares_no_rounding():
    """Rows that know nothing of their labels all have -g: where that is not a number of 16 bits, their common rounding must
    not become the gradient's (it was 2^-9 of it for 1 / 1,537)."""
    n, D, V = 1537, 64, 3000
    x, w, lab = _inputs(n, D, V, BF, seed=4, ignored=0.0, sharp=0.05)
    x = torch.randn(n, D, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    _, dx, dw = _run(x, w, lab, "mean", torch.tensor(1.0, device="cuda"))
    want = steps.cross_entropy(x, w, lab, g=torch.full((n,), 1.0 / n, device="cuda"))
    for got, k in ((dx, "dx"), (dw, "dweight")):
        v = want[k][0]
        assert abs(float((got.double() * v).sum() / (v * v).sum()) - 1) < 2.0 ** -11, k   # the common factor


@pytest.mark.parametrize("dt", [BF, F16])
def test_ignored_rows(dt):
    x, w, lab = _inputs(300, 64, 500, dt, seed=6, ignored=0.5)
    g = torch.tensor(1.0, device="cuda")
    loss, dx, dw = _run(x, w, lab, "mean", g)
    keep = lab >= 0
    assert not dx[~keep].any()
    kept = _run(x[keep], w, lab[keep], "mean", g)
    v = steps.cross_entropy(x[keep], w, lab[keep])["loss"][0].mean()
    assert abs(float(loss) - float(v)) < 1e-5 * float(v) and abs(float(kept[0]) - float(v)) < 1e-5 * float(v)
    want = steps.cross_entropy(x, w, lab, g=_rows(g, lab, "mean"))
    _check((steps.cross_entropy(x, w, lab)["loss"][0], dx, dw), want, dt)
    # their values do not matter to the losses and the other rows' gradients
    y = x.clone()
    y[~keep] = 1000.0
    other = _run(y, w, lab, "mean", g)
    assert torch.equal(other[0], loss) and torch.equal(other[1], dx) and torch.equal(other[2], dw)
    y[~keep] = float("nan")
    other = _run(y, w, lab, "mean", g)
    assert torch.equal(other[0], loss) and torch.equal(other[1], dx)
    # another number that means "ignored", one of the vocabulary's own among them
    for number in (7, -1, 1 << 40):
        renamed = torch.where(keep, lab, torch.full_like(lab, number))
        if number == 7:
            renamed = torch.where(lab == 7, torch.full_like(lab, 8), renamed)
            base = _run(x, w, torch.where(lab == 7, torch.full_like(lab, 8), lab), "mean", g)
        else:
            base = (loss, dx, dw)
        got = _run(x, w, renamed, "mean", g, ignore_index=number)
        assert all(torch.equal(a, b) for a, b in zip(got, base))


def test_every_row_ignored():
    x, w, lab = _inputs(40, 64, 100, BF, seed=7)
    lab[:] = -100
    for reduction in ("none", "mean", "sum"):
        g = torch.ones(40 if reduction == "none" else (), device="cuda")
        loss, dx, dw = _run(x, w, lab, reduction, g)
        assert bool(loss.isnan()) if reduction == "mean" else not loss.any()
        assert not dx.any() and not dw.any()


def test_impossible_labels():
    """A label outside the vocabulary gives NaN (its own row's, where rows are apart) and reads nothing that is not there."""
    x, w, lab = _inputs(300, 64, 130, BF, seed=8, ignored=0.0)
    good = lab.clone()
    bad = [5, 6, 70, 299]
    for i, v in zip(bad, (130, -1, 1 << 40, -(1 << 50))):
        lab[i] = v
    loss = linear_cross_entropy(x, w, lab, reduction="none")
    rest = [i for i in range(300) if i not in bad]
    assert bool(loss[bad].isnan().all()) and torch.equal(loss[rest], linear_cross_entropy(x, w, good, reduction="none")[rest])
    assert bool(linear_cross_entropy(x, w, lab).isnan())
    _, dx, _ = _run(x, w, lab, "none", torch.ones(300, device="cuda"))
    assert bool(dx[bad].isnan().all()) and bool(dx[rest].isfinite().all())


def test_large_logits():
    """Logits of thousands: no exponential overflows, sure rows have a loss of 0 and no gradient left."""
    x, w, lab = _inputs(200, 64, 300, BF, seed=9, ignored=0.0)
    x = x * 500
    loss, dx, dw = _run(x, w, lab, "none", torch.ones(200, device="cuda"))
    want = steps.cross_entropy(x, w, lab, g=torch.ones(200, device="cuda"))
    assert bool(loss.isfinite().all()) and bool((loss >= 0).all())
    _check((loss, dx, dw), want, BF)


def test_infinities_and_nan():
    x, w, lab = _inputs(150, 64, 200, BF, seed=10, ignored=0.0)
    clean = linear_cross_entropy(x, w, lab, reduction="none")
    x[3, 5], x[9, 0] = float("nan"), float("inf")
    loss = linear_cross_entropy(x, w, lab, reduction="none")
    rest = [i for i in range(150) if i not in (3, 9)]
    assert bool(loss[[3, 9]].isnan().all()) and torch.equal(loss[rest], clean[rest])


@pytest.mark.parametrize("size", [0.0, 2.0 ** -20, 1e-3, 1e4])
def test_float16_gradients_of_any_size(size):
    x, w, lab = _inputs(400, 64, 700, F16, seed=11)
    g = (size * (0.5 + torch.rand(400, generator=torch.Generator().manual_seed(3)))).cuda()
    got = _run(x, w, lab, "none", g)
    _check(got, steps.cross_entropy(x, w, lab, g=g), F16)


def test_special_gradients():
    x, w, lab = _inputs(64, 64, 100, BF, seed=12)
    g = torch.zeros(64, device="cuda")
    g[3] = -2.5
    lab[3], lab[4] = 17, -100
    got = _run(x, w, lab, "none", g)
    _check(got, steps.cross_entropy(x, w, lab, g=g), BF)
    assert not got[1][[i for i in range(64) if i != 3]].any()
    g[4] = float("nan")       # of an ignored row: not used
    assert all(torch.equal(a, b) for a, b in zip(_run(x, w, lab, "none", g), got))
    g[5], lab[5] = float("nan"), 1
    assert bool(_run(x, w, lab, "none", g)[1][5].isnan().all())


def test_strides():
    """Leading dimensions, room between rows, a transposed weight, labels with strides, an expanded gradient."""
    x, w, lab = _inputs(60, 64, 130, BF, seed=13)
    wide = torch.zeros(60, 80, dtype=BF, device="cuda")
    wide[:, 8:72] = x
    labs = torch.stack([lab, lab], 1)[:, 0]
    want = _run(x, w, lab, "mean", torch.tensor(1.0, device="cuda"))
    for args in ((wide[:, 8:72], w, labs), (x, w.t().contiguous().t(), lab), (x.view(3, 20, 64), w, lab.view(3, 20))):
        got = _run(*args, "mean", torch.tensor(1.0, device="cuda"))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].reshape(60, 64), want[1]) and torch.equal(got[2], want[2])
    leaf = x.view(3, 20, 64).detach().requires_grad_(True)
    loss = linear_cross_entropy(leaf, w, lab.view(3, 20), reduction="none")
    assert loss.shape == (3, 20)
    a, = torch.autograd.grad(loss.sum(), leaf)
    assert torch.equal(a.view(60, 64), _run(x, w, lab, "sum", torch.tensor(1.0, device="cuda"))[1])
    one = linear_cross_entropy(x[0], w, lab[0].clamp_min(0))
    assert one.shape == () and torch.equal(one, linear_cross_entropy(x[:1], w, lab[:1].clamp_min(0)))


def test_frozen_inputs():
    x, w, lab = _inputs(200, 64, 300, BF, seed=14)
    g = torch.tensor(1.0, device="cuda")
    _, dx, dw = _run(x, w, lab, "mean", g)
    a = x.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, w, lab), a)[0], dx)
    b = w.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, b, lab), b)[0], dw)


def test_no_rows():
    w = torch.randn(10, 64, device="cuda").bfloat16().requires_grad_(True)
    x = torch.zeros(0, 64, dtype=BF, device="cuda", requires_grad=True)
    lab = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert math.isnan(float(linear_cross_entropy(x, w, lab)))
    assert linear_cross_entropy(x, w, lab, reduction="none").shape == (0,)
    loss = linear_cross_entropy(x, w, lab, reduction="sum")
    assert float(loss) == 0
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert dx.shape == (0, 64) and not dw.any()


def test_captured():
    """A forward and backward captured on another stream, replayed on new inputs."""
    x, w, lab = _inputs(300, 64, 700, BF, seed=15)
    x2, w2, lab2 = _inputs(300, 64, 700, BF, seed=16)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]

    def run():
        loss = linear_cross_entropy(*leaves, lab)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = run()
    with torch.no_grad():
        x.copy_(x2), w.copy_(w2), lab.copy_(lab2)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    want = _run(x2, w2, lab2, "mean", torch.tensor(1.0, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    x, w, lab = _inputs(4, 64, 100, BF)
    for args in ((x, w, lab[:3]), (x[:, :32], w, lab), (x, w, lab[:, None])):
        with pytest.raises(ValueError, match="agree"):
            linear_cross_entropy(*args)
    with pytest.raises(ValueError, match="device"):
        linear_cross_entropy(x, w, lab.cpu())
    with pytest.raises(NotImplementedError, match="multiple of 8"):
        linear_cross_entropy(x[:, :60], w[:, :60], lab)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((NotImplementedError, RuntimeError)):
            linear_cross_entropy(dual, w, lab)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n,D,V", [(300, 64, 500), (65, 200, 70)])
def test_ignored_rows_may_hold_anything(n, D, V, value):
    """Their infinities and NaN reach no loss and neither gradient, the weight's included: they are not gathered."""
    x, w, lab = _inputs(n, D, V, BF, seed=21, ignored=0.4)
    g = torch.tensor(1.0, device="cuda")
    want = _run(x, w, lab, "mean", g)
    y = x.clone()
    y[lab < 0] = value
    got = _run(y, w, lab, "mean", g)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool(got[2].isfinite().all())


@pytest.mark.parametrize("dt", [BF, F16])
def test_a_kept_graph_and_changed_labels(dt):
    """The backward twice over one graph has the same bits, whatever became of the labels after the forward."""
    x, w, lab = _inputs(150, 64, 200, dt, seed=22)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    g = torch.rand(150, device="cuda")
    loss = linear_cross_entropy(*leaves, lab, reduction="none")
    first = torch.autograd.grad(loss, leaves, g, retain_graph=True)
    lab.fill_(-100)
    torch.autograd.grad(loss, leaves, 2 * g, retain_graph=True)
    again = torch.autograd.grad(loss, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_tied_weight():
    """x made from the weight itself, as with tied embeddings: both gradients arrive in it."""
    w = _inputs(4, 64, 90, BF, seed=23)[1].requires_grad_(True)
    tokens, lab = torch.tensor([3, 70, 3, 89, 0], device="cuda"), torch.tensor([70, 3, 89, 0, -100], device="cuda")
    got = torch.autograd.grad(linear_cross_entropy(w[tokens], w, lab), w)[0]
    x = w.detach()[tokens].requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, lab), [x, w])
    e = w.detach().clone().requires_grad_(True)
    want = dw.double() + torch.autograd.grad(e[tokens], e, dx)[0].double()
    # one rounding of the sum of two gradients in bf16
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-30).all())


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D", [512, 2048, 4096])
def test_the_adders_cut_is_taken_back(D, dt):
    """Losses of long sums are not shifted towards the smaller logits. A sum of D products in fp32 whose D / 16 steps are each cut
    by up to 2^-23 of it would be off by up to D / 16 x 2^-23 of a logit, always towards zero; half of that is the mean of such
    cuts. What is left on average is held to a fifth of it (the logits' own size: the difference of the label's and the mean one)."""
    n, V = 600, 1500
    gen = torch.Generator().manual_seed(D)
    w = (torch.randn(V, D, generator=gen) * 1.5 * D ** -0.5).to(dt)
    lab = torch.randint(0, V, (n,), generator=gen)
    x = (torch.randn(n, D, generator=gen) + 4 * torch.rand(n, 1, generator=gen) * w[lab].float()).to(dt)
    x, w, lab = x.cuda(), w.cuda(), lab.cuda()
    loss = linear_cross_entropy(x, w, lab, reduction="none").double()
    logits = x.double() @ w.double().t()
    at = logits.gather(1, lab[:, None])[:, 0]
    size = at - (logits.softmax(1) * logits).sum(1)
    off = loss - (logits.logsumexp(1) - at)
    assert abs(float((off * size).sum() / (size * size).sum())) <= D / 16 * 2.0 ** -24 / 5
