"""The gated feed-forward block against its float64 definition with bounds from the kernels' roundings: sizes, both kernels'
ranges, strides, gradients, float16's range, frozen weights, streams and graphs."""
import pytest
import torch

from macai_b200.feed_forward import gated_feed_forward
from oracle import decoder_steps_f64 as steps

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
NAMES = ("dx", "dw_gate", "dw_up", "dw_down")


def _inputs(n, D, F, O, dt, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda a, b, s: (torch.randn(a, b, generator=gen) * s).to(dt).cuda()  # noqa: E731
    return r(n, D, scale), r(F, D, D ** -0.5), r(F, D, D ** -0.5), r(O, F, F ** -0.5), r(n, O, 0.1)


def _check(got, want, dt):
    for k, v in got.items():
        assert v.dtype == dt and v.shape == want[k][0].shape
        assert steps.outside(v, *want[k], dt) <= 0, k


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("n,D,F,O", [(1, 8, 8, 8), (1, 64, 128, 64), (4, 256, 512, 256), (16, 200, 264, 136), (17, 1000, 72, 8),
                                     (31, 8, 1000, 520), (33, 512, 384, 264), (64, 136, 640, 128), (65, 264, 200, 72),
                                     (127, 96, 96, 1000), (128, 320, 448, 200)])
def test_few_tokens(n, D, F, O, dt):
    x, wg, wu, wd, _ = _inputs(n, D, F, O, dt, seed=n)
    _check({"y": gated_feed_forward(x, wg, wu, wd)}, steps.feed_forward(x, wg, wu, wd), dt)


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("n,D,F,O", [(1, 8, 8, 8), (3, 64, 72, 136), (129, 200, 264, 64), (256, 256, 256, 256),
                                     (257, 320, 136, 520), (700, 72, 1000, 264), (1025, 512, 328, 128)])
def test_training(n, D, F, O, dt):
    x, wg, wu, wd, dy = _inputs(n, D, F, O, dt, seed=n)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    want = steps.feed_forward(*(t.detach() for t in leaves), dy)
    _check({"y": y.detach(), **dict(zip(NAMES, grads))}, want, dt)
    if n > 128:   # the same kernels without a gradient
        with torch.no_grad():
            assert torch.equal(gated_feed_forward(*leaves), y)


@pytest.mark.parametrize("dt", [BF, F16])
def test_many_tiles(dt):
    """Every CTA pair walks several tiles of every problem."""
    x, wg, wu, wd, dy = _inputs(3000, 1032, 1544, 1288, dt, seed=5)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    _check({"y": y.detach(), **dict(zip(NAMES, grads))}, steps.feed_forward(*(t.detach() for t in leaves), dy), dt)


@pytest.mark.parametrize("n", [40, 300])
def test_strides(n):
    """Three dimensions, halves of one weight, a view with room between its rows, a transposed weight, an odd start, an
    expanded input and an expanded gradient."""
    x, wg, wu, wd, dy = _inputs(n, 64, 128, 72, BF, seed=1)
    both = torch.cat([wg, wu])
    wide = torch.zeros(n, 80, dtype=BF, device="cuda")
    wide[:, 8:72] = x
    odd = torch.zeros(n * 64 + 3, dtype=BF, device="cuda")[3:].view(n, 64).copy_(x)
    down = wd.t().contiguous().t()
    for need in (False, True):
        def run(x, wg, wu, wd, dy):
            ts = [t.detach().requires_grad_(need) for t in (x, wg, wu, wd)]
            y = gated_feed_forward(*ts)
            if not need:
                return [y]
            return [y.detach().flatten(0, -2), *(g.flatten(0, -2) for g in torch.autograd.grad(y, ts, dy))]
        want = run(x, wg, wu, wd, dy)
        for args in ((x.view(2, n // 2, 64), both[:128], both[128:], wd, dy.view(2, n // 2, 72)), (wide[:, 8:72], wg, wu, down, dy),
                     (odd, wg, wu, wd, dy.t().contiguous().t())):
            for a, b in zip(run(*args), want):
                assert torch.equal(a.flatten(0, -2) if a.dim() == 3 else a, b)
    one = x[:1].expand(n, 64)
    a = gated_feed_forward(one, wg, wu, wd)
    assert torch.equal(a, gated_feed_forward(one.contiguous(), wg, wu, wd))
    leaf = x.clone().requires_grad_(True)
    a, = torch.autograd.grad(gated_feed_forward(leaf, wg, wu, wd).sum(), leaf)     # a gradient with strides of 0
    b, = torch.autograd.grad(gated_feed_forward(leaf, wg, wu, wd), leaf, torch.ones(n, 72, dtype=BF, device="cuda"))
    assert torch.equal(a, b)


def test_frozen_inputs():
    x, wg, wu, wd, dy = _inputs(200, 64, 136, 72, F16, seed=2)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    full = torch.autograd.grad(gated_feed_forward(*leaves), leaves, dy)
    for mask in range(1, 15):
        ts = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(leaves)]
        need = [t for t in ts if t.requires_grad]
        got = torch.autograd.grad(gated_feed_forward(*ts), need, dy)
        want = [g for i, g in enumerate(full) if mask >> i & 1]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), mask


def test_same_bits_every_run():
    x, wg, wu, wd, dy = _inputs(900, 264, 520, 256, BF, seed=3)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]

    def run():
        y = gated_feed_forward(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))
    few = [gated_feed_forward(x[:9].detach(), wg.detach(), wu.detach(), wd.detach()) for _ in range(4)]
    assert all(torch.equal(a, few[0]) for a in few)


@pytest.mark.parametrize("scale", [2.0 ** -18, 2.0 ** -8, 1.0, 64.0])
def test_float16_gradients_of_any_size(scale):
    """Gradients of the output far below and above float16's middle: what the weights' sums are made of keeps its bits."""
    x, wg, wu, wd, dy = _inputs(600, 128, 256, 64, F16, seed=4, scale=4.0)
    dy = (dy.float() * scale).half()
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    _check({"y": y.detach(), **dict(zip(NAMES, grads))}, steps.feed_forward(*(t.detach() for t in leaves), dy), F16)


def test_zero_gradient():
    x, wg, wu, wd, dy = _inputs(300, 64, 72, 64, F16, seed=4)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    for g in torch.autograd.grad(gated_feed_forward(*leaves), leaves, torch.zeros_like(dy)):
        assert not g.any()


@pytest.mark.parametrize("dt,scale", [(BF, 200.0), (F16, 200.0), (F16, 30.0)])
def test_saturated_gates(dt, scale):
    """Gates far out on both sides: silu is 0 or the gate, and no exponential's overflow shows. Where h itself is past
    float16's end (scale 200: |h| up to 600,000) its row overflows, as in the formula rounded to float16, and no other does."""
    x, wg, wu, wd, dy = _inputs(140, 64, 128, 64, dt, seed=6, scale=scale)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        few = gated_feed_forward(x[:20], wg, wu, wd)
    x, wg, wu, wd = (t.detach() for t in leaves)
    want = steps.feed_forward(x, wg, wu, wd, dy)
    h = torch.nn.functional.silu(x.double() @ wg.double().T) * (x.double() @ wu.double().T)
    fits = (h.abs().amax(1) < 65000) & (want["y"][0].abs().amax(1) < 65000) if dt == F16 else torch.ones(140, dtype=torch.bool)
    fits = fits.cuda()
    assert bool(fits.any()) and bool(few[fits[:20]].isfinite().all())
    assert steps.outside(y.detach()[fits], want["y"][0][fits], want["y"][1][fits], dt) <= 0
    assert not bool(y[h.abs().amax(1) > 66000].isfinite().all(1).any()) or dt == BF
    if bool(fits.all()):
        _check(dict(zip(NAMES, grads)), want, dt)


def test_infinities_and_nan_stay_in_their_rows():
    for n in (20, 300):
        x, wg, wu, wd, _ = _inputs(n, 64, 128, 64, BF, seed=7)
        clean = gated_feed_forward(x, wg, wu, wd)
        x[3, 5], x[7, 0] = float("nan"), float("inf")
        y = gated_feed_forward(x, wg, wu, wd)
        rest = [i for i in range(n) if i not in (3, 7)]
        assert bool(y[3].isnan().all()) and not bool(y[7].isfinite().any()) and torch.equal(y[rest], clean[rest])


def test_no_tokens():
    _, wg, wu, wd, _ = _inputs(1, 64, 128, 72, BF)
    x = torch.zeros(2, 0, 64, dtype=BF, device="cuda", requires_grad=True)
    w = wg.requires_grad_(True)
    y = gated_feed_forward(x, w, wu, wd)
    assert y.shape == (2, 0, 72)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and not dw.any()


@pytest.mark.parametrize("n", [4, 200])
def test_captured(n):
    """Forward (and backward) captured on another stream, replayed on new inputs."""
    x, wg, wu, wd, dy = _inputs(n, 128, 264, 128, BF, seed=8)
    other = _inputs(n, 128, 264, 128, BF, seed=9)
    train = n > 128
    leaves = [t.clone().requires_grad_(train) for t in (x, wg, wu, wd)]

    def run(ts, dy):
        y = gated_feed_forward(*ts)
        return [y.detach(), *(torch.autograd.grad(y, ts, dy) if train else ())]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(leaves, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = run(leaves, dy)
    with torch.no_grad():
        for t, v in zip(leaves, other[:4]):
            t.copy_(v)
        dy.copy_(other[4])
    graph.replay()
    torch.cuda.synchronize()
    want = run([t.detach().clone().requires_grad_(train) for t in leaves], other[4])
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    a, b = _inputs(700, 128, 512, 128, BF, seed=10), _inputs(9, 512, 1024, 512, BF, seed=11)
    want = gated_feed_forward(*a[:4]), gated_feed_forward(*b[:4])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            y1 = gated_feed_forward(*a[:4])
        with torch.cuda.stream(s2):
            y2 = gated_feed_forward(*b[:4])
        got.append((y1, y2))
    torch.cuda.synchronize()
    assert all(torch.equal(u, want[0]) and torch.equal(v, want[1]) for u, v in got)


def test_refusals():
    x, wg, wu, wd, _ = _inputs(4, 64, 128, 64, BF)
    with pytest.raises(ValueError, match="agree"):
        gated_feed_forward(x, wg, wu[:64], wd)
    with pytest.raises(ValueError, match="agree"):
        gated_feed_forward(x[:, :32], wg, wu, wd)
    with pytest.raises(ValueError, match="agree"):
        gated_feed_forward(x, wg, wu, wd[:, :64])
    with pytest.raises(NotImplementedError, match="multiples of 8"):
        gated_feed_forward(x[:, :60], wg[:, :60], wu[:, :60], wd)
    with pytest.raises(ValueError, match="share"):
        gated_feed_forward(x, wg, wu.cpu(), wd)
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(gated_feed_forward(leaf, wg, wu, wd).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_forward_mode_is_refused():
    x, wg, wu, wd, _ = _inputs(4, 64, 128, 64, BF)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((NotImplementedError, RuntimeError)):
            gated_feed_forward(dual, wg, wu, wd)


@pytest.mark.parametrize("dt", [BF, F16])
def test_a_kept_graph_and_a_shared_weight(dt):
    """The backward twice over one graph has the same bits; a weight given twice gets the sum of its two gradients."""
    x, wg, wu, wd, dy = _inputs(150, 64, 136, 72, dt, seed=30)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    torch.autograd.grad(y, leaves, 3 * dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    one, two = wg.clone().requires_grad_(True), wg.clone().requires_grad_(True)
    both = torch.autograd.grad(gated_feed_forward(x, one, two, wd), [one, two], dy)
    same = torch.autograd.grad(gated_feed_forward(x, one, one, wd), [one], dy)[0]
    assert torch.equal(same, both[0] + both[1])


def test_checkpointed_block():
    """Formed again in the backward: the same gradients, in both of torch's forms of it."""
    from torch.utils.checkpoint import checkpoint
    x, wg, wu, wd, dy = _inputs(140, 64, 128, 64, BF, seed=31)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    want = torch.autograd.grad(gated_feed_forward(*leaves), leaves, dy)
    for reentrant in (False, True):
        copies = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
        checkpoint(gated_feed_forward, *copies, use_reentrant=reentrant).backward(dy)
        assert all(torch.equal(t.grad, v) for t, v in zip(copies, want))


def test_inference_mode():
    x, wg, wu, wd, _ = _inputs(5, 64, 128, 64, BF, seed=32)
    want = gated_feed_forward(x, wg, wu, wd)
    with torch.inference_mode():
        assert torch.equal(gated_feed_forward(x.clone(), wg, wu, wd), want)
