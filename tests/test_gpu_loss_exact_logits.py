"""Losses of logits that the products form exactly, or nearly: what is left is the float32 arithmetic of the softmax, however
wide the rows are. One non-zero entry a row, small whole numbers, rows padded with zeros."""
import pytest
import torch

from macai_b200.loss import linear_cross_entropy

pytestmark = pytest.mark.gpu


def _outside(x, w, lab, steps=0):
    """The largest excess of a loss's error over what float32 does to it. A difference to the largest logit is rounded, then
    multiplied by a rounded log2(e) and rounded again: three half steps of it in an exponent, one where it is the label's (and the
    last sum's rounding): 2^-22 of it covers them. Exponentials, their sum and its logarithm: 2^-19. A product of `steps` steps of
    16 terms may be cut by 2^-23 of its terms' magnitudes in each."""
    loss = linear_cross_entropy(x, w, lab, reduction="none").double()
    logits = x.double() @ w.double().t()
    top = logits.max(1, keepdim=True).values
    p = torch.softmax(logits, 1)
    at = logits.gather(1, lab[:, None])
    size = (p * (top - logits)).sum(1) + (top - at)[:, 0]
    cut = steps * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).max(1).values
    off = (loss - (logits.logsumexp(1) - at[:, 0])).abs()
    return float((off - (2.0 ** -22 * size + 2.0 ** -19 + 2 * cut)).max())


def _numbers(n, D, V, seed):
    gen = torch.Generator().manual_seed(seed)
    return (lambda *s: torch.randn(*s, generator=gen)), (lambda lo, hi, s: torch.randint(lo, hi, s, generator=gen)), \
        torch.randint(0, V, (n,), generator=gen).cuda()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 512, 2048, 8192])
def test_one_entry_a_row(D, dt):
    n, V = 300, 700
    rand, whole, lab = _numbers(n, D, V, D)
    w = rand(V, D).to(dt).cuda()
    x = torch.zeros(n, D, dtype=dt, device="cuda")
    x[torch.arange(n), whole(0, D, (n,)).cuda()] = (30 * rand(n)).to(dt).cuda()   # logits up to about 100
    assert _outside(x, w, lab) <= 0


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [512, 2048, 8192])
def test_whole_numbers(D, dt):
    """Sums that no adder of 24 bits cuts."""
    n, V = 300, 700
    _, whole, lab = _numbers(n, D, V, D)
    x, w = whole(-2, 3, (n, D)).to(dt).cuda(), whole(-1, 2, (V, D)).to(dt).cuda()   # logits of about 1.2 sqrt(D), up to 400
    assert _outside(x, w, lab) <= 0


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [2048, 8192])
def test_rows_padded_with_zeros(D, dt):
    n, V = 300, 700
    rand, _, lab = _numbers(n, D, V, D)
    x, w = torch.zeros(n, D, dtype=dt, device="cuda"), rand(V, D).to(dt).cuda()
    x[:, 128:160] = (3 * rand(n, 32)).to(dt).cuda()
    assert _outside(x, w, lab, steps=2) <= 0


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [512, 2048, 8192])
@pytest.mark.parametrize("kind", ["any", "one sign"])
def test_losses_are_not_shifted(D, kind, dt):
    """The adder cuts towards zero, by half a step of the accumulator on average (2^-23 of it at most is a step). Logits are summed
    in runs of 768 terms or less, 48 steps of the adder, and the runs added in float32. A run's sum grows evenly, so that a cut
    costs half of what it costs at its end: 48 x 1/2 x 1/2 x 2^-23 of the logit, whatever D is (in one go it would be D / 16 in
    place of 48). float16's products have 22 bits, where bfloat16's have 16: next to an accumulator of one sign's many terms each of
    a step's 16 products loses bits of its own, half a step on average, towards zero like the sum: 17 cuts for one."""
    n, V = 600, 1500
    rand, _, lab = _numbers(n, D, V, D)
    w, x = rand(V, D) * 1.5 * D ** -0.5, rand(n, D)
    if kind == "any":   # logits as a trained model has them: the label's stands out
        x = x + 4 * torch.rand(n, 1, generator=torch.Generator().manual_seed(1)) * w[lab.cpu()]
    else:
        x, w = x.abs(), w.abs()
    x, w = x.to(dt).cuda(), w.to(dt).cuda()
    loss = linear_cross_entropy(x, w, lab, reduction="none").double()
    logits = x.double() @ w.double().t()
    at = logits.gather(1, lab[:, None])[:, 0]
    size = at - (logits.softmax(1) * logits).sum(1)
    off = loss - (logits.logsumexp(1) - at)
    # half a step of float32 of the logits' size for what is not the cut
    floor = 2.0 ** -24 * float(logits.abs().max()) / float(size.abs().max())
    cuts = 17 if dt == torch.float16 and kind == "one sign" else 1
    assert abs(float((off * size).sum() / (size * size).sum())) <= cuts * 12 * 2.0 ** -23 + floor
