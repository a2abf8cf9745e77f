"""Many rows of which none or a few count, so that most pairs of CTAs have no tile and end at once: what runs on their SMs next
has its own shared memory to itself. Many launches in a row, each followed by kernels that keep their operands there."""
import pytest
import torch

from macai_b200.feed_forward import gated_feed_forward
from macai_b200.loss import linear_cross_entropy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("live", [0, 1, 257])
def test_pairs_without_a_tile(live, dt):
    gen = torch.Generator().manual_seed(live)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    n, D, V = 8192, 128, 1000
    x, w = rand(n, D).to(dt).cuda(), (rand(V, D) * 0.1).to(dt).cuda()
    lab = torch.full((n,), -100)
    at = torch.randperm(n, generator=gen)[:live]
    lab[at] = torch.randint(0, V, (live,), generator=gen)
    lab = lab.cuda()
    few = [rand(9, 512).to(dt).cuda(), *((rand(*s) * 0.05).to(dt).cuda() for s in ((1024, 512), (1024, 512), (512, 1024)))]
    many = [rand(600, 256).to(dt).cuda(), *((rand(*s) * 0.05).to(dt).cuda() for s in ((640, 256), (640, 256), (256, 640)))]
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]

    def run():
        loss = linear_cross_entropy(*leaves, lab, reduction="sum")
        a = gated_feed_forward(*few)
        grads = torch.autograd.grad(loss, leaves)
        return [loss.detach(), *grads, a, gated_feed_forward(*many)]
    torch.cuda.synchronize()
    # each alone, the GPU waited for in between
    loss = linear_cross_entropy(*leaves, lab, reduction="sum")
    torch.cuda.synchronize()
    grads = torch.autograd.grad(loss, leaves)
    torch.cuda.synchronize()
    want = [loss.detach(), *grads, gated_feed_forward(*few)]
    torch.cuda.synchronize()
    want.append(gated_feed_forward(*many))
    torch.cuda.synchronize()
    for _ in range(5):
        got = [run() for _ in range(20)]
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for one in got for u, v in zip(one, want))
    assert bool(want[0].isfinite()) and not want[1][lab < 0].any() and (live > 0 or not (want[0].any() or want[2].any()))
