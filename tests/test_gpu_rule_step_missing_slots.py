"""A request whose slot the pool does not have neither reads nor writes one: it contests no other request's slot. Runs of any
number of tokens, none among them."""
import pytest
import torch

from macai_b200.gated_delta import gated_delta_step

pytestmark = pytest.mark.gpu


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("T", [1, 2, 9])
@pytest.mark.parametrize("slots,out,live,bad", [
    ((0, 99), (1, 1), (0,), (1,)),                    # reads a slot that is not there, would write another's
    ((0, 1), (1, 4), (0,), (1,)),                     # reads the slot another writes, would write one that is not there
    ((0, 4, 2), (1, 1, 1 << 30), (0,), (1, 2)),       # both beside one that holds
    ((0, 1, 99), (2, 2, 2), (), (0, 1, 2)),           # two that hold still contest
    ((0, 99, 1), (3, 1, 1), (0, 2), (1,)),
    ((2, -1, 99), (2, 2, 2), (0,), (2,))])        # an idle one and a missing one
def test_missing_slots_contest_nothing(T, slots, out, live, bad):
    B, H, D = len(slots), 3, 64
    gen = torch.Generator().manual_seed(T)
    rand = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    q, k, v = (rand(B, T, H, D).bfloat16() for _ in range(3))
    g, beta = -torch.rand(B, T, H, generator=gen).cuda(), torch.rand(B, T, H, generator=gen).cuda()
    pool = rand(4, H, D, D)
    a = pool.clone()
    o = gated_delta_step(q, k, v, g, beta, a, _i32(*slots), _i32(*out), use_qk_l2norm_in_kernel=True)
    written = []
    for b in live:   # the same bits as alone
        one, at = pool.clone(), slice(b, b + 1)
        want = gated_delta_step(q[at], k[at], v[at], g[at], beta[at], one, _i32(slots[b]), _i32(out[b]), use_qk_l2norm_in_kernel=True)
        assert bool(want.isfinite().all()) and torch.equal(o[b], want[0]) and torch.equal(a[out[b]], one[out[b]])
        written.append(out[b])
    rest = [i for i in range(4) if i not in written]
    assert torch.equal(a[rest], pool[rest])
    assert all(bool(o[b].isnan().all()) for b in bad)
    assert all(not o[b].any() for b in range(B) if b not in live and b not in bad)


def test_no_tokens():
    """A run of no tokens copies its state, whatever a missing slot's request names."""
    pool = torch.randn(4, 2, 64, 64, device="cuda")
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    a = pool.clone()
    gated_delta_step(z(2, 0, 2, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), z(2, 0, 2).float(), z(2, 0, 2).float(), a, _i32(0, 99), _i32(1, 1))
    assert torch.equal(a[1], pool[0]) and torch.equal(a[[0, 2, 3]], pool[[0, 2, 3]])
