"""The gated delta rule's recurrent form against its float64 recurrence: single tokens and runs, types, head layouts, slots
(idle, missing, contested), the drop-in, graphs, streams."""
import pytest
import torch

from macai_b200.gated_delta import chunk_gated_delta_rule, gated_delta_step, recurrent_gated_delta_rule
from oracle import decoder_steps_f64 as steps

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}   # half a step of the subnormal numbers


def _inputs(B, T, HK, H, DK, DV, dt, vdt=None, seed=0, decay=1.0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k = rand(B, T, HK, DK).to(dt).cuda(), rand(B, T, HK, DK).to(dt).cuda()
    v = rand(B, T, H, DV).to(vdt or dt).cuda()
    g = (-decay * torch.rand(B, T, H, generator=gen)).cuda()
    beta = torch.rand(B, T, H, generator=gen).cuda()
    return q, k, v, g, beta, (rand(B, H, DK, DV) * 0.3).cuda()


def _near(got, want, bound, dt=torch.float32):
    """|got - want| <= the bound of the float32 arithmetic and the output's own rounding."""
    err = (got.double() - want).abs()
    assert bool((err <= bound + HALF[dt] * (want.abs() + bound) + TINY[dt] + 1e-30).all()), float((err - bound).max())


@pytest.mark.parametrize("B,T,HK,H,DK,DV", [(1, 1, 1, 1, 128, 128), (3, 1, 2, 4, 128, 128), (2, 7, 2, 2, 64, 96),
                                            (5, 8, 1, 3, 32, 32), (2, 9, 2, 6, 96, 160), (1, 17, 1, 2, 256, 256),
                                            (2, 33, 2, 2, 160, 64), (40, 2, 4, 8, 128, 128)])
@pytest.mark.parametrize("dt,vdt", [(torch.bfloat16, None), (torch.bfloat16, torch.float32), (torch.float16, None),
                                    (torch.float16, torch.float32), (torch.float32, None)])
def test_recurrence(B, T, HK, H, DK, DV, dt, vdt):
    q, k, v, g, beta, s0 = _inputs(B, T, HK, H, DK, DV, dt, vdt, seed=T)
    o, s, eo, es = steps.rule_step(q, k, v, g, beta, s0, l2norm=True)
    state = s0.clone()
    got = gated_delta_step(q, k, v, g, beta, state, use_qk_l2norm_in_kernel=True)
    assert got.dtype == dt and got.shape == (B, T, H, DV)
    _near(got, o, eo, dt)
    _near(state, s, es)
    # the drop-in: the same bits, its inputs left alone
    kept = s0.clone()
    got2, sT = recurrent_gated_delta_rule(q, k, v, g, beta, s0, True, True)
    assert torch.equal(got2, got) and torch.equal(sT, state) and torch.equal(s0, kept)


@pytest.mark.parametrize("B,HK,H,DK,DV", [(38, 4, 4, 32, 32), (75, 1, 2, 64, 96), (50, 1, 3, 96, 128), (19, 4, 8, 128, 128),
                                          (160, 1, 1, 160, 64), (38, 2, 4, 256, 256), (300, 2, 4, 128, 32)])
@pytest.mark.parametrize("dt,vdt", [(torch.bfloat16, None), (torch.bfloat16, torch.float32), (torch.float16, None),
                                    (torch.float16, torch.float32), (torch.float32, None)])
def test_tokens_of_many_heads(B, HK, H, DK, DV, dt, vdt):
    """One token of more heads than the GPU has SMs (another kernel), with a state, without one, and without keeping it."""
    q, k, v, g, beta, s0 = _inputs(B, 1, HK, H, DK, DV, dt, vdt, seed=DK)
    for norm in (True, False):
        o, s, eo, es = steps.rule_step(q, k, v, g, beta, s0, l2norm=norm)
        got, sT = recurrent_gated_delta_rule(q, k, v, g, beta, s0, True, norm)
        _near(got, o, eo, dt)
        _near(sT, s, es)
        only, none = recurrent_gated_delta_rule(q, k, v, g, beta, s0, False, norm)
        assert none is None and torch.equal(only, got)
    o, s, eo, es = steps.rule_step(q, k, v, g, beta, torch.zeros_like(s0), l2norm=True)
    got, sT = recurrent_gated_delta_rule(q, k, v, g, beta, None, True, True)
    _near(got, o, eo, dt)
    _near(sT, s, es)


def test_without_norm_and_without_a_state():
    q, k, v, g, beta, s0 = _inputs(2, 5, 2, 4, 64, 64, torch.float32, seed=3)
    k = k * 0.1
    o, s, eo, es = steps.rule_step(q, k, v, g, beta, torch.zeros_like(s0))
    got, sT = recurrent_gated_delta_rule(q, k, v, g, beta, None, output_final_state=True)
    _near(got, o, eo)
    _near(sT, s, es)
    got2, none = recurrent_gated_delta_rule(q, k, v, g, beta)
    assert none is None and torch.equal(got, got2)


@pytest.mark.parametrize("decay", [0.0, 30.0, 1000.0])
def test_decays(decay):
    """No decay at all, and decays whose factor is nearly or exactly 0."""
    q, k, v, g, beta, s0 = _inputs(2, 3, 1, 2, 128, 128, torch.bfloat16, seed=4, decay=decay)
    o, s, eo, es = steps.rule_step(q, k, v, g, beta, s0, l2norm=True)
    got, sT = recurrent_gated_delta_rule(q, k, v, g, beta, s0, True, True)
    tiny = 2.0 ** -126 * 1000   # factors below the normal range may come out as 0
    _near(got, o, eo + tiny, torch.bfloat16)
    _near(sT, s, es + tiny)


def test_a_row_of_zeros():
    q, k, v, g, beta, s0 = _inputs(1, 2, 1, 1, 128, 128, torch.bfloat16, seed=5)
    q[:, 0], k[:, 1] = 0, 0
    o, s, eo, es = steps.rule_step(q, k, v, g, beta, s0, l2norm=True)
    got, sT = recurrent_gated_delta_rule(q, k, v, g, beta, s0, True, True)
    assert not got[:, 0].any()
    _near(got, o, eo, torch.bfloat16)
    _near(sT, s, es)


def test_slots():
    """A pool in any order: read and written in place, or from one slot into another; other slots stay as they are."""
    q, k, v, g, beta, s0 = _inputs(4, 2, 1, 2, 64, 64, torch.bfloat16, seed=6)
    pool = torch.randn(11, 2, 64, 64, device="cuda")
    slots = torch.tensor([7, 0, -1, 10], dtype=torch.int32, device="cuda")
    live = [0, 1, 3]
    o, s, eo, es = steps.rule_step(q, k, v, g, beta, pool[slots.long().clamp_min(0)], l2norm=True)
    a = pool.clone()
    got = gated_delta_step(q, k, v, g, beta, a, slots, use_qk_l2norm_in_kernel=True)
    assert not got[2].any()
    _near(got[live], o[live], eo[live], torch.bfloat16)
    at = slots.long()[live]
    _near(a[at], s[live], es[live])
    rest = [i for i in range(11) if i not in (7, 0, 10)]
    assert torch.equal(a[rest], pool[rest])
    b = pool.clone()
    out = torch.tensor([1, 2, -1, 3], dtype=torch.int32, device="cuda")
    got2 = gated_delta_step(q, k, v, g, beta, b, slots, out, use_qk_l2norm_in_kernel=True)
    assert torch.equal(got2, got) and torch.equal(b[out.long()[live]], a[at])
    rest = [i for i in range(11) if i not in (1, 2, 3)]
    assert torch.equal(b[rest], pool[rest])


def test_slots_that_cannot_be():
    """A slot the pool does not have, and slots that another request writes: NaN, and no state changes. A slot that several
    requests only read is fine."""
    q, k, v, g, beta, _ = _inputs(5, 1, 1, 2, 64, 64, torch.bfloat16, seed=7)
    pool = torch.randn(6, 2, 64, 64, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    a = pool.clone()
    o = gated_delta_step(q, k, v, g, beta, a, i32(0, 3, 3, 6, 1 << 30))
    assert bool(o[1:].isnan().all()) and bool(o[0].isfinite().all())
    assert torch.equal(a[1:], pool[1:]) and not torch.equal(a[0], pool[0])
    a = pool.clone()   # request 1 writes what request 2 reads; requests 3 and 4 read one slot
    o = gated_delta_step(q, k, v, g, beta, a, i32(0, 1, 2, 5, 5), i32(0, 2, 3, 4, -1))
    assert bool(o[1].isnan().all()) and bool(o[[0, 2, 3]].isfinite().all()) and not o[4].any()
    assert torch.equal(a[[1, 2, 5]], pool[[1, 2, 5]])
    a = pool.clone()
    o = gated_delta_step(q, k, v, g, beta, a, i32(5, 5, 5, 5, 5), i32(0, 1, 2, 3, 4))
    assert bool(o.isfinite().all()) and torch.equal(a[5], pool[5])


@pytest.mark.parametrize("B", [2, 100])
def test_many_heads_and_an_empty_pool(B):
    """The same refusals where heads outnumber the SMs (another kernel), and a pool without a slot."""
    q, k, v, g, beta, _ = _inputs(B, 1, 2, 4, 64, 64, torch.bfloat16, seed=12)
    pool = torch.randn(B + 3, 4, 64, 64, device="cuda")
    slots = torch.arange(B, dtype=torch.int32, device="cuda")
    slots[1] = B + 3
    if B > 2:
        slots[7], slots[40], slots[50] = -5, 41, 1 << 30
    live = [i for i in range(B) if i not in (1, 7, 40, 41, 50)]
    o, s, eo, es = steps.rule_step(q[live], k[live], v[live], g[live], beta[live], pool[live], l2norm=True)
    a = pool.clone()
    got = gated_delta_step(q, k, v, g, beta, a, slots, use_qk_l2norm_in_kernel=True)
    _near(got[live], o, eo, torch.bfloat16)
    _near(a[live], s, es)
    rest = [i for i in range(B + 3) if i not in live]
    assert torch.equal(a[rest], pool[rest]) and bool(got[1].isnan().all())
    if B > 2:
        assert not got[7].any() and bool(got[[40, 41, 50]].isnan().all())
    none = gated_delta_step(q, k, v, g, beta, pool[:0], slots)
    assert bool(none[[i for i in range(B) if B == 2 or i != 7]].isnan().all())


def test_a_run_equals_its_tokens():
    """A run of 13 tokens, the same tokens one call each, and (within the chunked kernels' bar) the chunked form."""
    q, k, v, g, beta, s0 = _inputs(2, 13, 2, 4, 128, 128, torch.bfloat16, seed=8)
    o, sT = recurrent_gated_delta_rule(q, k, v, g, beta, s0, True, True)
    state = s0.clone()
    rows = [gated_delta_step(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], g[:, t:t + 1], beta[:, t:t + 1], state,
                             use_qk_l2norm_in_kernel=True) for t in range(13)]
    assert torch.equal(torch.cat(rows, 1), o) and torch.equal(state, sT)
    oc, sc = chunk_gated_delta_rule(q, k, v, g, beta, initial_state=s0, output_final_state=True, use_qk_l2norm_in_kernel=True)
    assert float((oc.float() - o.float()).norm() / o.float().norm()) < 2e-2
    assert float((sc - sT).norm() / sT.norm()) < 2e-2


def test_no_tokens_and_no_requests():
    q, k, v, g, beta, s0 = _inputs(2, 0, 1, 2, 64, 64, torch.bfloat16)
    state = s0.clone()
    assert gated_delta_step(q, k, v, g, beta, state).shape == (2, 0, 2, 64) and torch.equal(state, s0)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    gated_delta_step(q[:1], k[:1], v[:1], g[:1], beta[:1], state, i32(0), i32(1))
    assert torch.equal(state[1], s0[0])
    assert gated_delta_step(q[:0], k[:0], v[:0], g[:0], beta[:0], state).shape == (0, 0, 2, 64)


def test_views_and_other_types():
    """q, k, v as views of one projection, g and beta in 16 bits, a key and value of another type than the query's."""
    B, T, H, D = 2, 3, 2, 64
    qkv = torch.randn(B, T, 3 * H * D, device="cuda", dtype=torch.bfloat16)
    q, k, v = (x.view(B, T, H, D) for x in qkv.split(H * D, -1))
    g, beta = -torch.rand(B, T, H, device="cuda").half(), torch.rand(B, T, H, device="cuda").half()
    s0 = torch.zeros(B, H, D, D, device="cuda")
    a, _ = recurrent_gated_delta_rule(q, k, v, g, beta, s0, False, True)
    b, _ = recurrent_gated_delta_rule(q.contiguous(), k.contiguous(), v.contiguous(), g.float(), beta.float(), s0, False, True)
    assert torch.equal(a, b)
    c, _ = recurrent_gated_delta_rule(q, k.float(), v.half(), g, beta, s0, False, True)
    d, _ = recurrent_gated_delta_rule(q, k, v.half().bfloat16(), g, beta, s0, False, True)
    assert torch.equal(c, d)


def test_captured_steps():
    """Steps captured into a graph and replayed on another stream, slots changed between replays."""
    q, k, v, g, beta, _ = _inputs(3, 1, 1, 2, 128, 128, torch.bfloat16, seed=9)
    pool = torch.randn(5, 2, 128, 128, device="cuda") * 0.1
    eager = pool.clone()
    slots = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    gated_delta_step(q, k, v, g, beta, pool.clone(), slots)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        o = gated_delta_step(q, k, v, g, beta, pool, slots)
    for order in ([0, 1, 2], [4, -1, 0], [1, 2, 3]):
        slots.copy_(torch.tensor(order, dtype=torch.int32))
        want = gated_delta_step(q, k, v, g, beta, eager, slots)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(pool, eager)


def test_version_counter_and_gradients():
    q, k, v, g, beta, s0 = _inputs(1, 1, 1, 1, 64, 64, torch.bfloat16)
    before = s0._version
    gated_delta_step(q, k, v, g, beta, s0)
    assert s0._version == before + 1
    with pytest.raises(RuntimeError, match="no gradient"):
        gated_delta_step(q.requires_grad_(True), k, v, g, beta, s0)
    with pytest.raises(RuntimeError, match="no gradient"):
        recurrent_gated_delta_rule(q, k, v, g, beta, s0)
    with torch.no_grad():
        gated_delta_step(q, k, v, g, beta, s0)


def test_refusals():
    q, k, v, g, beta, s0 = _inputs(2, 1, 1, 2, 64, 64, torch.bfloat16)
    i32 = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for bad in (s0[:1], s0.half(), s0.cpu(), s0.transpose(2, 3), s0[:, :1], s0.flatten()[1:8193].view(1, 2, 64, 64)):
        with pytest.raises(ValueError, match="state|slots"):
            gated_delta_step(q, k, v, g, beta, bad)
    for kw in ({"slots": i32.long()}, {"slots": i32[:1]}, {"slots": i32.cpu()}, {"out_slots": i32},
               {"slots": i32, "out_slots": i32.long()}):
        with pytest.raises(ValueError, match="slots"):
            gated_delta_step(q, k, v, g, beta, s0, **kw)
    with pytest.raises(ValueError, match="initial_state"):
        recurrent_gated_delta_rule(q, k, v, g, beta, s0[:1])


def test_a_value_of_another_type():
    """A float16 value beside bfloat16 queries is not rounded to their type; inference mode's tensors are taken."""
    q, k, v, g, beta, s0 = _inputs(2, 3, 2, 2, 64, 64, torch.bfloat16, torch.float16, seed=40)
    a, sa = recurrent_gated_delta_rule(q, k, v, g, beta, s0, True, True)
    b, sb = recurrent_gated_delta_rule(q, k, v.float(), g, beta, s0, True, True)
    assert torch.equal(a, b) and torch.equal(sa, sb)
    with torch.inference_mode():
        pool = s0.clone()
        c = gated_delta_step(q, k, v, g, beta, pool, use_qk_l2norm_in_kernel=True)
    assert torch.equal(a, c) and torch.equal(sa, pool)


@pytest.mark.parametrize("HK,H,DK,DV", [(2, 4, 128, 128), (1, 3, 64, 96), (2, 2, 96, 160), (1, 2, 256, 64), (4, 8, 32, 32)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_same_bits_in_any_company(HK, H, DK, DV, dt):
    """Tokens one at a time of one request at a time, and a run of all requests: the same bits."""
    q, k, v, g, beta, s0 = _inputs(40, 11, HK, H, DK, DV, dt, seed=41)
    o, state = recurrent_gated_delta_rule(q, k, v, g, beta, s0, True, True)
    for b in (0, 7, 39):
        pool = s0[b:b + 1].clone()
        for t in range(11):
            at = slice(b, b + 1), slice(t, t + 1)
            assert torch.equal(gated_delta_step(q[at], k[at], v[at], g[at], beta[at], pool, use_qk_l2norm_in_kernel=True), o[at])
        assert torch.equal(pool[0], state[b])
    pool, at = s0.clone(), slice(0, 1)
    assert torch.equal(gated_delta_step(q[:, at], k[:, at], v[:, at], g[:, at], beta[:, at], pool, use_qk_l2norm_in_kernel=True),
                       o[:, at])
