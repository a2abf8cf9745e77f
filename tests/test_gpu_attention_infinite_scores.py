"""Queries whose visible scores are all -inf: softmax has no value there, so the result is NaN as the formula's, not the zeros
of a query that sees no key (macai_b200.window_attention and its step)."""
import pytest
import torch

from test_gpu_window_attention import BF, DEV, HF, _inputs, _run

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_query_of_infinite_scores_is_nan(D, dt):
    q, k, v, do = _inputs(1, 300, 300, 2, 1, D, dt, 21)
    k[..., 0] = -1 - k[..., 0].abs()
    want = _run(q, k, v, do, window=100)
    w = q.clone()
    w[0, 170, 1, 0] = float("inf")                  # query 170 of head 1: -inf with every key
    o, dq, dk, dv = _run(w, k, v, do, window=100)
    assert o[0, 170, 1].isnan().all() and dq[0, 170, 1].isnan().all()
    o[0, 170, 1], want[0][0, 170, 1] = 0, 0
    assert torch.equal(o, want[0])                  # no other query
    seen = torch.zeros(300, dtype=torch.bool, device=DEV)
    seen[71:171] = True
    assert dv[:, seen].isnan().all() and dk[:, seen].isnan().all()


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
def test_the_step(dt):
    from macai_b200.window_attention import window_attention_step
    for S, n, D in ((200, 150, 64), (20000, 19000, 128), (700, 5, 256)):
        q, k, v, _ = _inputs(2, 1, 1, 4, 2, D, dt, 22)
        kc, vc = (torch.randn(2, S, 2, D, device=DEV).to(dt) for _ in range(2))
        for t in (k, kc):
            t[..., 0] = -1 - t[..., 0].abs()
        L = torch.tensor([n, -1], dtype=torch.int32, device=DEV)
        want = window_attention_step(q, k, v, kc, vc, L)
        q[0, 0, 2, 0] = q[1, 0, 2, 0] = float("inf")
        o = window_attention_step(q, k, v, kc, vc, L)
        assert o[0, 0, 2].isnan().all() and (o[1] == 0).all()      # the idle request: zeros
        o[0, 0, 2], want[0, 0, 2] = 0, 0
        assert torch.equal(o, want)
