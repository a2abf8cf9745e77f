"""window_attention_step writes the caches in place, and autograd knows: a tensor saved for a gradient that the step has
changed since is refused, not used."""
import pytest
import torch

from test_gpu_window_attention import BF, DEV, _inputs

gpu = pytest.mark.gpu


@gpu
def test_a_saved_cache_that_changed_is_noticed():
    from macai_b200.window_attention import window_attention_step
    q, k, v, _ = _inputs(2, 1, 1, 4, 2, 64, BF)
    kc, vc = (torch.randn(2, 32, 2, 64, device=DEV).to(BF) for _ in range(2))
    L = torch.full((2,), 5, dtype=torch.int32, device=DEV)
    before = kc._version, vc._version
    w = torch.ones(64, device=DEV, dtype=BF, requires_grad=True)
    for cache in (kc, vc):
        y = (cache * w).sum()
        with torch.no_grad():
            window_attention_step(q, k, v, kc, vc, L)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    assert kc._version > before[0] and vc._version > before[1]
    with torch.inference_mode():
        a, b = (torch.zeros(2, 32, 2, 64, device=DEV, dtype=BF) for _ in range(2))
        window_attention_step(q, k, v, a, b, L)
