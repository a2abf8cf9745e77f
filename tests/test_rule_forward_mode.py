"""Forward-mode derivatives of the rule and its layer's steps: there are none, and a call with a tangent says so (on the CPU:
the refusal comes before any kernel)."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


def _calls():
    from macai_b200.conv import conv_qkv
    from macai_b200.gated_delta import chunk_gated_delta_rule
    from macai_b200.gated_delta.op import GatedDeltaRule
    from macai_b200.gated_norm import gated_rms_norm
    from macai_b200.gates import gates
    q, k, v = (torch.randn(1, 64, 2, 128).to(torch.bfloat16) for _ in range(3))
    g, beta = -torch.rand(1, 64, 2), torch.rand(1, 64, 2)
    s0 = torch.zeros(1, 2, 128, 128)
    cu = torch.tensor([0, 30, 64])
    b, a = (torch.randn(1, 64, 2).to(torch.bfloat16) for _ in range(2))
    A, bias = torch.rand(2), torch.zeros(2)
    x, cw = torch.randn(1, 64, 768).to(torch.bfloat16), torch.randn(768, 1, 4)
    return [lambda d: chunk_gated_delta_rule(q, d(k), v, g, beta), lambda d: chunk_gated_delta_rule(q, k, v, d(g), beta),
            lambda d: chunk_gated_delta_rule(q, k, v, g, beta, initial_state=d(s0)),
            lambda d: chunk_gated_delta_rule(q, k, d(v), g, beta, cu_seqlens=cu),
            lambda d: GatedDeltaRule.apply(d(q), k, v, g, beta, None), lambda d: gates(b, d(a), A, bias),
            lambda d: gated_rms_norm(d(v), v, torch.ones(128), 1e-6), lambda d: conv_qkv(x, d(cw), 256, 128, 1, 128)]


@pytest.mark.parametrize("i", range(8))
def test_a_tangent_is_refused(i):
    call = _calls()[i]
    with fwad.dual_level():
        for mode in (torch.enable_grad(), torch.no_grad()):
            with mode, pytest.raises(NotImplementedError, match="forward-mode"):
                call(lambda t: fwad.make_dual(t, torch.ones_like(t)))
