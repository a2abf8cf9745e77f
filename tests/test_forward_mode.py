"""Forward-mode derivatives (torch.autograd.forward_ad): the operators have none, and say so instead of returning a result
without its tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

gpu = pytest.mark.gpu
DEV = "cuda"


def test_a_dual_tensor_is_recorded():
    """On the CPU: a call with a tangent goes to the autograd function, which refuses it, also without gradients."""
    from macai_b200._call import recorded
    x, plain = torch.randn(3), torch.randn(3)
    assert not recorded(x, None)
    with fwad.dual_level():
        d = fwad.make_dual(x, torch.ones(3))
        assert recorded(plain, None, d) and not recorded(plain, None, x)
        with torch.no_grad():
            assert recorded(d)
    assert not recorded(x)


@gpu
def test_the_softmax_layers_operators():
    from macai_b200.norm import add_rms_norm, add_rms_norm_fp8
    from macai_b200.rotary import rotary, rotary_table
    from macai_b200.window_attention import window_attention, window_attention_step
    x, w = torch.randn(4, 64, device=DEV), torch.ones(64, device=DEV)
    q, k, v = (torch.randn(1, 8, 2, 64, device=DEV).to(torch.bfloat16) for _ in range(3))
    table = rotary_table(8, 16)
    cache = [torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    L = torch.zeros(1, dtype=torch.int32, device=DEV)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: add_rms_norm(dual(x), x, w), lambda: add_rms_norm(x, None, dual(w)),
                     lambda: rotary(q, dual(k), table), lambda: window_attention(q, k, dual(v)),
                     lambda: add_rms_norm_fp8(dual(x), x, w),
                     lambda: window_attention_step(dual(q[:, :1]), k[:, :1], v[:, :1], *cache, L)):
            for mode in (torch.enable_grad(), torch.no_grad()):
                with mode, pytest.raises((NotImplementedError, RuntimeError), match="jvp|no gradient"):
                    call()
        y, _ = add_rms_norm(x, x, w)      # no tangent among the inputs: as ever
    assert torch.equal(y, add_rms_norm(x, x, w)[0])
