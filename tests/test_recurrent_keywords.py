"""The drop-in's keywords: what it does not know it refuses (another scale, another layout would give other numbers)."""
import pytest
import torch

from macai_b200.gated_delta import recurrent_gated_delta_rule


@pytest.mark.parametrize("kw", [{"scale": 0.5}, {"head_first": True}, {"inplace_final_state": True}, {"initial_sate": None}])
def test_unknown_keywords(kw):
    q, v, g = torch.zeros(1, 1, 2, 64), torch.zeros(1, 1, 4, 64), torch.zeros(1, 1, 4)
    with pytest.raises(TypeError, match=next(iter(kw))):
        recurrent_gated_delta_rule(q, q, v, g, g, **kw)


def test_known_keywords():
    """transformers' own, and a cu_seqlens of None: past the keywords, refused only for want of a GPU."""
    q, v, g = torch.zeros(1, 1, 2, 64), torch.zeros(1, 1, 4, 64), torch.zeros(1, 1, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        recurrent_gated_delta_rule(q, q, v, g=g, beta=g, initial_state=None, output_final_state=True, use_qk_l2norm_in_kernel=True,
                                   cu_seqlens=None)
