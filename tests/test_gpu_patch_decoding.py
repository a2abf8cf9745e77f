"""A transformers layer's decoding steps through the drop-in of the rule's recurrent form: the same tokens, one at a time, with
the patch and without it, from copies of one cache; and prefill and steps both patched, against the whole row."""
import copy

import pytest
import torch

from macai_b200 import patch
from macai_b200.gated_delta import recurrent_gated_delta_rule

pytestmark = pytest.mark.gpu
M = pytest.importorskip("transformers.models.qwen3_5.modeling_qwen3_5")


def _layer(dt, value_heads):
    cfg = M.Qwen3_5TextConfig(vocab_size=97, hidden_size=128, intermediate_size=256, num_hidden_layers=1, layer_types=["linear_attention"],
                              num_attention_heads=2, num_key_value_heads=1, head_dim=64, linear_key_head_dim=64,
                              linear_value_head_dim=64, linear_num_key_heads=2, linear_num_value_heads=value_heads)
    torch.manual_seed(0)
    layer = M.Qwen3_5GatedDeltaNet(cfg, 0)
    # transformers' own forms, also where another library's kernels were found
    layer.chunk_gated_delta_rule, layer.recurrent_gated_delta_rule = M.torch_chunk_gated_delta_rule, M.torch_recurrent_gated_delta_rule
    layer.norm = M.Qwen3_5RMSNormGated(64, eps=cfg.rms_norm_eps)
    layer = layer.to("cuda", dt).eval()
    return layer, M.DynamicCache(config=cfg)


def _near(a, b, bar):
    return a.dtype == b.dtype and float((a.float() - b.float()).norm() / b.float().norm()) < bar


# an output passes about ten roundings of the layer's type on either side (2^-8 and 2^-11 at most, about a third of that rms), in
# float32 sums of a few hundred terms in another order
BARS = [(torch.float32, 1e-4), (torch.bfloat16, 2e-2), (torch.float16, 2.5e-3)]


@torch.no_grad()
@pytest.mark.parametrize("dt,bar", BARS)
@pytest.mark.parametrize("value_heads", [2, 4])
def test_decoding_steps(dt, bar, value_heads):
    layer, cache = _layer(dt, value_heads)
    x = torch.randn(3, 30, 128, generator=torch.Generator().manual_seed(1)).to(dt).cuda()
    layer(x[:, :20], cache_params=cache)
    ours = copy.deepcopy(cache)
    for t in range(20, 30):
        at = x[:, t:t + 1]
        want = layer(at, cache_params=cache)
        with patch.installed(model=layer, recurrent=True):
            assert layer.recurrent_gated_delta_rule is recurrent_gated_delta_rule
            assert _near(layer(at, cache_params=ours), want, bar)
        assert _near(ours.layers[0].recurrent_states, cache.layers[0].recurrent_states, bar)


@torch.no_grad()
def test_prefill_and_steps():
    dt = torch.bfloat16   # (the chunked form refuses the others)
    layer, cache = _layer(dt, 4)
    x = torch.randn(2, 33, 128, generator=torch.Generator().manual_seed(2)).to(dt).cuda()
    whole = layer(x)
    with patch.installed(model=layer, recurrent=True):
        got = [layer(x[:, :21], cache_params=cache)] + [layer(x[:, t:t + 1], cache_params=cache) for t in range(21, 33)]
    # the chunked rule's own bar and the layer's roundings
    assert _near(torch.cat(got, 1), whole, 3e-2)
