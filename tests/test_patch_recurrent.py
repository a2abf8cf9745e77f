"""install(recurrent=True) routes transformers' single-token form of the rule as well; without it that form is left alone."""
import importlib

import torch

from macai_b200 import patch
from macai_b200.gated_delta import recurrent_gated_delta_rule

PATH = "transformers.models.qwen3_5.modeling_qwen3_5"


def test_names():
    mod = importlib.import_module(PATH)
    before = mod.torch_recurrent_gated_delta_rule, mod.fused_recurrent_gated_delta_rule
    with patch.installed():
        assert (mod.torch_recurrent_gated_delta_rule, mod.fused_recurrent_gated_delta_rule) == before
    with patch.installed(recurrent=True):
        assert mod.torch_recurrent_gated_delta_rule is recurrent_gated_delta_rule
        assert mod.fused_recurrent_gated_delta_rule is recurrent_gated_delta_rule
        assert (PATH, "torch_recurrent_gated_delta_rule") in patch.patched()
    assert (mod.torch_recurrent_gated_delta_rule, mod.fused_recurrent_gated_delta_rule) == before


def test_built_layers():
    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.chunk_gated_delta_rule = lambda *a, **k: "chunk"
            self.recurrent_gated_delta_rule = lambda *a, **k: "recurrent"
    model = torch.nn.Sequential(Layer(), Layer())
    with patch.installed(model=model, recurrent=True):
        assert all(m.recurrent_gated_delta_rule is recurrent_gated_delta_rule for m in model)
    assert all(m.recurrent_gated_delta_rule() == "recurrent" and m.chunk_gated_delta_rule() == "chunk" for m in model)
    with patch.installed(model=model):
        assert all(m.recurrent_gated_delta_rule() == "recurrent" for m in model)
