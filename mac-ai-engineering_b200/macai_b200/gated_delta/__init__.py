"""The gated delta rule on B200 (sm_100a): the drop-in, its autograd op and the reference's utilities
(the reference's src/macai/gated_delta/__init__.py exports the same four names), and the recurrent form for decoding."""
from .op import GatedDeltaRule, chunk_gated_delta_rule, l2norm, recurrent_reference
from .step import gated_delta_step, recurrent_gated_delta_rule

__all__ = ["GatedDeltaRule", "chunk_gated_delta_rule", "gated_delta_step", "l2norm", "recurrent_gated_delta_rule",
           "recurrent_reference"]
