"""float16's range in window_attention_step. P is relative to the running maximum and is rounded as 2^15 P: besides u P it is
within 2^-25 2^-15 of the maximum's own weight, so o within 2^-40 sum_j |v_j|."""
import pytest
import torch

from oracle import layer_steps_f64 as ref
from test_gpu_attention_fp16_forward import _outlier
from test_gpu_window_attention import DEV, F, HF, U

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_step_many_keys_beside_one_that_outweighs_them(D):
    from macai_b200.window_attention import window_attention_step
    n = 60000
    q, k, v = _outlier(n, D)
    L = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    o = window_attention_step(q, k[:, -1:].clone(), v[:, -1:].clone(), k, v, L, scale=1.0)
    r = ref.attention(q, k, v, scale=1.0)
    tol = U[HF] * r.abs() + (U[HF] + F) * r.abs() + n * 2.0 ** -40
    assert ((o.double() - r).abs() <= tol).all(), (float(o[0, 0, 0, 0]), float(r[0, 0, 0, 0]))
