"""float16's range in window_attention's forward. P is relative to a maximum that is at most 2^8 below the row's, and is
rounded as 2^7 P: besides u P it is within 2^-25 2^-7 of the maximum's own weight, so o within 2^-32 sum_j |v_j|."""
import math

import pytest
import torch

from oracle import layer_steps_f64 as ref
from test_gpu_window_attention import DEV, F, HF, U

gpu = pytest.mark.gpu


def _outlier(n, D):
    """One key that outweighs each of the others by 2^25.5; its value is zero, the others' are one."""
    q, k = torch.zeros(1, 1, 1, D), torch.zeros(1, n, 1, D)
    q[..., 0] = 25.5 * math.log(2)
    k[:, 3, :, 0] = 1
    v = torch.ones(1, n, 1, D)
    v[:, 3] = 0
    return [t.half().to(DEV) for t in (q, k, v)]


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_forward_many_keys_beside_one_that_outweighs_them(D):
    from macai_b200.window_attention import window_attention
    n = 60000
    q, k, v = _outlier(n, D)
    o, r = window_attention(q, k, v, scale=1.0), ref.attention(q, k, v, scale=1.0)
    tol = U[HF] * r.abs() + (U[HF] + F) * r.abs() + n * 2.0 ** -32
    assert ((o.double() - r).abs() <= tol).all(), (float(o[0, 0, 0, 0]), float(r[0, 0, 0, 0]))
