"""The rotary table has no gradient: a table that needs one is refused, not left without it."""
import pytest
import torch

gpu = pytest.mark.gpu


@gpu
def test_a_table_that_needs_a_gradient_is_refused():
    from macai_b200.rotary import rotary, rotary_table
    q = torch.randn(1, 4, 2, 16, device="cuda", requires_grad=True)
    table = rotary_table(8, 16).requires_grad_(True)
    for x in (q, q.detach()):
        with pytest.raises(RuntimeError, match="no gradient"):
            rotary(x, None, table)
    with torch.no_grad():
        o, _ = rotary(q, None, table)
    assert torch.equal(o, rotary(q.detach(), None, table.detach())[0])
