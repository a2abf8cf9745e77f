"""The example's whole model: its loss and gradients through all operators together, against the same model with torch's own
cross entropy on its logits, and its single tokens against the whole row."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_decoder.py")
    spec = importlib.util.spec_from_file_location("hybrid_decoder", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_loss_and_gradients():
    m = _example()
    torch.manual_seed(0)
    model = m.Decoder().cuda().bfloat16()
    table = m.rotary_table(256, m.WIDTH // 4, device="cuda")
    tokens = torch.randint(0, m.VOCAB, (3, 70), device="cuda")
    loss = model.loss(tokens, table)
    grads = torch.autograd.grad(loss, list(model.parameters()))
    assert all(bool(g.isfinite().all()) and g.shape == p.shape and g.dtype == p.dtype for g, p in zip(grads, model.parameters()))
    assert all(bool(g.any()) for g in grads)
    logits = model(tokens, table)[:, :-1].flatten(0, 1).float()
    other = torch.nn.functional.cross_entropy(logits, tokens[:, 1:].flatten())
    # the logits of order 1 rounded to bfloat16, off by 2^-9 of themselves at most, 207 of them averaged
    assert abs(float(loss) - float(other)) < 2.0 ** -8
    want = torch.autograd.grad(other, list(model.parameters()))
    for (name, _), a, b in zip(model.named_parameters(), grads, want):
        # both sides round the logits' gradient and each operator's output to bfloat16 on the way (about ten roundings of 2^-9
        # rms each, apart from one another): 2^-9 sqrt(20) of the norm, four times that at most
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 0.04, name


def test_single_tokens():
    m = _example()
    torch.manual_seed(1)
    model = m.Decoder().cuda().bfloat16()
    table = m.rotary_table(256, m.WIDTH // 4, device="cuda")
    start = torch.randint(0, m.VOCAB, (4, 50), device="cuda")
    tokens, logits = m.generate(model, table, start, 40)
    assert tokens.shape == (4, 90) and logits.shape == (4, 40, m.VOCAB) and torch.equal(tokens[:, :50], start)
    assert torch.equal(tokens[:, 50:], logits.argmax(-1))
    with torch.no_grad():
        whole = model(tokens, table)[:, 49:89]
    # logits of order 1 after about twenty roundings to bfloat16 (2^-9 rms) on either side: 0.02 rms; ten times that at most
    assert float((whole.float() - logits.float()).abs().max()) < 0.2
