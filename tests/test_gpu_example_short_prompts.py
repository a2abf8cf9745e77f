"""The example's model served from prompts shorter than the convolution's filter: its single tokens against the whole row."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_decoder.py")
    spec = importlib.util.spec_from_file_location("hybrid_decoder", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("prompt", [1, 2, 3, 4])
def test_short_prompts(example, prompt):
    m = example
    torch.manual_seed(prompt)
    model = m.Decoder().cuda().bfloat16()
    table = m.rotary_table(256, m.WIDTH // 4, device="cuda")
    start = torch.randint(0, m.VOCAB, (5, prompt), device="cuda")
    tokens, logits = m.generate(model, table, start, 12)
    with torch.no_grad():
        whole = model(tokens, table)[:, prompt - 1:prompt + 11]
    # logits of order 1 after about twenty roundings to bfloat16 (2^-9 rms) on either side: 0.02 rms; ten times that at most
    assert float((whole.float() - logits.float()).abs().max()) < 0.2


@torch.no_grad()
@pytest.mark.parametrize("prompt", [1, 2, 3, 7])
def test_the_mixer_alone(example, prompt):
    """The rule's mixer, where a lost input is a large part of the output."""
    m = example
    torch.manual_seed(10 + prompt)
    mixer = m.DeltaMixer().cuda().bfloat16()
    x = torch.randn(3, prompt + 6, m.DIM, device="cuda", dtype=torch.bfloat16)
    whole = mixer(x)
    _, before, state = mixer.prefill(x[:, :prompt])
    assert before.shape[1] == 3
    for t in range(prompt, prompt + 6):
        y = mixer.step(x[:, t:t + 1], before, state)
        # the chunked rule's roundings (2e-2 of the norm at most, the bar of its own tests) and the projections'
        assert float((y - whole[:, t:t + 1]).float().norm() / whole[:, t:t + 1].float().norm()) < 3e-2
