"""The example runs its operators together: the counting task's loss falls, and single tokens through the rolling cache agree
with the whole row. Both sides of the second round P and the output to bfloat16 (2^-8 each) of values of order 1, and the
projection adds 256 of them: 0.1 is ten standard deviations."""
import importlib.util
import os

import pytest

gpu = pytest.mark.gpu


@gpu
def test_hybrid_decoder():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_decoder.py")
    spec = importlib.util.spec_from_file_location("hybrid_decoder", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    model, table, first, last = m.train(steps=25, B=2, T=150)
    assert last < 0.7 * first, (first, last)
    assert m.serve(model, table, B=2, prompt=70, more=40) < 0.1
