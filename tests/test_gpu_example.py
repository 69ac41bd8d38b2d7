"""The example that uses the operators together: it learns, with states in 8 bits as with states in 32."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_mixture_of_experts_learns():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_moe.py")
    spec = importlib.util.spec_from_file_location("train_moe", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = {bits: example.train(steps=80, width=96, layers=2, experts=4, state_bits=bits) for bits in (8, 32)}
    for run in losses.values():
        # ln 128 = 4.85 at the start; the chain itself has 1.1 nats
        assert run[0] > 4.5 and sum(run[-10:]) / 10 < 3.0
    assert abs(sum(losses[8][-10:]) - sum(losses[32][-10:])) / 10 < 0.3
