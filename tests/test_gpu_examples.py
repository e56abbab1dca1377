"""The example layers run the operators together as a model would."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_layers.py")


def _load():
    spec = importlib.util.spec_from_file_location("hybrid_layers", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_tokens_after_a_prompt_match_one_prompt():
    # two paths through bf16 products and roundings: a few bf16 ulp (2^-8) of the result
    assert _load().serve() <= 4 * 2.0 ** -8


def test_training_steps_lower_the_loss():
    losses = _load().train()
    assert losses[-1] < losses[0]
