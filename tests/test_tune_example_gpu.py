"""The tuning example end to end: losses, reversible backward and 8-bit optimizer together move the model the way
the data ask for."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tune():
    spec = importlib.util.spec_from_file_location("tune", Path(__file__).resolve().parents[1] / "examples" / "tune.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_preference_margin_rises(tune):
    margins = tune.main(["--mode", "preference", "--steps", "25", "--batch", "4", "--length", "64", "--layers", "2",
                         "--vocab", "1001", "--lr", "3e-3"])
    assert abs(margins[0]) < 0.05  # the model is its own reference at first
    assert sum(margins[-5:]) / 5 > 0.5


def test_policy_reward_rises(tune):
    rewards = tune.main(["--mode", "policy", "--steps", "25", "--batch", "8", "--length", "64", "--layers", "2",
                         "--vocab", "1001", "--lr", "3e-3"])
    assert 0.4 < rewards[0] < 0.6
    assert sum(rewards[-5:]) / 5 > 0.75
