"""examples/speculative_decode.py: when it says that it failed."""
import importlib.util
import os

import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "speculative_decode.py")


@pytest.fixture
def example():
    spec = importlib.util.spec_from_file_location("speculative_decode", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("error,status", [(0.0, 0), (2.0 ** -8, 0), (2.0 ** -7, 1), (float("nan"), 1), (float("inf"), 1)])
def test_exit_status(example, monkeypatch, error, status):
    monkeypatch.setattr(example, "main", lambda fmt, steps: error)
    assert example.run(["--fmt", "fp8", "--steps", "2"]) == status


@pytest.mark.parametrize("steps", ["0", "-1"])
def test_no_steps_are_refused(example, monkeypatch, steps):
    """Without a last step nothing would be compared."""
    monkeypatch.setattr(example, "main", lambda fmt, steps: 0.0)
    with pytest.raises(SystemExit) as e:
        example.run(["--steps", steps])
    assert e.value.code == 2


def test_main_refuses_no_steps(example):
    with pytest.raises(ValueError):
        example.main(steps=0)
