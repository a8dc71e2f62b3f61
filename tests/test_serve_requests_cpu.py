"""examples/serve_requests.py: when it says that it failed."""
import importlib.util
import os

import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_requests.py")


@pytest.fixture
def example():
    spec = importlib.util.spec_from_file_location("serve_requests", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("error,status", [(0.0, 0), (2.0 ** -7, 0), (2.0 ** -6, 1), (float("nan"), 1), (float("inf"), 1)])
def test_exit_status(example, monkeypatch, error, status):
    monkeypatch.setattr(example, "main", lambda fmt, chunk: error)
    assert example.run(["--fmt", "fp8", "--chunk", "2"]) == status


def test_empty_chunks_are_refused(example, monkeypatch):
    with pytest.raises(ValueError):
        example.main(chunk=0)
    monkeypatch.setattr(example, "main", lambda fmt, chunk: 0.0)
    with pytest.raises(SystemExit) as e:
        example.run(["--chunk", "0"])
    assert e.value.code == 2
