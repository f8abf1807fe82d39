"""examples/kv8_steps.py end to end: prompts, decode steps, a fork and a
prefix through the 8-bit operators beside the 16-bit ones."""
import importlib.util
import os

import pytest

pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_example_runs_and_stays_close():
    spec = importlib.util.spec_from_file_location(
        "kv8_steps", os.path.join(ROOT, "examples", "kv8_steps.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    errors, keys = ex.main(["--layers", "2", "--batch", "3", "--prompt", "300", "--steps", "5"])
    # e4m3 holds a normal value to 2^-4, uniformly spread: 2^-4 / sqrt(3) = 0.036
    # at most in the norm of the keys; the outputs take V's error and that of
    # the scores (of a standard deviation near 1), each at most as large, and
    # both are averaged with the values they err in
    assert keys <= 0.036
    for e in errors.values():
        assert max(e) <= 2 * 0.036
