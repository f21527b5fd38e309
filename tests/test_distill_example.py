"""The distillation example runs its losses, gradients and optimizers together
and learns: a chain with four successors per token has an entropy of log 4."""

import importlib.util
import math
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("distill_lm", os.path.join(ROOT, "pytorch-opt_amd", "examples",
                                                                             "distill_lm.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_learns_on_the_cpu():
    r = _example().main(["--device", "cpu", "--vocab", "50", "--d", "32", "--steps", "40", "--rows", "8", "--length",
                         "32", "--top", "8"])
    assert r["teacher"][-1] < r["teacher"][0] - 1.0
    assert r["student"][-1] < r["student"][0] - 1.0
    assert math.log(4) - 0.1 < r["teacher_held_out"] < math.log(50) - 1.0


@pytest.mark.gpu
def test_example_learns_on_the_gpu(native_backend):
    r = _example().main(["--vocab", "1000", "--d", "256", "--steps", "80"])
    assert r["teacher"][-1] < r["teacher"][0] - 2.0
    assert r["student"][-1] < r["student"][0] - 2.0
    assert math.log(4) - 0.1 < r["teacher_held_out"] < math.log(1000) - 2.0
    assert r["student_held_out"] < math.log(1000) - 2.0
