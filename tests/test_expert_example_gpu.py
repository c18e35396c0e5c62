"""The experts' feed-forward example on a B200: an INT8 router, the module, and its steps one by one.

Tolerance, derived: the steps round h to bf16 before its e4m3 codes, which moves a code to its neighbour (1/16 to 1/8
of the value) where the half step of bf16 (2^-9) crosses a boundary between codes, for about one value in fifty: 2^-6.8
of h in the mean square, and as much of y where the weights are random.  z and y rounded to bf16 add 2^-9 each.  Bound:
2^-5 of y's norm.
"""
from __future__ import annotations

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "expert_feed_forward.py")


@pytest.mark.parametrize("streams", [1, 64])
def test_example(streams):
    spec = importlib.util.spec_from_file_location("expert_feed_forward", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    out = example.run(streams, 14)
    assert out["rows"] == 14 * streams and sum(out["rows of each expert"]) == 2 * 14 * streams
    assert out["y"].float().isfinite().all()
    assert out["difference"] < 2.0 ** -5
