"""GPU: the example that quantises experts, merges into one, routes tokens through them and differentiates runs and
gives what its parts promise."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "fp4_experts.py"


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_example(fmt, cuda_device):
    spec = importlib.util.spec_from_file_location("fp4_experts", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.run(experts=5, tokens=203, hidden=256, inner=416, fmt=fmt)
    # e2m1 keeps one mantissa bit: a uniform error within half a step is 10 to 20 % of the values' norm
    assert 0.02 < got["quantisation_error"] < 0.2
    assert got["largest_change_elsewhere"] == 0.0
    # the merge rounds the sum to the same grid
    assert 0.02 < got["merge_error"] < 0.2
    # two products of tokens quantised on the way, each within a grid's error, and a non-linearity between
    assert 0.0 < got["output_error"] < 0.4
    assert math.isfinite(got["gradient_norm"]) and got["gradient_norm"] > 0.0
