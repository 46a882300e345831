"""The example that runs the block operators together learns, in both types and
for ragged sizes of the last patch."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

_PATH = Path(__file__).resolve().parents[1] / "examples" / "point_attention.py"


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_example_learns(kind):
    spec = importlib.util.spec_from_file_location("point_attention", _PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.main(points=3_001, steps=40, kind=kind)
    assert losses[-1] < 0.5 * losses[0]
