"""The example that runs the class-logit operators together: a field distilled
from a teacher's top logits learns its labels. Marked gpu."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parent.parent / "examples" / "semantic_field.py"


def test_semantic_field_learns_its_labels():
    spec = importlib.util.spec_from_file_location("semantic_field", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.main(steps=150)
    # 16 classes: chance is 1 / 16; the sites' regions are far larger than a grid cell
    assert got["last_loss"] < 0.25 * got["first_loss"], got
    assert got["accuracy"] > 0.8 and got["in_top_3"] >= got["accuracy"], got
    assert got["mean_entropy"] > 0.0 > got["mean_logprob"], got
