"""The serving example: drafted trees over the paged cache say what one token at a time says."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_serving_step():
    spec = importlib.util.spec_from_file_location(
        "serving_step", os.path.join(ROOT, "examples", "serving_step.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    same, one, many = example.main()
    assert same
    assert many.steps < one.steps
    for s in (one, many):  # no block lost: the free ones and the tables' are all of them
        left = s.count.item()
        used = [t for row, n in zip(s.table.tolist(), s.lens.tolist())
                for t in row[:-(-n // example.BLOCK)]]
        assert sorted(used + s.free[:left].tolist()) == list(range(example.BLOCKS))
        assert all(t >= 8 for r, p in zip(s.tokens, s.prompt) for t in r[p:])
