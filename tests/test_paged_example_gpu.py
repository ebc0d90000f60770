"""The serving example runs, takes all of its paths and gives the rows that
the same layers give over whole sequences."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_paged_serving_example(capsys):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import paged_serving
        steps, worst = paged_serving.main()
    finally:
        sys.path.pop(0)
    assert steps["packed"] > 0 and steps["paged"] > 0 and steps["refused"] > 0
    assert worst < 2e-2
    assert "10 requests" in capsys.readouterr().out
