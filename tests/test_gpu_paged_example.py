"""The example of a caller's own speculative step over the paged cache operators: every continuation
decoded from drafted trees is the one that decoding a row at a time gives, in fewer steps."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_trees_give_the_rows_tokens():
    import paged_step
    same, steps = paged_step.main(4, 40)
    assert same == 4
    assert steps < 39
