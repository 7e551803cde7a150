"""The bounded-cache example without a GPU: layers that it must not start."""
import os
import sys

import pytest

EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "serving-engine_b200", "examples")
sys.path.insert(0, EXAMPLES)


@pytest.mark.parametrize("capacity,budget,sinks,recent", [(64, 64, 4, 8), (64, 65, 4, 8), (64, 0, 0, 0), (64, 32, 30, 3),
                                                          (64, 32, -1, 3), (64, 32, 1, -3)])
def test_layer_refuses_budgets_that_make_no_room(capacity, budget, sinks, recent):
    """An eviction has to leave a free row, or the next token is written past the block table."""
    from bounded_cache import BoundedLayer
    with pytest.raises(ValueError, match="budget"):
        BoundedLayer(1, 4, 2, 64, capacity=capacity, budget=budget, sinks=sinks, recent=recent)
