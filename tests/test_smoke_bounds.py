"""The smoke's comparison against error bounds, without a GPU."""

import pytest
import torch

from __graft_entry__ import _within

ONE = torch.ones(3, dtype=torch.float64)
INSIDE = (ONE + 0.25, ONE, ONE)


def test_the_worst_of_several_counts():
    assert _within("a", [INSIDE, (ONE + 0.5, ONE, ONE), INSIDE]) == 0.5


@pytest.mark.parametrize("bad", [3.0, float("nan"), float("inf")])
@pytest.mark.parametrize("place", [0, 1, 2])
def test_an_error_past_its_bound_or_no_number_fails(bad, place):
    wrong = ONE.clone()
    wrong[1] = bad
    pairs = [INSIDE, INSIDE]
    pairs.insert(place, (wrong, ONE, ONE))
    with pytest.raises(AssertionError, match="error bound"):
        _within("a", pairs)
