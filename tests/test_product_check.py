"""CPU: the check of products refuses what is not a number, wherever it stands."""
import numpy as np
import pytest

from product_check import check


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["all", (0, 0), (2, 4)], ids=str)
def test_check_refuses_what_is_not_a_number(bad, where):
    rng = np.random.default_rng(0)
    x, w = rng.normal(size=(3, 7)), rng.normal(size=(5, 7))
    right = (x @ w.T).astype(np.float32)
    check(right, x, w, False, 0)
    got = right.copy()
    got[... if where == "all" else where] = bad
    with pytest.raises(AssertionError):
        check(got, x, w, False, 0)


def test_check_refuses_a_value_that_is_off():
    x, w = np.ones((1, 8)), np.ones((1, 8))
    with pytest.raises(AssertionError):
        check(np.array([[8.001]], np.float32), x, w, False, 0)
