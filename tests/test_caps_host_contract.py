"""Caps that the C entry points refuse, before any device work (no pointer is followed): as the
Python functions, they take 0 (none) and 1e-30 to 1e30. Beyond, the reciprocal of a cap or
twice the cap leaves float32's range."""

import pytest

from test_attend_host_contract import attend, logprobs
from test_rows_host_contract import INVALID, cache


@pytest.mark.parametrize("cap", [1e-45, 1e-39, 1e-38, 9e-31, 1.1e30, 2e38, 3.4e38])
def test_caps_out_of_range(cap):
    assert attend(cache(), cap=cap) == INVALID
    assert logprobs(cap=cap) == INVALID
