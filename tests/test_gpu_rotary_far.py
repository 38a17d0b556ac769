"""Head norms with rotation where the small tests of test_gpu_rotary.py do not reach: positions
past 32 bits, and prompts so large that a wave takes several rounds of heads. Oracle and
tolerances are theirs (30 * 2^-24 holds at any position: an angle of 64 bits is off by some
2^-52 of it, 2^-21 at 2^31, which is 8 * 2^-24)."""

import numpy as np
import pytest

from test_gpu_rotary import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R", [64, 90])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_positions_past_32_bits(R, dtype):
    """Tokens behind a start near the largest number of 32 bits."""
    run(2, 80, 3, 1, 128, R, dtype, start=2 ** 31 - 60)
