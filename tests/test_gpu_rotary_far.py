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


@pytest.mark.parametrize("B,N,Hq,H,D,R,kw", [
    (3, 3650, 17, 3, 128, 128, dict()),                        # two rounds, then a part of one
    (3, 3650, 17, 3, 128, 32, dict(interleaved=True, explicit=True)),
    (5, 3300, 17, 3, 128, 128, dict(wdtype="bfloat16", explicit=True)),    # all three in one
    (2, 8200, 5, 2, 256, 256, dict(interleaved=True)),         # two, the second of three heads
    (1, 11003, 32, 9, 64, 64, dict(explicit=True, start=100000)),
    (4, 2800, 4, 15, 128, 64, dict(norm=False))], ids=str)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rounds_of_heads(B, N, Hq, H, D, R, kw, dtype):
    """From 32768 rounds of 1024 channels on a wave takes several: the change from queries to
    keys within one, a last round that is not full, a last group of rounds with fewer."""
    total = -(-(Hq + H) * D // 1024)
    assert B * N * total // 16384 >= 2 and (Hq + H) * D % 1024
    run(B, N, Hq, H, D, R, dtype, **kw)
