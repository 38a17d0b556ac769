"""How many bits the attention of a few cached tokens keeps of a weight for 16-bit outputs: 16
(bfloat16 and float32 values) or 22 (float16 ones), so that an output is almost always the
rounded exact one. An output o off by d before its rounding is rounded elsewhere if it lies
within d of the middle of a step s: 2 d / s of evenly spread ones. With weights off by 2^-16
of themselves, independently, d is 2^-16 * sqrt(sum p^2 v^2) at most, which for values around 0
is about the size of o, or c times it where o is small; s is at least 2^-8 |o|: 2^-7 c of the
outputs, and with c = 3 (one output in five is that small) below 1 %; float32 values lose
2^-15 of a value by two terms besides: 2 %, and scores another 2^-16 (keys of 2^-21 and a sum
in float32 over products of up to 100): 4 % at most. Weights of 8 or 11 bits, those of the
values' type, turn a quarter."""

import numpy as np
import pytest

import test_gpu_attend as attend_test
from test_gpu_rows import _t, device_args, make_cache

pytestmark = pytest.mark.gpu


def turned(types, D, N, **kw):
    """The share of outputs that are not the rounded exact ones."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(51, 4, 2, D, [900, 700, 333, 800], types[1])
    q, q64 = attend_test.make_queries(np.random.RandomState(6), 4, 4, N, D, types[0])
    cnt = [N] * 4
    out = ops.flash_attend_paged(q, *device_args(c), counts=torch.tensor(cnt).int().cuda(),
                                 logit_cap=kw.get("cap"))
    want = attend_test.oracle(c, q64, cnt, query=types[0], values=types[1], **kw)[0]
    return float((out.cpu() != torch.from_numpy(want).to(_t(types[0]))).double().mean())


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float16", "float16"),
                                   ("bfloat16", "float32")])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N,kw", [(1, {}), (5, {}), (1, dict(cap=30.0))], ids=str)
def test_outputs_are_the_rounded_exact_ones(N, kw, D, types):
    share = turned(types, D, N, **kw)
    assert share <= 0.04, share
