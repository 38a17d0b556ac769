"""Scores and logits under caps of every accepted size, 1e-30 to 1e30, against float64.

Tolerances, derived. y = cap * tanh(x / cap) in float32. Where the cap is large the error is
relative to y: the reciprocal of the cap, its product with x and the product with the cap
round by 2^-24 each; below 0.35 tanh is a series of eight roundings of falling weight (3 *
2^-24 in all), from there on (1 - e) / (1 + e) with e = exp(-2z) at most 1/2: e is off by
(2z e 2^-23 + 2^-23 e) <= 0.9 * 2^-23, so 1 - e >= 1/2 by 2^-22 of itself and its rounding,
and 1 + e, the reciprocal and the product by 4 * 2^-24 more. 16 * 2^-24 = 2^-20 bounds the
sum: 2^-20 |y|, whatever the cap. Up to a cap of 64 (log probabilities) or 512 (attention with
16-bit outputs) a form may be taken whose error is 2^-22 of the cap instead. A logit's error EC
is the larger of the two at such caps, the first beyond. It joins the other errors of test_gpu_logprobs.py and test_gpu_attend.py in the place
of their 2^-22 of the cap: a log probability and the entropy move by EC (and the entropy by EC
times its own size), an output by 2.2 EC max|v| at most.
"""

import numpy as np
import pytest

import test_gpu_attend as attend_test
from test_gpu_logprobs import U, make, oracle
from test_gpu_rows import dense64, device_args, make_cache

pytestmark = pytest.mark.gpu

CAPS = [1e-30, 1e-6, 0.5, 64.0, 65.0, 500.0, 600.0, 1e3, 1e4, 1e5, 1e6, 1e9, 1e20, 1e30]


def cap_error(cap, largest, quick):
    rel = 2.0 ** -20 * np.minimum(largest, cap)
    return np.maximum(rel, 2.0 ** -22 * cap) if cap <= quick else rel


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(3, 1003), (3, 40001), (300, 9001)])
@pytest.mark.parametrize("cap", CAPS)
def test_log_probabilities(cap, rows, vocab, dtype):
    import torch
    from flash_decode_int4.quality import token_logprobs
    x, tok = make((rows,), vocab, dtype, spread=4.0)
    at = float(np.float32(cap))
    lp, ent, tl, ids, m = oracle(x, tok, 5, at)
    ec = cap_error(at, x.double().abs().amax(1).cpu().numpy(), 64)
    base = (64 + 45) * U + ec + 4 * U * (m + 30)
    out = token_logprobs(x, tok, 5, logit_cap=cap)
    assert (out.top_ids.cpu().numpy() == ids).all()
    got = out.logprobs.double().cpu().numpy()
    assert (np.abs(got - lp) <= base + ec + 4 * U * np.abs(lp)).all()
    got = out.top_logprobs.double().cpu().numpy()
    assert (np.abs(got - tl) <= (base + ec)[:, None] + 4 * U * np.abs(tl)).all()
    got = out.entropy.double().cpu().numpy()
    assert (np.abs(got - ent) <= 2 * base + base * np.abs(ent) + 4 * U * np.abs(ent)).all()


@pytest.mark.parametrize("cap", [65.0, 1e30])
@pytest.mark.parametrize("rows,vocab", [(6, 5003), (300, 777)])
def test_logits_that_are_not_finite(rows, vocab, cap):
    """-infinity stays masked under a large cap, NaN and +infinity make a row NaN."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    inf = float("inf")
    x, tok = make((rows,), vocab, "float32")
    x[0, ::2] = -inf
    tok[0] = 1
    x[1, 9], x[2, 9] = inf, float("nan")
    x[3] = -inf
    out = token_logprobs(x, tok, 3, logit_cap=cap)
    odd = token_logprobs(x[:1, 1::2].contiguous(), tok[:1] * 0, 3, logit_cap=cap)
    assert abs(float(out.logprobs[0] - odd.logprobs[0])) < 1e-4
    assert abs(float(out.entropy[0] - odd.entropy[0])) < 1e-4
    assert torch.equal(out.top_ids[0], 2 * odd.top_ids[0] + 1)
    assert torch.isnan(out.logprobs[1:4]).all() and torch.isnan(out.entropy[1:4]).all()
    assert torch.isfinite(out.entropy[4:]).all()


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float16", "float16"),
                                   ("float32", "float32"), ("bfloat16", "float32")])
@pytest.mark.parametrize("D,N", [(64, 1), (128, 1), (256, 2), (64, 70), (128, 90), (256, 80)])
@pytest.mark.parametrize("cap", CAPS)
def test_attention(cap, D, N, types):
    import torch
    from flash_decode_int4 import ops
    lens, cnt = [300, 131], [N, N]
    c = make_cache(31, 2, 1, D, lens, types[1])
    q, q64 = attend_test.make_queries(np.random.RandomState(8), 2, 3, N, D, types[0], size=3.0)
    at = float(np.float32(cap))
    names = dict(query=types[0], values=types[1])
    want = attend_test.oracle(c, q64, cnt, cap=at, **names)[0]
    # (The tolerance without its term of the cap: that of the same logits uncapped, whose
    # weights differ; so every distance to an output is taken as twice the largest value.)
    far = max(np.abs(dense64(c, b)[1]).max() for b in range(2))
    most = max(np.abs(q64[b] @ dense64(c, b)[0][0].T).max() for b in range(2))
    e = 2.0 ** -11 if types[0] != "float32" else 3 * 2.0 ** -22
    terms = max(np.abs(q64[b]).max(axis=(0, 1)) @ np.abs(dense64(c, b)[0][0]).max(axis=0)
                for b in range(2))
    hp = {"float32": 2.0 ** -21, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
    hp = hp["float32"] if types[0] == "float32" else hp[
        "bfloat16" if types[1] == "float32" else types[1]]
    ec = cap_error(at, most, 0 if types[0] == "float32" else 512)
    # (A score's own error shrinks under a cap: its slope is at most 1, and its size the cap.)
    E = (min(e * terms + D * 2.0 ** -24 * terms, 2 * at) + ec + hp
         + 200 * 2.0 ** -24)
    tol = attend_test.EPS[types[0]] * np.abs(want) + 1.1 * E * 2 * far
    out = ops.flash_attend_paged(q, *device_args(c), logit_cap=cap,
                                 counts=torch.tensor(cnt).int().cuda()).double().cpu().numpy()
    assert np.isfinite(out).all()
    assert (np.abs(out - want) <= tol).all(), (np.abs(out - want) / tol).max()
    # The 2-norm: independent errors, so less than a third of the sum of the bounds; that of
    # an output that ignores its logits is of the order of the outputs themselves.
    rel = np.linalg.norm(out - want) / np.linalg.norm(want)
    assert rel <= attend_test.EPS[types[0]] + 4 * (hp + ec) + 2 * e * 3


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float16", "float16"),
                                   ("float32", "float32")])
@pytest.mark.parametrize("N", [1, 90])
def test_caps_far_above_the_logits_do_nothing(N, types):
    """cap * tanh(x / cap) of a cap of 1e9 and more is x to 2^-20: outputs as without a cap, to
    what a logit's error and one more rounding make of a weight."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(32, 2, 2, 128, [500, 260], types[1])
    q, _ = attend_test.make_queries(np.random.RandomState(9), 2, 4, N, 128, types[0], size=3.0)
    want = ops.flash_attend_paged(q, *device_args(c)).double()
    for cap in (1e9, 1e30):
        got = ops.flash_attend_paged(q, *device_args(c), logit_cap=cap).double()
        half = 2 * attend_test.EPS[types[0]] + (2 * attend_test.EPS[types[1]]
                                                if types[0] != "float32" else 0)
        assert float((got - want).norm() / want.norm()) <= half + 2.0 ** -20 * 100
