"""Attention of cached tokens with scores near the end of float32's range: finite, of unlike
size in the sequence's scale groups. The softmax of scores that far apart is one-hot, so
an output is the value of the key with the largest score of float64, exactly, where that
score leads the next by more than float32's sums of the products could be off (D additions
and the roundings of a key and a product, (D + 4) * 2^-24 of the sum of their sizes, and as much
again for a kernel of several terms). float32 values of bfloat16 outputs may be held in two
bfloat16 terms: their last bits, 2^-16 of them, may turn a rounding."""

import numpy as np
import pytest

import test_gpu_attend as attend_test
from test_gpu_rows import _t, dense64, device_args, make_cache

pytestmark = pytest.mark.gpu


def check(c, q, types, least=0.5, **kw):
    """One-hot rows of a causal call by the last N tokens; at least `least` of them lead."""
    import torch
    from flash_decode_int4 import ops
    q = q.to(_t(types[0])).cuda()
    out = ops.flash_attend_paged(q, *device_args(c), **kw)
    q64, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    B, Hq, N, D = q64.shape
    tested = 0
    for b in range(B):
        k, v = dense64(c, b)
        n = int(c["lens"][b])
        for h in range(Hq):
            for i in range(N):
                kk = k[h // (Hq // c["H"])][:n - N + i + 1]
                x = kk @ q64[b, h, i]
                size = np.abs(kk * q64[b, h, i]).sum(1).max()
                assert size < 2.0 ** 127, np.log2(size)
                two = np.sort(x)[-2:]
                if two[1] - two[0] <= 2 * (D + 4) * 2.0 ** -24 * size + 200:
                    continue
                tested += 1
                want = v[h // (Hq // c["H"])][x.argmax()]
                if types == ("bfloat16", "float32"):
                    near = np.abs(got[b, h, i] - want) <= (2.0 ** -8 + 2.0 ** -15) * np.abs(want)
                else:
                    want = torch.from_numpy(want.copy()).to(_t(types[0])).double().numpy()
                    near = got[b, h, i] == want
                assert near.all(), (b, h, i)
    assert tested >= least * B * Hq * N
    return q


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32"),
                                   ("float32", "float16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N", [1, 3, 8])
def test_products_of_queries_and_scales(N, D, types):
    """Few rows: a query times a scale from 2^112 to 2^119."""
    import torch
    c = make_cache(41, 2, 2, D, [500, 333], types[1])
    up = np.array([2.0 ** 58, 2.0 ** 55, 2.0 ** 52, 2.0 ** 57])[:c["s"].shape[2]]
    c["s"] = (c["s"] * up[None, None, :, None] * np.sqrt(64 / D)).astype(np.float32)
    rng = np.random.RandomState(N + D)
    q = torch.from_numpy((rng.randn(2, 4, N, D) * 2.0 ** 59).astype(np.float32))
    check(c, q, types)
    check(c, q, types, num_splits=3)


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32")])
def test_the_sign_of_such_scores_under_a_cap(types):
    """Capped, they are the cap or its negative: the mean of the values of positive scores."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(42, 1, 1, 64, [400], types[1])
    c["s"] *= np.float32(2.0 ** 58)
    rng = np.random.RandomState(3)
    q = torch.from_numpy((rng.randn(1, 4, 2, 64) * 2.0 ** 59).astype(np.float32))
    q = q.to(_t(types[0])).cuda()
    out = ops.flash_attend_paged(q, *device_args(c), logit_cap=30.0).double().cpu().numpy()
    k, v = dense64(c, 0)
    q64 = q.double().cpu().numpy()
    for h in range(4):
        for i in range(2):
            x = k[0][:399 + i] @ q64[0, h, i]
            p = np.exp(30 * np.tanh(x / 30) - 30)
            p /= p.sum()
            want = p @ v[0][:399 + i]
            # (Equal weights are exact; additions and the output's rounding.)
            tol = attend_test.EPS[types[0]] * np.abs(want) + 400 * 2.0 ** -24 * (
                p @ np.abs(v[0][:399 + i]))
            assert (np.abs(out[0, h, i] - want) <= tol + 1e-6).all()


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32"),
                                   ("float32", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_largest_channels_that_do_not_meet(D, types):
    """Many rows: queries of 2^68 in one channel and keys of 2^71 in another, so that the
    product of their units passes 2^120 and the scores do not."""
    import torch
    c = make_cache(43, 1, 1, D, [500], types[1])
    rng = np.random.RandomState(D)
    c["s"] *= np.float32(2.0 ** 43)
    c["s"][..., 1] = np.array([2.0 ** 68, 2.0 ** 64, 2.0 ** 66, 2.0 ** 63])[None, None]
    q = rng.randn(1, 4, 40, D) * 2.0 ** 46
    q[..., 0] = 2.0 ** 68 * np.sign(rng.randn(1, 4, 40))
    q[..., 1] = 2.0 ** 50 * rng.uniform(0.5, 1.0, size=(1, 4, 40)) * np.sign(rng.randn(1, 4, 40))
    # Zero-points of one channel, so that a group's best score is that of its best code.
    c["z"][..., 1] = [5.3, 7.1, 6.2, 8.4]
    q = torch.from_numpy(q.astype(np.float32))
    check(c, q, types, least=0.05)
    check(c, q, types, least=0.05, num_splits=3)
