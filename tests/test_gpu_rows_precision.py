"""Logits of the windowed and tree attention where the queries and the key scales differ
much between channels: products of ordinary size made of a large query and a small scale,
or the other way round, and one product far larger than the others. Against float64."""

import numpy as np
import pytest

from test_gpu_rows import (attend64, check, dense64, device_args, make_cache, tree_mask, visible,
                           _t)

pytestmark = pytest.mark.gpu


def balance(c, q, r):
    """Channel 17 with r times the scale and 1/r times the query, channel 40 the other way
    round: every product of a query and a scale stays as it was."""
    c["s"][..., 17] *= r
    q[..., 17] /= r
    c["s"][..., 40] /= r
    q[..., 40] *= r


@pytest.mark.parametrize("r", [1, 100, 1000, 30000])
@pytest.mark.parametrize("values", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D,Hq,N", [(64, 4, 0), (128, 6, 0), (256, 2, 0), (128, 4, 9)])
def test_balanced_channels_to_float32(r, values, D, Hq, N):
    """The error is that of float32 products (check's bound, which the balancing leaves as
    it is: it sums products): largest query times largest scale says nothing of it."""
    import torch
    from flash_decode_int4 import ops
    rng = np.random.RandomState(D + N)
    B, H = 2, 2
    c = make_cache(D + Hq, B, H, D, [500, 131], values)
    shape = (B, Hq, N, D) if N else (B, Hq, D)
    q = (rng.randn(*shape) * 2 / np.sqrt(D)).astype(np.float32)
    balance(c, q, np.float32(r))
    qc = torch.from_numpy(q).cuda()
    if not N:
        out = ops.flash_decode_paged(qc, *device_args(c), c["group"], window=300, sinks=3)
        want = np.stack([attend64(q[b].astype(np.float64)[:, None], *dense64(c, b),
                                  visible(int(c["lens"][b]), [0], 300, 3))[:, 0]
                         for b in range(B)])
        check(out.double().cpu().numpy(), want, c, q.astype(np.float64), values=values)
        return
    mask = tree_mask(rng, B, N)
    kd = (0.1 * rng.randn(B, H, N, D)).astype(np.float32)
    kd[..., 17] *= r
    kd[..., 40] /= r
    vd = torch.from_numpy(rng.randn(B, H, N, D).astype(np.float32)).to(_t(values))
    out = ops.flash_decode_paged_tree(qc, torch.from_numpy(kd).cuda(), vd.cuda(),
                                      torch.from_numpy(mask).cuda(), *device_args(c), c["group"])
    want = np.zeros(out.shape)
    for b in range(B):
        k, v = dense64(c, b)
        seen = np.concatenate([np.ones((N, k.shape[1]), bool), mask[b]], 1)
        want[b] = attend64(q[b].astype(np.float64), np.concatenate([k, kd[b]], 1),
                           np.concatenate([v, vd[b].double().numpy()], 1), seen)
    check(out.double().cpu().numpy(), want, c, q.astype(np.float64), kd, values=values)


@pytest.mark.parametrize("r", [1, 1000])
@pytest.mark.parametrize("values,query", [("float16", "float16"), ("bfloat16", "bfloat16"),
                                          ("float32", "float16"), ("bfloat16", "float16")])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_logits_of_16_bit_outputs(r, values, query, D):
    """A window of two tokens of values +1 and -1 and nearly equal logits x and y: the output
    is tanh((x - y) / 2), a small number rounded relative to itself, so it shows the error of
    the logits that the half step of an ordinary output hides.

    That error, per logit: a product v = q*s of a channel, 2^e <= |v| < 2^(e+1), is cut to
    two float16 terms, 11 bits and 11 bits of what they leave: by up to 2^(e-21), and by a
    half, a quarter .. of that where the rest begins with zeros (so a third of the limit's
    square, times 1/2 + 1/8 + .. = 2/3, is the variance), times the nibble. A matrix product
    keeps 24 bits below its largest one (up to 2^-24 of that off each of D products, twice).
    Float32 sums round by up to 2^-24 of partial sums no larger than M: D/16 in the matrix
    products, ten at most for the constant sum of v zp (four in a thread, two and four
    levels of a tree), five on the way to the exponent. The output takes half the
    difference of two logits, and of two probabilities near 1, which bfloat16 values
    multiply rounded to 16 bits (2^-17 at most) and others to 22. All of this is
    independent: the root mean square over 256 rows stays below the standard deviation."""
    import torch
    from flash_decode_int4 import ops
    rng = np.random.RandomState(D)
    B, H, n = 32, 8, 34
    c = make_cache(D, B, H, D, [n] * B, values)
    q = (rng.randn(B, H, D) * 2 / np.sqrt(D)).astype(np.float32)
    q[..., 21] *= 16
    balance(c, q, np.float32(r))
    q = torch.from_numpy(q).to(_t(query))
    q64 = q.double().numpy()
    c["v"][c["table"][:, 2], :, 0] = 1
    c["v"][c["table"][:, 2], :, 1] = -1
    want, var = np.zeros((B, H)), 0.0
    for b in range(B):
        for h in range(H):
            # Of 300 keys the two next to each other.
            raw = rng.randint(0, 256, size=(300, D // 2)).astype(np.uint8)
            nib = np.stack([raw & 15, raw >> 4], -1).reshape(300, D).astype(np.float64)
            s, z = c["s"][b, h, 0].astype(np.float64), c["z"][b, h, 0].astype(np.float64)
            x = (nib - z) * s @ q64[b, h]
            order = np.argsort(x)
            i = np.argmin(np.diff(x[order]))
            pair = order[[i, i + 1]]
            c["kp"][c["table"][b, 2], h, :2] = raw[pair]
            want[b, h] = np.tanh((x[pair[0]] - x[pair[1]]) / 2)
            v = q64[b, h] * s
            M = max(np.abs(np.cumsum(v * w)).max() for w in (nib[pair[0]], nib[pair[1]], z))
            cut = 2.0 ** (np.floor(np.log2(np.abs(v))) - 21)
            for w in nib[pair]:
                var += (((cut * w) ** 2).sum() * 2 / 3
                        + 2 * D * (2.0 ** -24 * np.abs(v * w).max()) ** 2
                        + (D / 16 + 15) * (2.0 ** -24 * M) ** 2) / 3
    out = ops.flash_decode_paged(q.cuda(), *device_args(c), c["group"], window=2)
    assert (out == out[..., :1]).all()
    err = out[..., 0].double().cpu().numpy() - want
    rms, size = np.sqrt((err ** 2).mean()), np.sqrt((want ** 2).mean())
    var = var / (B * H) / 4
    var += (2.0 ** -17 if values == "bfloat16" else 2.0 ** -22) ** 2 / 6
    bound = np.sqrt(var) + torch.finfo(_t(query)).eps / 2 * size
    assert rms <= bound, (rms, bound, size)
