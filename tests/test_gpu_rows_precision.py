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
