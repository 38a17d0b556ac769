"""Rows read from caches whose scale groups are not the usual 128: groups larger than the
sequences (down to one group a sequence, of 2^30 rows), smaller than a workgroup's rows, and
no multiple of them; ranges that begin and end anywhere, bit for bit."""

import numpy as np
import pytest

from test_gpu_rows import device_args, make_cache

pytestmark = pytest.mark.gpu


def dense32(c, b, start, length):
    """float32 keys and the stored values of rows start .. of sequence b, zeros behind it."""
    H, D, R = c["H"], c["D"], c["R"]
    k, v = np.zeros((H, length, D), np.float32), np.zeros((H, length, D), np.float32)
    t = np.arange(start, min(start + length, int(c["lens"][b])))
    if len(t):
        raw = c["kp"][c["table"][b, t // R], :, t % R].transpose(1, 0, 2)
        q = np.empty((H, len(t), D), np.float32)
        q[..., 0::2], q[..., 1::2] = raw & 15, raw >> 4
        s, z = c["s"][b][:, t // c["group"]], c["z"][b][:, t // c["group"]]
        k[:, :len(t)] = q * s - z * s
        v[:, :len(t)] = c["v"].float().numpy()[c["table"][b, t // R], :, t % R].transpose(1, 0, 2)
    return k, v


def read(c, start, length):
    from flash_decode_int4 import ops
    k, v = ops.dequantize_int4_paged(*device_args(c), start, length, c["group"])
    return k.cpu().numpy(), v.cpu().numpy()


@pytest.mark.parametrize("page_rows,group", [(16, 1 << 30), (16, 4096), (8, 8), (1, 1), (16, 48),
                                             (24, 72), (64, 320), (16, 256)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_groups_of_any_size(D, page_rows, group):
    import torch
    c = make_cache(D + group % 97, 3, 2, D, [700, 131, 0], "float32", page_rows, group)
    for start, length in ((0, 1), (0, 700), (47, 1), (47, 2), (63, 130), (129, 500), (699, 1),
                          (700, 40), (5000, 3)):
        k, v = read(c, start, length)
        for b in range(3):
            wk, wv = dense32(c, b, start, length)
            assert np.array_equal(k[b], wk) and np.array_equal(v[b], wv), (start, length, b)
    for starts, length in (([0, 130, 5], 1), ([47, 127, 0], 33), ([255, 1, 0], 129),
                           ([1, 63, 0], 640), ([699, 130, 7], 90)):
        k, v = read(c, torch.tensor(starts, dtype=torch.int32, device="cuda"), length)
        for b in range(3):
            wk, wv = dense32(c, b, starts[b], length)
            assert np.array_equal(k[b], wk) and np.array_equal(v[b], wv), (starts, length, b)


def test_one_group_a_sequence_is_attended_and_read():
    """The cache that the attention takes is one that can be read."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(1, 2, 2, 64, [300, 40], "float16", 16, 1 << 30)
    q = torch.ones(2, 4, 64, device="cuda")
    assert ops.flash_decode_paged(q, *device_args(c), c["group"], window=50).isfinite().all()
    k, v = read(c, 10, 30)
    for b in range(2):
        wk, wv = dense32(c, b, 10, 30)
        assert np.array_equal(k[b], wk) and np.array_equal(v[b], wv)
