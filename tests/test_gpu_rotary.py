"""Norm of query and key heads with the position rotation, against the formula in float64.

Tolerances, derived. A result is a sum of two products of a normed value with a cosine or
sine of the exact angle: the norm's factor carries the roundings of the mean of squares
(log2(D) + 1 additions along the tree of sums and a few in a lane, 16 at most, halved by the
root), of the root and reciprocal (2 each), and one each for the factor and the weight; cosine and sine 2
units of 2^-24 relative to one plus the angle's own rounding (2^-24 of a turn: pi * 2^-24);
products, sum and scales 5 more. 30 * 2^-24 of |a| + |b| bounds it, plus half a step of
a 16-bit query (and half its smallest quantum).
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def freqs(R, base=10000.0):
    return (base ** (-np.arange(0, R, 2) / R)).astype(np.float32)


def oracle(x, w, eps, scale, rscale, pos, inv, interleaved):
    """x [B, H, N, D] float64, pos [B, N]: result and the bound's |a| + |b|."""
    y = x
    if w is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    R = 2 * len(inv)
    u = (pos[..., None].astype(np.float64) * inv.astype(np.float64))[:, None]
    i0 = np.arange(0, R, 2) if interleaved else np.arange(R // 2)
    i1 = i0 + 1 if interleaved else i0 + R // 2
    a, b = y[..., i0], y[..., i1]
    out, mag = y.copy(), np.abs(y)
    out[..., i0] = (a * np.cos(u) - b * np.sin(u)) * rscale
    out[..., i1] = (b * np.cos(u) + a * np.sin(u)) * rscale
    mag[..., i0] = mag[..., i1] = (np.abs(a) + np.abs(b)) * abs(rscale)
    return out * scale, mag * abs(scale)


def run(B, N, Hq, H, D, R, dtype, norm=True, interleaved=False, wdtype="float32", start=0,
        explicit=False, fused=True, offset=0, eps=1e-6, qs=0.125, rs=1.0, seed=0):
    import torch
    from flash_decode_int4 import ops
    rng = np.random.RandomState(seed + D + N)
    t = getattr(torch, dtype)
    wide = rng.randn(B, N, Hq + 2 * H, D + offset).astype(np.float32) * 3
    qkv = torch.from_numpy(wide).to(t).cuda()[..., offset:].transpose(1, 2)
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + H]
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    inv = freqs(R)
    if explicit:
        pos = rng.randint(0, max(2 * start, 50), size=(B, N))
        dev_pos = torch.from_numpy(pos.astype(np.int32)).cuda()
    else:
        first = start + rng.randint(0, 50, size=B)
        pos = first[:, None] + np.arange(N)[None]
        dev_pos = torch.from_numpy(first.astype(np.int32)).cuda()
    w = [None, None]
    if norm:
        w = [torch.from_numpy((1 + 0.2 * rng.randn(D)).astype(np.float32)).to(
            getattr(torch, wdtype)).cuda() for _ in range(2)]
    got = ops.norm_rotary(q, k, dev_pos, torch.from_numpy(inv).cuda(), w[0], w[1], eps, qs, rs,
                          interleaved)
    assert got[0].dtype == t and got[1].dtype == torch.float32
    for out, x, wt, scale, kind in ((got[0], q, w[0], qs, dtype), (got[1], k, w[1], 1.0, "float32")):
        assert out.is_contiguous() and out.shape == x.shape
        want, mag = oracle(x.double().cpu().numpy(),
                           None if wt is None else wt.double().cpu().numpy(), eps,
                           float(np.float32(scale)), float(np.float32(rs)), pos, inv, interleaved)
        tol = 30 * 2.0 ** -24 * mag + HALF[kind] * np.abs(want) * 1.001 + 2.0 ** -25 * (
            kind == "float16")
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    return got


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D,R", [(64, 64), (128, 128), (256, 256), (128, 32), (256, 64), (64, 2),
                                 (128, 90), (256, 254), (64, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_dims_and_types(D, R, dtype, interleaved):
    run(2, 3, 5, 2, D, R, dtype, interleaved=interleaved, norm=True)
    run(1, 1, 4, 1, D, R, dtype, interleaved=interleaved, norm=False)


@pytest.mark.parametrize("B,N,Hq,H", [(1, 1, 1, 1), (3, 1, 32, 8), (1, 257, 4, 4), (5, 33, 7, 7),
                                      (2, 64, 71, 1), (40, 2, 9, 3)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_shapes(B, N, Hq, H, dtype):
    run(B, N, Hq, H, 128, 128, dtype)


@pytest.mark.parametrize("kw", [dict(wdtype="bfloat16"), dict(wdtype="float16"),
                                dict(explicit=True), dict(explicit=True, start=1000000),
                                dict(fused=False), dict(offset=1), dict(offset=3, norm=False),
                                dict(eps=0.5), dict(rs=1.7), dict(start=1000000),
                                dict(start=2 ** 31 - 200), dict(qs=-3.0)], ids=str)
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_options(kw, dtype):
    run(2, 19, 6, 2, 128, 64, dtype, **kw)
    run(2, 1, 6, 2, 64, 64, dtype, interleaved=True, **kw)


def test_one_weight_and_zero_rows():
    import torch
    from flash_decode_int4 import ops
    q = torch.zeros(1, 2, 3, 64, device="cuda")
    k = torch.randn(1, 1, 3, 64, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    inv = torch.from_numpy(freqs(64)).cuda()
    w = torch.ones(64, device="cuda")
    a, b = ops.norm_rotary(q, k, pos, inv, q_weight=w)
    assert not a.any()
    _, raw = ops.norm_rotary(q, k, pos, inv)
    assert torch.equal(b, raw) and torch.equal(b[:, :, 0], k[:, :, 0])
    _, normed = ops.norm_rotary(q, k, pos, inv, k_weight=w)
    assert not torch.equal(normed, raw)


def test_a_row_that_is_not_finite_keeps_to_itself():
    import torch
    from flash_decode_int4 import ops
    q = torch.randn(1, 5, 4, 128, device="cuda").bfloat16()
    k = torch.randn(1, 3, 4, 128, device="cuda").bfloat16()
    pos = torch.tensor([7], dtype=torch.int32, device="cuda")
    inv = torch.from_numpy(freqs(128)).cuda()
    w = torch.ones(128, device="cuda")
    want = ops.norm_rotary(q, k, pos, inv, w, w)
    q[0, 2, 1, 5], k[0, 1, 3, 100] = float("nan"), float("inf")
    got = ops.norm_rotary(q, k, pos, inv, w, w)
    assert torch.isnan(got[0][0, 2, 1]).all() and torch.isnan(got[1][0, 1, 3]).any()
    got[0][0, 2, 1], got[1][0, 1, 3] = want[0][0, 2, 1], want[1][0, 1, 3]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_streams_and_a_graph():
    import torch
    from flash_decode_int4 import ops
    q = torch.randn(4, 8, 9, 128, device="cuda").bfloat16()
    k = torch.randn(4, 2, 9, 128, device="cuda").bfloat16()
    pos = torch.tensor([0, 5, 100, 7000], dtype=torch.int32, device="cuda")
    inv = torch.from_numpy(freqs(128)).cuda()
    w = torch.rand(128, device="cuda")

    def call():
        return ops.norm_rotary(q, k, pos, inv, w, w, q_scale=0.1)

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(3):
        pos.add_(9)
        graph.replay()
        now = [x.clone() for x in out]
        torch.cuda.synchronize()
        ref = call()
        assert torch.equal(now[0], ref[0]) and torch.equal(now[1], ref[1])


def test_refused():
    import torch
    from flash_decode_int4 import ops
    q = torch.zeros(2, 4, 3, 64, device="cuda")
    k = torch.zeros(2, 2, 3, 64, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    inv = torch.ones(32, device="cuda")
    w = torch.ones(64, device="cuda")

    def bad(q=q, k=k, pos=pos, inv=inv, **kw):
        with pytest.raises(RuntimeError):
            ops.norm_rotary(q, k, pos, inv, **kw)

    bad(q=q.double(), k=k.double())
    bad(k=k.half())
    bad(k=k[:1])
    bad(k=k[:, :, :2])
    bad(k=k.cpu())
    bad(q=q[..., :32], k=k[..., :32])
    bad(q=q.transpose(2, 3))
    bad(q=q[0], k=k[0])
    bad(pos=pos.long())
    bad(pos=pos[:1])
    bad(pos=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    bad(pos=torch.zeros(2, 1, dtype=torch.int32, device="cuda").expand(2, 3))
    bad(inv=inv.double())
    bad(inv=torch.ones(33, device="cuda"))
    bad(inv=inv[:0])
    bad(inv=inv[::2])
    bad(q_weight=w[:32])
    bad(q_weight=w, k_weight=w.half())
    bad(k_weight=w.cpu())
    bad(eps=-1.0)
    bad(eps=float("nan"))
    e = ops.norm_rotary(q[:0], k[:0], pos[:0], inv)
    assert tuple(e[0].shape) == (0, 4, 3, 64) and tuple(e[1].shape) == (0, 2, 3, 64)
