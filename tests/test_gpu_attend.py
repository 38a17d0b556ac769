"""Attention of the last tokens of every sequence over the paged INT4 cache that holds
them (causal, window and sinks, prefix, capped and distance-biased scores), against the
definition in float64 from the stored codes and values.

Tolerances, derived. Let E bound the relative error of every weight exp(x_t); then an output
is off by at most E * sum_t p_t |v_t - out| (to first order; 1.1 for the rest), plus half
a step of its type, plus what the float32 sum of the products rounds: its T additions, 64
in a tile and the tiles', a product, the normalizing reciprocal and its product, and two
rescalings, each by up to 2^-24 of sum_t p_t |v_t| (that sum's own terms, not their
distances to out): (64 + T / 64 + 5) * 2^-24 of it. E is the error of a logit plus what the weight is rounded to:
  key terms  float32 queries: q and k as two float16 terms each, the product of the second
             ones left out: 3 * 2^-22 of each product; 16-bit queries: k as one
             float16, 2^-11 of each product
  sum        D float32 additions: D * 2^-24 of A = sum_d |q_d k_d|
  weight     one 16-bit term for 16-bit outputs (half a step of the value's type; bfloat16
             for float32 values, whose second term is left out at 2^-16), 2^-21 for
             float32 ones
  cap        2^-22 of the cap; bias: 2^-23 of it, where it is not hopeless (below 100);
             exponent: 2^-24 of 100, and 2^-22 for 2^x
  sums       of up to 64 weights and then of the tiles: (64 + T / 64) * 2^-24
In the 2-norm over all outputs independent roundings add as squares: sqrt(sum_d (q_d
k_d)^2) in the place of A for the key terms, sqrt(D) for D, and sqrt(sum_t p_t^2 (v_t -
out)^2) for the sum over keys.
"""

import numpy as np
import pytest

from test_gpu_rows import EPS, _t, dense64, device_args, make_cache

pytestmark = pytest.mark.gpu


def make_queries(rng, B, Hq, N, D, dtype, size=2.0):
    import torch
    q = rng.randn(B, Hq, N, D).astype(np.float32) * np.float32(size / np.sqrt(D))
    q = torch.from_numpy(q).to(_t(dtype))
    return q.cuda(), q.double().numpy()


def seen_by(n, cnt, N, window=None, sinks=0, prefix=0):
    """bool [N, n] and positions [N]."""
    p = n - cnt + np.arange(N)
    t = np.arange(n)[None]
    s = t <= p[:, None]
    if window:
        s &= (t < sinks) | (t > p[:, None] - window)
    s |= t < prefix
    return s & (np.arange(N) < cnt)[:, None], p


def oracle(c, q64, cnt, window=None, sinks=0, prefix=None, cap=None, slopes=None,
           query="float32", values="float32"):
    """(out, elementwise tolerance, 2-norm tolerance), float64."""
    B, Hq, N, D = q64.shape
    per = Hq // c["H"]
    out, tol = np.zeros(q64.shape), np.zeros(q64.shape)
    spread = adds = 0.0
    e2max = 0.0
    half = EPS[query]
    if query == "float32":
        hk, hp = 3 * 2.0 ** -22, 2.0 ** -21
    else:
        hk, hp = 2.0 ** -11, (EPS[values] if values != "float32" else EPS["bfloat16"])
    for b in range(B):
        n = int(c["lens"][b])
        if not n:
            continue
        k, v = dense64(c, b)
        seen, pos = seen_by(n, int(cnt[b]), N, window, sinks, 0 if prefix is None else prefix[b])
        far = np.abs(pos[:, None] - np.arange(n)[None])
        for h in range(Hq):
            kh, vh = k[h // per], v[h // per]
            for i in range(N):
                at = np.nonzero(seen[i])[0]
                if not len(at):
                    continue
                x = kh[at] @ q64[b, h, i]
                if cap:
                    x = cap * np.tanh(x / cap)
                bias = slopes[h] * far[i, at] if slopes is not None else 0.0
                x = x - bias
                p = np.exp(x - x.max())
                p /= p.sum()
                o = p @ vh[at]
                terms = np.abs(kh[at] * q64[b, h, i])
                A, A2 = terms.sum(1).max(), np.sqrt((terms ** 2).sum(1).max())
                rest = (2.0 ** -22 * (cap or 0) + 100 * (2.0 ** -23 + 2.0 ** -24) + 2.0 ** -22
                        + (64 + n / 64) * 2.0 ** -24)
                E = hk * A + D * 2.0 ** -24 * A + hp + rest
                e2max = max(e2max, hk * A2 + np.sqrt(D) * 2.0 ** -24 * A + hp + rest)
                out[b, h, i] = o
                add = (64 + n / 64 + 5) * 2.0 ** -24 * (p @ np.abs(vh[at]))
                tol[b, h, i] = half * np.abs(o) + 1.1 * E * (p @ np.abs(vh[at] - o)) + add
                spread += ((p ** 2) @ (vh[at] - o) ** 2).sum()
                adds += (add ** 2).sum()
    norm = np.linalg.norm(out) or 1.0
    return out, tol, half + e2max * np.sqrt(spread) / norm + np.sqrt(adds) / norm


def check(got, want, tol, tol2, scale=1.0):
    import torch
    got = got.double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    assert np.isfinite(got).all()
    # (A subnormal result of a 16-bit type is off by half its quantum.)
    over = np.abs(got - want) - tol - 2.0 ** -25
    assert over.max(initial=-1.0) <= 0, (over.max(), np.unravel_index(over.argmax(), over.shape))
    norm = np.linalg.norm(want)
    if norm:
        rel = np.linalg.norm(got - want) / norm
        assert rel <= tol2, (rel, tol2)


def run(c, Hq, N, cnt, query="float32", values="float32", seed=0, prefix=None, slopes=None,
        cap=None, window=None, sinks=0, **kw):
    import torch
    from flash_decode_int4 import ops
    rng = np.random.RandomState(seed + 77)
    q, q64 = make_queries(rng, c["B"], Hq, N, c["D"], query)
    dev = dict(counts=torch.tensor(cnt, dtype=torch.int32).cuda(), window=window, sinks=sinks,
               logit_cap=cap)
    if prefix is not None:
        dev["prefix_lens"] = torch.tensor(prefix, dtype=torch.int32).cuda()
    if slopes is not None:
        dev["slopes"] = torch.tensor(slopes, dtype=torch.float32).cuda()
    out = ops.flash_attend_paged(q, *device_args(c), group_rows=c["group"], **dev, **kw)
    assert out.dtype == q.dtype and tuple(out.shape) == tuple(q.shape)
    want = oracle(c, q64, cnt, window, sinks, prefix, cap,
                  None if slopes is None else np.asarray(slopes, np.float32).astype(np.float64),
                  query, values)
    check(out, *want)
    return out


LENS = [1, 64, 63, 130, 0, 300]
SLOPES8 = [2.0 ** -(h + 1) for h in range(8)]


@pytest.mark.parametrize("query,values", [("float32", "float32"), ("float32", "bfloat16"),
                                          ("float32", "float16"), ("bfloat16", "bfloat16"),
                                          ("float16", "float16"), ("bfloat16", "float32"),
                                          ("float16", "bfloat16")])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_types_and_ragged_lengths(D, query, values):
    c = make_cache(D, len(LENS), 2, D, LENS, values)
    run(c, 8, 1, [1] * 6, query, values, cap=30.0)
    run(c, 8, 5, [1, 5, 3, 5, 0, 2], query, values)
    run(c, 4, 70, [1, 64, 63, 70, 0, 9], query, values, slopes=SLOPES8[:4])


@pytest.mark.parametrize("kw", [
    dict(window=1), dict(window=40), dict(window=70, sinks=3), dict(window=5, sinks=200),
    dict(prefix=[1, 10, 63, 130, 0, 299]), dict(prefix=[0, 0, 1, 64, 5, 65], window=20, sinks=2),
    dict(cap=2.0), dict(cap=50.0, slopes=SLOPES8), dict(slopes=[0.0, -0.01] * 4),
    dict(window=2 ** 31 - 1, sinks=2 ** 31 - 1)], ids=str)
@pytest.mark.parametrize("N,per", [(1, 4), (3, 8), (41, 4), (150, 1)])
@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32")])
def test_masks_caps_and_biases(kw, N, per, types):
    c = make_cache(3, len(LENS), 8 // per, 64, LENS, types[1])
    cnt = [min(N, n) for n in LENS]
    cnt[3] = min(cnt[3], max(1, N - 2))
    run(c, 8, N, cnt, *types, seed=N, **kw)


@pytest.mark.parametrize("page_rows,group", [(1, 64), (16, 64), (32, 256), (64, 128), (8, 128),
                                             (48, 1200)])
@pytest.mark.parametrize("N", [1, 37])
def test_page_and_group_sizes(page_rows, group, N):
    lens = [517, 200]
    c = make_cache(5, 2, 2, 128, lens, "float16", page_rows=page_rows, group=group)
    if group == 1200:
        c["s"], c["z"] = c["s"][:, :, :1].copy(), c["z"][:, :, :1].copy()
    run(c, 6, N, [N, N - N // 3], "float16", "float16", seed=1)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
@pytest.mark.parametrize("N", [1, 20, 130])
def test_splits(splits, N):
    lens = [700, 65, 1]
    c = make_cache(6, 3, 1, 128, lens, "bfloat16")
    cnt = [min(N, n) for n in lens]
    run(c, 4, N, cnt, "bfloat16", "bfloat16", num_splits=splits, cap=50.0)
    run(c, 4, N, cnt, "float32", "bfloat16", num_splits=splits, window=100, sinks=1,
        prefix=[3, 0, 1])


@pytest.mark.parametrize("query,values,D,N,Hq,H", [
    ("bfloat16", "bfloat16", 128, 333, 8, 2), ("float16", "float16", 256, 300, 4, 2),
    ("float32", "float32", 64, 290, 6, 1), ("float32", "float16", 256, 140, 4, 2),
    ("float16", "float32", 128, 260, 7, 1), ("float32", "bfloat16", 128, 260, 2, 2)])
def test_chunks_of_several_tiles(query, values, D, N, Hq, H):
    lens = [900, 640]
    c = make_cache(9, 2, H, D, lens, values)
    run(c, Hq, N, [N, N - 35], query, values, seed=2, window=500, sinks=4, cap=50.0)
    run(c, Hq, N, [N - 1, N], query, values, seed=3)


@pytest.mark.parametrize("group,page_rows", [(512, 16), (1024, 16), (1024, 8), (2048, 16),
                                             (704, 16)])
@pytest.mark.parametrize("N", [1, 40])
@pytest.mark.parametrize("window,sinks", [(None, 0), (3000, 70)])
def test_groups_of_many_tiles(group, page_rows, N, window, sinks):
    """A wave takes several tiles of a group, and several groups, at whatever tile the
    window begins."""
    c = make_cache(17, 1, 1, 64, [6001, 4900], "float32", page_rows=page_rows, group=group)
    run(c, 1, N, [N, N], window=window, sinks=sinks, num_splits=1)
    run(c, 1, N, [N, N], window=window, sinks=sinks)


def test_many_heads_for_one_and_odd_groups():
    c = make_cache(10, 2, 1, 64, [333, 70], "bfloat16")
    run(c, 71, 1, [1, 1], "bfloat16", "bfloat16")
    run(c, 33, 4, [4, 2], "bfloat16", "bfloat16")
    c = make_cache(11, 1, 3, 128, [140], "float16")
    run(c, 15, 9, [9], "float16", "float16")


def test_strided_and_unaligned_queries():
    import torch
    from flash_decode_int4 import ops
    c = make_cache(12, 2, 2, 128, [200, 333], "bfloat16")
    dev = device_args(c)
    for N in (1, 3, 80):
        q = (torch.randn(2, 4, N, 128, device="cuda") * 0.2).bfloat16()
        want = ops.flash_attend_paged(q, *dev)
        for other in (q.transpose(1, 2).contiguous().transpose(1, 2),
                      torch.empty(2, 4, N, 131, device="cuda",
                                  dtype=torch.bfloat16)[..., 1:129].copy_(q),
                      q[:1].expand(2, -1, -1, -1)):
            got = ops.flash_attend_paged(other, *dev)
            ref = ops.flash_attend_paged(other.contiguous(), *dev)
            assert torch.equal(got, ref)
        assert torch.equal(ops.flash_attend_paged(q, *dev), want)


def test_counts_out_of_range_and_missing():
    import torch
    from flash_decode_int4 import ops
    c = make_cache(13, 3, 1, 64, [40, 2, 100], "float32")
    dev = device_args(c)
    q = torch.randn(3, 2, 5, 64, device="cuda") * 0.3

    def at(cnt):
        return ops.flash_attend_paged(q, *dev, counts=torch.tensor(cnt).int().cuda())

    assert torch.equal(at([5, 5, 5]), ops.flash_attend_paged(q, *dev))
    assert torch.equal(at([9, 70000, 2 ** 31 - 1]), at([5, 5, 5]))
    assert not at([-1, 0, -2 ** 31]).any()
    # Five queries of two tokens: the first three are before the sequence and see nothing.
    out = at([5, 5, 5])[1]
    assert not out[:, :3].any() and out[:, 3:].any(-1).all()
    two = ops.flash_attend_paged(q[:, :, 3:], *dev)
    assert torch.equal(out[:, 3:], two[1])
    # Prefixes past the length and below zero are clamped.
    a = ops.flash_attend_paged(q, *dev, prefix_lens=torch.tensor([2 ** 31 - 1] * 3).int().cuda())
    b = ops.flash_attend_paged(q, *dev, prefix_lens=torch.tensor([40, 2, 100]).int().cuda())
    assert torch.equal(a, b)
    a = ops.flash_attend_paged(q, *dev, prefix_lens=torch.tensor([-5] * 3).int().cuda())
    assert torch.equal(a, ops.flash_attend_paged(q, *dev))


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32"),
                                   ("float16", "float16")])
@pytest.mark.parametrize("N", [2, 40, 200])
def test_padding_queries_may_hold_anything(types, N):
    import torch
    from flash_decode_int4 import ops
    c = make_cache(14, 2, 2, 64, [250, 260], types[1])
    dev = device_args(c)
    q = (torch.randn(2, 4, N, 64, device="cuda") * 0.3).to(_t(types[0]))
    cnt = torch.tensor([N // 2, N - 1]).int().cuda()
    want = ops.flash_attend_paged(q, *dev, counts=cnt)
    bad = q.clone()
    bad[0, :, N // 2:] = float("nan")
    bad[1, :, N - 1:] = float("inf")
    got = ops.flash_attend_paged(bad, *dev, counts=cnt)
    assert torch.equal(got, want)
    assert not got[0, :, N // 2:].any() and not got[1, :, N - 1:].any()


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32"),
                                   ("float32", "float16")])
@pytest.mark.parametrize("N", [1, 20, 200])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite(types, N, bad):
    """Rows that see the value have it as the formula does, the others do not know of it."""
    c = make_cache(15, 2, 2, 128, [260, 250], types[1])
    import torch
    from flash_decode_int4 import ops
    rng = np.random.RandomState(4)
    q, q64 = make_queries(rng, 2, 4, N, 128, types[0])
    cnt = [N, N]
    want, tol, tol2 = oracle(c, q64, cnt, query=types[0], values=types[1])
    at = [260 - max(1, N // 2), 20]         # a token of the chunk; an early one
    for b, t in enumerate(at):
        c["v"][c["table"][b, t // 16], 1, t % 16, 5] = bad
    out = ops.flash_attend_paged(q, *device_args(c),
                                 counts=torch.tensor(cnt).int().cuda()).double().cpu().numpy()
    pos = np.stack([260 - N + np.arange(N), 250 - N + np.arange(N)])
    sees = pos >= np.array(at)[:, None]
    hit = np.zeros(out.shape, bool)
    for b in range(2):
        hit[b, 2:, sees[b], 5] = True
    if np.isnan(bad):
        assert np.isnan(out[hit]).all()
    else:
        # (A weight that underflows to zero times infinity is NaN.)
        assert (np.isnan(out[hit]) | (out[hit] == bad)).all()
    good = np.where(hit, 0.0, out)
    check(good, np.where(hit, 0.0, want), tol, 2 * tol2)


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32")])
@pytest.mark.parametrize("N", [1, 150])
def test_scales_and_queries_that_are_not_finite(types, N):
    import torch
    from flash_decode_int4 import ops
    c = make_cache(16, 1, 1, 64, [400], types[1])
    dev = list(device_args(c))
    q = (torch.randn(1, 2, N, 64, device="cuda") * 0.3).to(_t(types[0]))
    want = ops.flash_attend_paged(q, *dev, window=100)
    # A scale of the first group: rows whose window does not reach it are as before.
    for i, x in ((2, float("inf")), (3, float("nan"))):
        bad = list(dev)
        bad[i] = dev[i].clone()
        bad[i][0, 0, 0, 7] = x
        got = ops.flash_attend_paged(q, *bad, window=100)
        assert torch.equal(got, want)
        full = ops.flash_attend_paged(q, *bad)
        assert torch.isnan(full).all()
    # One query row of infinity: that row alone is NaN, capped or not it stays a row.
    if N > 1:
        inf = q.clone()
        inf[0, 1, 3, 9] = float("inf")
        got = ops.flash_attend_paged(inf, *dev, window=100)
        assert torch.isnan(got[0, 1, 3]).all()
        got[0, 1, 3] = want[0, 1, 3]
        assert torch.isfinite(got).all()
        norm = want.double().norm()
        assert (got.double() - want.double()).norm() <= 4 * EPS[types[0]] * norm + 1e-3 * norm * (
            types[0] != "float32") + 1e-5 * norm
        got = ops.flash_attend_paged(inf, *dev, window=100, logit_cap=5.0)
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32"),
                                   ("float16", "float16")])
@pytest.mark.parametrize("N", [1, 70])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -9, 2.0 ** 9, 2.0 ** 60])
def test_far_from_one(types, N, size):
    """Keys of the size 2^a and queries of 2^-a give the scores of keys and queries near
    one (float16 queries hold less)."""
    if types[0] == "float16" and not 2.0 ** -10 < size < 2.0 ** 10:
        size = 2.0 ** -8 if size < 1 else 2.0 ** 8
    c = make_cache(17, 2, 1, 128, [150, 200], types[1])
    import torch
    from flash_decode_int4 import ops
    q, q64 = make_queries(np.random.RandomState(1), 2, 4, N, 128, types[0], size=4.0)
    dev = list(device_args(c))
    cnt = torch.tensor([N, N]).int().cuda()
    a = ops.flash_attend_paged(q, *dev, counts=cnt)
    dev[2] = dev[2] * size
    b = ops.flash_attend_paged((q.double() / size).to(q.dtype), *dev, counts=cnt)
    want, tol, tol2 = oracle(c, q64, [N, N], query=types[0], values=types[1])
    check(a, want, tol, tol2)
    if types[0] != "float16":
        assert torch.equal(a, b)


@pytest.mark.parametrize("types", [("bfloat16", "bfloat16"), ("float32", "float32")])
@pytest.mark.parametrize("N", [1, 90])
def test_outlier_channels(types, N):
    """A few channels of keys that are a thousand times the others, and queries that are
    small there."""
    c = make_cache(18, 1, 2, 128, [300], types[1])
    c["s"][..., ::37] *= 1000.0
    import torch
    from flash_decode_int4 import ops
    q, q64 = make_queries(np.random.RandomState(2), 1, 4, N, 128, "float32")
    q64[..., ::37] /= 1000.0
    q = torch.from_numpy(q64).to(_t(types[0])).cuda()
    out = ops.flash_attend_paged(q, *device_args(c), counts=torch.tensor([N]).int().cuda())
    check(out, *oracle(c, q.double().cpu().numpy(), [N], query=types[0], values=types[1]))


def test_one_hot_and_huge_logits():
    """Scores of thousands: the row is the value of its best token."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(19, 1, 1, 64, [200], "float32")
    q = torch.randn(1, 2, 100, 64, device="cuda") * 300
    out = ops.flash_attend_paged(q, *device_args(c)).double().cpu().numpy()
    k, v = dense64(c, 0)
    for h in range(2):
        for i in range(100):
            x = k[0][:101 + i] @ q[0, h, i].double().cpu().numpy()
            p = np.exp(x - x.max())
            p /= p.sum()
            if np.sort(p)[-2] < 1e-9:
                assert np.abs(out[0, h, i] - v[0][x.argmax()]).max() <= 1e-5


@pytest.mark.parametrize("D,values,N", [(128, "float16", 1), (128, "float16", 200),
                                        (256, "float16", 150), (64, "bfloat16", 100),
                                        (128, "float32", 100), (64, "bfloat16", 1)])
def test_float16_outputs_keep_their_bits(D, values, N):
    """Two terms of keys, and of probabilities where the values' type is no float16: the
    2-norm of the error is that of the output's rounding and of one rounding of the
    probabilities, each at most 2^-11 / sqrt(3) of a uniform error: 4.0e-4 as squares. (One
    term of keys alone made it 5e-4.)"""
    c = make_cache(23, 2, 2, D, [900, 700], values)
    import torch
    from flash_decode_int4 import ops
    q, q64 = make_queries(np.random.RandomState(6), 2, 4, N, D, "float16")
    cnt = [N, N]
    out = ops.flash_attend_paged(q, *device_args(c), counts=torch.tensor(cnt).int().cuda())
    want = oracle(c, q64, cnt, query="float16", values="float16")[0]
    rel = np.linalg.norm(out.double().cpu().numpy() - want) / np.linalg.norm(want)
    assert rel <= np.sqrt(2 / 3) * 2.0 ** -11, rel


def test_streams_devices_and_a_graph():
    import torch
    from flash_decode_int4 import ops
    c = make_cache(20, 3, 2, 128, [300, 250, 500], "bfloat16")
    dev = list(device_args(c))
    lens = dev[5]
    slopes = torch.tensor(SLOPES8).cuda()
    for N in (1, 7, 100):
        q = (torch.randn(3, 8, N, 128, device="cuda") * 0.2).bfloat16()
        cnt = torch.full((3,), N, dtype=torch.int32, device="cuda")

        def call():
            return ops.flash_attend_paged(q, *dev, counts=cnt, logit_cap=20.0, slopes=slopes)

        want = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [call() for _ in range(3)]
        again = call()
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got + [again])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for step in range(3):
            lens.copy_(torch.tensor([300 - 50 * step, 250 - step, 500 - 7 * step]))
            cnt.copy_(torch.tensor([N, max(N - step, 0), N]))
            graph.replay()
            got = out.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, call())
        lens.copy_(torch.tensor([300, 250, 500]))


def test_a_long_cache_past_32_bits():
    """Pages behind 4 GiB of keys and of values."""
    import torch
    from flash_decode_int4 import ops
    H, D, R, n = 8, 256, 16, 4000
    pages = 70000                     # 1.1 GB of keys, 9.2 GB of float32 values
    kp = torch.zeros(pages, H, R, D // 2, dtype=torch.uint8, device="cuda")
    v = torch.zeros(pages, H, R, D, device="cuda")
    cols = n // R
    g = torch.Generator(device="cuda").manual_seed(3)
    table = (pages - 1 - torch.randperm(cols, device="cuda", generator=g)).int().view(1, cols)
    near = torch.arange(cols, device="cuda").int().view(1, cols)
    kp[table[0].long()] = torch.randint(0, 256, (cols, H, R, D // 2), device="cuda",
                                        dtype=torch.uint8, generator=g)
    v[table[0].long()] = torch.randn(cols, H, R, D, device="cuda", generator=g)
    s = torch.full((1, H, -(-n // 128), D), 0.05, device="cuda")
    z = torch.full_like(s, 7.5)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    small = kp[table[0].long()], v[table[0].long()]
    for N in (1, 100):
        q = torch.randn(1, H, N, D, device="cuda") * 0.1
        a = ops.flash_attend_paged(q, kp, v, s, z, table, lens)
        b = ops.flash_attend_paged(q, *small, s, z, near, lens)
        assert torch.equal(a, b)


@pytest.mark.parametrize("kw", [dict(logit_cap=0.0), dict(logit_cap=-3.0),
                                dict(logit_cap=float("nan")), dict(logit_cap=float("inf")),
                                dict(window=0), dict(sinks=2), dict(window=3, sinks=-1),
                                dict(group_rows=32), dict(group_rows=100)], ids=str)
def test_refused_values(kw):
    import torch
    from flash_decode_int4 import ops
    c = make_cache(21, 1, 1, 64, [200], "float32")
    q = torch.zeros(1, 1, 2, 64, device="cuda")
    with pytest.raises(ValueError):
        ops.flash_attend_paged(q, *device_args(c), **kw)


def test_refused_tensors():
    import torch
    from flash_decode_int4 import ops
    c = make_cache(22, 2, 2, 64, [200, 100], "float32")
    dev = device_args(c)
    q = torch.zeros(2, 4, 3, 64, device="cuda")
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")

    def bad(query=q, error=RuntimeError, args=dev, **kw):
        with pytest.raises(error):
            ops.flash_attend_paged(query, *args, **kw)

    bad(query=q[:, :, 0], error=ValueError)
    bad(query=q[:, :3])
    bad(query=q[..., :32])
    bad(query=q.double())
    bad(query=q.int())
    bad(query=torch.zeros(2, 4, 64, 3, device="cuda").transpose(2, 3))
    bad(query=torch.zeros(3, 4, 3, 64, device="cuda"))
    bad(counts=i32.long())
    bad(counts=i32[:1])
    bad(counts=i32.cpu())
    bad(prefix_lens=i32.float())
    bad(prefix_lens=torch.zeros(4, dtype=torch.int32, device="cuda")[::2])
    bad(slopes=torch.zeros(3, device="cuda"))
    bad(slopes=torch.zeros(4, device="cuda").half())
    bad(slopes=torch.zeros(4))
    bad(args=dev[:5] + (i32.long(),))
    empty = ops.flash_attend_paged(q[:0], *dev)
    assert tuple(empty.shape) == (0, 4, 3, 64)
    assert tuple(ops.flash_attend_paged(q[:, :, :0], *dev).shape) == (2, 4, 0, 64)
