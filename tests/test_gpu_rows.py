"""Windowed decode (sliding window and sinks) and attention of drafted trees over the
paged INT4 cache, against the definition in float64 from the stored codes and values.

Tolerances, derived: a logit is a sum of D products q*s*(nib - zp), each rounded a
fixed number of times to float32 (half a step, 2^-24 of its size): the errors of
independent roundings add as their squares, so a logit is off by about
2^-24 * 2 * A / sqrt(D), A the largest sum_d |q_d| s_d (15 + |zp_d|) of any row. An
output is an average of values with weights exp(logit), so its relative error in the
2-norm is that, plus what the probabilities are rounded to (2^-17 at least against
16-bit values where the output has 8 bits, 2^-22 otherwise) and half a step of the
output's type. Single elements are held to the worst case: 8 * 2^-24 * A (every
rounding of both the logit and the maximum at its limit) of the largest value.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _t(name):
    import torch
    return getattr(torch, name)


def make_cache(seed, B, H, D, lens, values="float32", page_rows=16, group=128, spare=3,
               max_len=None):
    """A cache in the device layout with random codes; pages in random order and rows
    behind each sequence's end that hold NaN (values) and huge codes."""
    import torch
    rng = np.random.RandomState(seed)
    R = page_rows
    cols = max(1, -(-(max_len or max(max(lens), 1)) // R))
    groups = -(-cols * R // group)
    P = B * cols + spare
    table = rng.permutation(P)[:B * cols].reshape(B, cols).astype(np.int32)
    kp = rng.randint(0, 256, size=(P, H, R, D // 2)).astype(np.uint8)
    s = (0.3 * np.exp(0.4 * rng.randn(B, H, groups, D))).astype(np.float32)
    z = (7.5 + rng.randn(B, H, groups, D)).astype(np.float32)
    v = torch.from_numpy(rng.randn(P, H, R, D).astype(np.float32)).to(_t(values))
    keep = torch.zeros(P, R, dtype=torch.bool)
    for b in range(B):
        for t in range(lens[b]):
            keep[table[b, t // R], t % R] = True
    v[~keep[:, None, :].expand(P, H, R)] = float("nan")
    return dict(kp=kp, s=s, z=z, v=v, table=table, lens=np.asarray(lens, np.int32), group=group,
                B=B, H=H, D=D, R=R)


def device_args(c):
    import torch
    return (torch.from_numpy(c["kp"]).cuda(), c["v"].cuda(), torch.from_numpy(c["s"]).cuda(),
            torch.from_numpy(c["z"]).cuda(), torch.from_numpy(c["table"]).cuda(),
            torch.from_numpy(c["lens"]).cuda())


def dense64(c, b):
    """float64 keys and values [H, n, D] of sequence b, and zp-scaled magnitudes."""
    n, R, G = int(c["lens"][b]), c["R"], c["group"]
    t = np.arange(n)
    raw = c["kp"][c["table"][b, t // R], :, t % R].transpose(1, 0, 2)      # [H, n, D/2]
    q = np.empty((c["H"], n, c["D"]))
    q[..., 0::2], q[..., 1::2] = raw & 15, raw >> 4
    s, z = c["s"][b].astype(np.float64)[:, t // G], c["z"][b].astype(np.float64)[:, t // G]
    v = c["v"].double().numpy()[c["table"][b, t // R], :, t % R].transpose(1, 0, 2)
    return (q - z) * s, v


def attend64(q, k, v, seen):
    """q [Hq, N, D], k and v [H, T, D], seen [N, T] -> [Hq, N, D]; rows of nothing: 0."""
    Hq, N, D = q.shape
    per = Hq // k.shape[0]
    out = np.zeros((Hq, N, D))
    for h in range(Hq):
        for i in range(N):
            at = np.nonzero(seen[i])[0]
            if not len(at):
                continue
            x = k[h // per][at] @ q[h, i]
            p = np.exp(x - x.max())
            out[h, i] = (p @ v[h // per][at]) / p.sum()
    return out


def visible(n, mine, window, sinks):
    t = np.arange(n)
    if not window:
        return np.ones((len(mine), n), bool)
    return (t[None] < sinks) | (t[None] >= n + np.asarray(mine)[:, None] - window)


def check(out, want, c, q, kd=None, query="float32", values="float32"):
    assert np.isfinite(out).all()
    bound = 15 + np.abs(c["z"]).max(axis=(0, 1, 2))
    A = float((np.abs(q).reshape(-1, c["D"]) @ (c["s"].max(axis=(0, 1, 2)) * bound)).max())
    if kd is not None and kd.size:
        A = max(A, float((np.abs(q).reshape(-1, c["D"])
                          @ np.abs(kd).reshape(-1, c["D"]).max(0)).max()))
    p = 2.0 ** -17 if query == "bfloat16" and values == "bfloat16" else 2.0 ** -22
    half = EPS[query]
    norm = np.linalg.norm(want)
    err = np.abs(out - want)
    if norm:
        rel = np.linalg.norm(err) / norm
        assert rel <= 2.0 ** -23 * A / np.sqrt(c["D"]) + p + half, rel
    vmax = max(1.0, np.abs(want).max())
    # (Values up to 5 standard deviations are averaged.)
    assert err.max() <= 8 * 2.0 ** -24 * A * 5 + 5 * p + half * vmax, err.max()


def queries(rng, shape, D, dtype):
    import torch
    q = torch.from_numpy((rng.randn(*shape) * 2 / np.sqrt(D)).astype(np.float32)).to(_t(dtype))
    return q.cuda(), q.double().numpy()


def tree_mask(rng, B, N):
    mask = np.zeros((B, N, N), bool)
    for b in range(B):
        for i in range(N):
            up = rng.randint(-1, i) if i else -1
            if up >= 0:
                mask[b, i] = mask[b, up]
            mask[b, i, i] = True
    return mask


# ---------------------------------------------------------------------------
# window
# ---------------------------------------------------------------------------

def run_window(c, Hq, window, sinks, query="float32", seed=0, **kw):
    from flash_decode_int4 import ops
    rng = np.random.RandomState(seed)
    q, q64 = queries(rng, (c["B"], Hq, c["D"]), c["D"], query)
    out = ops.flash_decode_paged(q, *device_args(c), c["group"], window=window, sinks=sinks, **kw)
    assert out.dtype == q.dtype and tuple(out.shape) == (c["B"], Hq, c["D"])
    want = np.stack([attend64(q64[b][:, None], *dense64(c, b),
                              visible(int(c["lens"][b]), [0], window, sinks))[:, 0]
                     for b in range(c["B"])])
    return out.double().cpu().numpy(), want, q64


@pytest.mark.parametrize("values,query", [("float32", "float32"), ("float16", "float16"),
                                          ("bfloat16", "bfloat16"), ("bfloat16", "float32"),
                                          ("float16", "bfloat16"), ("float32", "float16")])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hkv,Hq", [(2, 2), (2, 8), (1, 7)])
def test_window_types_and_heads(values, query, D, Hkv, Hq):
    c = make_cache(D + Hq, 3, Hkv, D, [700, 129, 0], values)
    out, want, q = run_window(c, Hq, 200, 5, query)
    check(out, want, c, q, query=query, values=values)
    assert not out[2].any()


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 127, 128, 129, 300, 511, 512, 513, 10000])
@pytest.mark.parametrize("sinks", [0, 1, 16, 130])
def test_window_edges(window, sinks):
    """Windows and sinks that end inside a 16-row chunk, a page and a scale group, that
    meet, and that hold everything; lengths of one and around a chunk."""
    c = make_cache(window + sinks, 6, 2, 64, [512, 511, 1, 17, 300, 128])
    out, want, q = run_window(c, 4, window, sinks)
    check(out, want, c, q)


@pytest.mark.parametrize("page_rows,group", [(1, 64), (2, 64), (8, 128), (16, 64), (16, 256),
                                             (32, 128), (64, 64), (128, 128), (256, 256)])
@pytest.mark.parametrize("D", [64, 256])
def test_window_pages_and_groups(page_rows, group, D):
    c = make_cache(page_rows + group, 3, 2, D, [777, 260, 63], "float16", page_rows, group)
    for window, sinks in ((100, 3), (400, 70)):
        out, want, q = run_window(c, 6, window, sinks, "float16")
        check(out, want, c, q, query="float16", values="float16")


def test_window_pages_that_no_group_holds_evenly():
    """page_rows that is not a power of two: groups of three 24-row pages."""
    c = make_cache(5, 2, 2, 128, [500, 73], "bfloat16", 24, 72)
    out, want, q = run_window(c, 8, 90, 30, "bfloat16")
    check(out, want, c, q, query="bfloat16", values="bfloat16")


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
def test_window_explicit_splits(splits):
    c = make_cache(11, 2, 2, 128, [3000, 1000])
    out, want, q = run_window(c, 4, 1500, 200, num_splits=splits)
    check(out, want, c, q)


def test_window_of_everything_equals_the_decode():
    from flash_decode_int4 import ops
    c = make_cache(3, 3, 2, 128, [900, 33, 256], "bfloat16")
    q, q64 = queries(np.random.RandomState(1), (3, 8, 128), 128, "float32")
    a = device_args(c)
    full = ops.flash_decode_paged(q, *a).double().cpu().numpy()
    out = ops.flash_decode_paged(q, *a, window=900).double().cpu().numpy()
    check(out, full, c, q64, values="bfloat16")


def test_window_reads_no_page_outside_it():
    """NaN values and scales everywhere outside the window and the sinks' groups."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(21, 2, 2, 64, [1000, 900], "float32", 16, 128)
    window, sinks = 140, 20
    out0, want, q64 = run_window(c, 4, window, sinks)
    for b in range(2):
        n = int(c["lens"][b])
        for t in range(n):
            if sinks <= t < n - window:
                c["v"][c["table"][b, t // 16], :, t % 16] = float("inf")
        for g in range(c["s"].shape[2]):
            if g * 128 >= sinks and (g + 1) * 128 <= n - window:
                c["s"][b, :, g] = np.nan
    q = torch.from_numpy(q64.astype(np.float32)).cuda()
    out = ops.flash_decode_paged(q, *device_args(c), window=window, sinks=sinks)
    assert np.array_equal(out.double().cpu().numpy(), out0)


def test_window_infinite_values_and_queries_inside():
    """An infinite value in the window makes its channel infinite or NaN for the heads
    that see it, as the formula does, and touches nothing else."""
    c = make_cache(8, 1, 2, 64, [300])
    t = 250
    c["v"][c["table"][0, t // 16], 1, t % 16, 7] = float("inf")
    from flash_decode_int4 import ops
    q, q64 = queries(np.random.RandomState(2), (1, 4, 64), 64, "float32")
    out = ops.flash_decode_paged(q, *device_args(c), window=100).cpu().numpy()
    assert np.isposinf(out[0, 2:, 7]).all()
    out[0, 2:, 7] = 0
    assert np.isfinite(out).all()


def test_window_strided_views_and_other_streams():
    """Queries, pages and lengths as views of larger tensors, on a side stream."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(31, 2, 2, 128, [600, 450], "float16")
    kp, v, s, z, table, lens = device_args(c)
    q, q64 = queries(np.random.RandomState(3), (2, 8, 128), 128, "float16")
    want = ops.flash_decode_paged(q, kp, v, s, z, table, lens, window=300, sinks=4)
    big = torch.zeros(2, 16, 256, dtype=torch.float16, device="cuda")
    big[:, ::2, 64:192] = q
    v2 = torch.full((v.shape[0], 4, 20, 128), float("nan"), dtype=v.dtype, device="cuda")
    v2[:, 1:3, 2:18] = v
    k2 = torch.zeros(kp.shape[0], 2, 16, 128, dtype=torch.uint8, device="cuda")
    k2[..., 32:96] = kp
    t2 = torch.zeros(2, table.shape[1] + 9, dtype=torch.int32, device="cuda")
    t2[:, :table.shape[1]] = table
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.flash_decode_paged(big[:, ::2, 64:192], k2[..., 32:96], v2[:, 1:3, 2:18], s, z,
                                     t2, lens, window=300, sinks=4, max_pages=table.shape[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


# ---------------------------------------------------------------------------
# trees
# ---------------------------------------------------------------------------

def run_tree(c, Hq, N, mask, window=None, sinks=0, query="float32", seed=0, **kw):
    import torch
    from flash_decode_int4 import ops
    rng = np.random.RandomState(seed)
    B, H, D = c["B"], c["H"], c["D"]
    q, q64 = queries(rng, (B, Hq, N, D), D, query)
    kd = rng.randn(B, H, N, D).astype(np.float32)
    vd = torch.from_numpy(rng.randn(B, H, N, D).astype(np.float32)).to(c["v"].dtype)
    out = ops.flash_decode_paged_tree(q, torch.from_numpy(kd).cuda(), vd.cuda(),
                                      torch.from_numpy(mask).cuda(), *device_args(c), c["group"],
                                      window=window, sinks=sinks, **kw)
    assert out.dtype == q.dtype and tuple(out.shape) == (B, Hq, N, D)
    want = np.zeros((B, Hq, N, D))
    full = np.broadcast_to(mask if mask.ndim == 3 else mask[None], (B, N, N))
    for b in range(B):
        k, v = dense64(c, b)
        k = np.concatenate([k, kd[b].astype(np.float64)], 1)
        v = np.concatenate([v, vd[b].double().numpy()], 1)
        seen = visible(int(c["lens"][b]), full[b].sum(-1), window, sinks)
        want[b] = attend64(q64[b], k, v, np.concatenate([seen, full[b]], 1))
    return out.double().cpu().numpy(), want, q64, kd


@pytest.mark.parametrize("values,query", [("float32", "float32"), ("float16", "float16"),
                                          ("bfloat16", "bfloat16"), ("bfloat16", "float32"),
                                          ("float32", "bfloat16")])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hkv,Hq,N", [(2, 2, 5), (1, 4, 16), (2, 6, 11)])
def test_tree_types_and_heads(values, query, D, Hkv, Hq, N):
    c = make_cache(D + N, 3, Hkv, D, [400, 129, 0], values)
    mask = tree_mask(np.random.RandomState(N), 3, N)
    out, want, q, kd = run_tree(c, Hq, N, mask, query=query)
    check(out, want, c, q, kd, query, values)


@pytest.mark.parametrize("N", [1, 2, 3, 15, 16, 17, 31, 33, 64, 65, 100, 130])
@pytest.mark.parametrize("Hkv,Hq", [(1, 1), (1, 8)])
def test_tree_sizes(N, Hkv, Hq):
    c = make_cache(N, 2, Hkv, 64, [290, 1])
    out, want, q, kd = run_tree(c, Hq, N, tree_mask(np.random.RandomState(N), 2, N))
    check(out, want, c, q, kd)


def test_tree_of_1024_nodes():
    c = make_cache(4, 1, 1, 64, [200], "bfloat16")
    out, want, q, kd = run_tree(c, 2, 1024, np.tril(np.ones((1024, 1024), bool)),
                                query="bfloat16")
    check(out, want, c, q, kd, "bfloat16", "bfloat16")


@pytest.mark.parametrize("window,sinks", [(20, 0), (21, 3), (64, 16), (128, 1), (333, 40),
                                          (5000, 2)])
def test_tree_in_a_window(window, sinks):
    """Every node has a window of its own, some ending inside the same 16-row chunk."""
    c = make_cache(window, 4, 2, 64, [500, 333, 12, 0], "float16")
    mask = tree_mask(np.random.RandomState(5), 4, 20)
    out, want, q, kd = run_tree(c, 4, 20, mask, window, sinks, "float16")
    check(out, want, c, q, kd, "float16", "float16")


def test_tree_masks_that_are_no_tree():
    """Nodes that see nothing, not themselves, later ones, or all; a shared mask; on an
    empty cache a row of nothing is zero."""
    rng = np.random.RandomState(7)
    for lens in ([200, 50], [0, 0]):
        c = make_cache(7, 2, 2, 64, lens, max_len=256)
        mask = rng.rand(9, 9) < 0.4
        mask[3], mask[5] = False, True
        out, want, q, kd = run_tree(c, 4, 9, mask)
        check(out, want, c, q, kd)
        if not any(lens):
            assert not out[:, :, 3].any()


@pytest.mark.parametrize("values", ["float32", "float16", "bfloat16"])
def test_tree_infinite_drafts_in_masked_places(values):
    """NaN and infinite keys and values of a draft reach only the nodes that see it."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(9, 1, 2, 128, [150], values)
    rng = np.random.RandomState(9)
    N, bad = 21, 6
    mask = tree_mask(rng, 1, N)[0]
    q, q64 = queries(rng, (1, 4, N, 128), 128, "float32")
    kd = torch.from_numpy(rng.randn(1, 2, N, 128).astype(np.float32)).cuda()
    vd = torch.from_numpy(rng.randn(1, 2, N, 128).astype(np.float32)).to(_t(values)).cuda()
    args = device_args(c)
    m = torch.from_numpy(mask).cuda()
    clean = ops.flash_decode_paged_tree(q, kd, vd, m, *args).double().cpu().numpy()
    for what in ("nan_key", "inf_value", "nan_value"):
        k2, v2 = kd.clone(), vd.clone()
        if what == "nan_key":
            k2[0, :, bad] = float("nan")
        else:
            v2[0, :, bad, 5:90] = float(what[:3])
        out = ops.flash_decode_paged_tree(q, k2, v2, m, *args).double().cpu().numpy()
        sees = mask[:, bad]
        assert sees.any() and not sees.all()
        # (Another path computes such rows; the same formula, other roundings.)
        np.testing.assert_allclose(out[:, :, ~sees], clean[:, :, ~sees], rtol=2.0 ** -12,
                                   atol=2.0 ** -14)
        if what == "nan_key":
            assert np.isnan(out[:, :, sees]).all()
        elif what == "inf_value":
            assert np.isposinf(out[:, :, sees, 5:90]).all()
            assert np.isfinite(out[:, :, sees, :5]).all()
        else:
            assert np.isnan(out[:, :, sees, 5:90]).all()


def test_tree_infinite_value_behind_one_nodes_window():
    """A cached row that only some nodes' windows hold is infinite."""
    from flash_decode_int4 import ops
    import torch
    c = make_cache(17, 1, 1, 64, [100], "bfloat16")
    N, window = 8, 30
    mask = np.tril(np.ones((N, N), bool))
    t = 100 + 4 - window          # seen by nodes of up to 4 visible drafts
    c["v"][c["table"][0, t // 16], 0, t % 16] = float("inf")
    q, _ = queries(np.random.RandomState(0), (1, 2, N, 64), 64, "float32")
    kd = torch.randn(1, 1, N, 64, device="cuda")
    vd = torch.randn(1, 1, N, 64, device="cuda").bfloat16()
    out = ops.flash_decode_paged_tree(q, kd, vd, torch.from_numpy(mask).cuda(), *device_args(c),
                                      window=window).cpu().numpy()
    assert np.isposinf(out[:, :, :4]).all() and np.isfinite(out[:, :, 4:]).all()


def test_tree_of_one_equals_append_and_decode_of_the_closed_part():
    """A single node that sees itself is the decode over the cache and one float key."""
    c = make_cache(2, 2, 2, 128, [256, 128])
    out, want, q, kd = run_tree(c, 2, 1, np.ones((1, 1), bool))
    check(out, want, c, q, kd)


def test_tree_strided_operands():
    """[batch, nodes, heads, head_dim] tensors as transposed views; a mask of a wider
    one."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(13, 2, 2, 64, [100, 77], "bfloat16")
    rng = np.random.RandomState(13)
    N = 10
    m = torch.from_numpy(tree_mask(rng, 2, N)).cuda()
    q, _ = queries(rng, (2, N, 6, 64), 64, "bfloat16")
    kd = torch.randn(2, N, 2, 64, device="cuda")
    vd = torch.randn(2, N, 2, 64, device="cuda").bfloat16()
    wide = torch.zeros(2, N + 3, N + 7, dtype=torch.bool, device="cuda")
    wide[:, :N, :N] = m
    args = device_args(c)
    want = ops.flash_decode_paged_tree(q.transpose(1, 2).contiguous(),
                                       kd.transpose(1, 2).contiguous(),
                                       vd.transpose(1, 2).contiguous(), m, *args)
    out = ops.flash_decode_paged_tree(q.transpose(1, 2), kd.transpose(1, 2), vd.transpose(1, 2),
                                      wide[:, :N, :N], *args)
    assert torch.equal(out, want)


@pytest.mark.parametrize("scale", [1.0, 12.0])
def test_tree_large_logits(scale):
    """Logits of standard deviation 3 and 36: the maximum moves late, weights vanish."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(23, 1, 2, 64, [2000], "float16")
    rng = np.random.RandomState(23)
    q64 = (rng.randn(1, 4, 6, 64) * scale * 2 / 8).astype(np.float32)
    kd = rng.randn(1, 2, 6, 64).astype(np.float32)
    vd = rng.randn(1, 2, 6, 64).astype(np.float16)
    mask = np.tril(np.ones((6, 6), bool))
    out = ops.flash_decode_paged_tree(torch.from_numpy(q64).cuda(), torch.from_numpy(kd).cuda(),
                                      torch.from_numpy(vd).cuda(), torch.from_numpy(mask).cuda(),
                                      *device_args(c)).double().cpu().numpy()
    k, v = dense64(c, 0)
    k = np.concatenate([k, kd[0].astype(np.float64)], 1)
    v = np.concatenate([v, vd[0].astype(np.float64)], 1)
    seen = np.concatenate([np.ones((6, 2000), bool), mask], 1)
    check(out, attend64(q64[0].astype(np.float64), k, v, seen)[None], c, q64, kd,
          values="float16")


def test_tree_and_window_in_a_graph():
    """Captured once, replayed over changed lengths and inputs, with eager calls in
    between; every replay equals the eager result."""
    import torch
    from flash_decode_int4 import ops
    c = make_cache(41, 2, 2, 128, [900, 700], "bfloat16")
    args = device_args(c)
    lens = args[-1]
    rng = np.random.RandomState(41)
    N = 7
    m = torch.from_numpy(tree_mask(rng, 2, N)).cuda()
    q = torch.randn(2, 8, N, 128, device="cuda").bfloat16() * 0.1
    kd = torch.randn(2, 2, N, 128, device="cuda")
    vd = torch.randn(2, 2, N, 128, device="cuda").bfloat16()

    def call():
        return (ops.flash_decode_paged_tree(q, kd, vd, m, *args, window=500, sinks=4),
                ops.flash_decode_paged(q[:, :, 0], *args, window=128, sinks=4))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        lens.copy_(torch.tensor([900 - 200 * i, 700 - 131 * i], dtype=torch.int32))
        q.normal_(0, 0.1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, call()):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

def test_refusals_of_window_and_tree():
    import torch
    from flash_decode_int4 import ops
    c = make_cache(1, 2, 2, 64, [64, 40])
    a = device_args(c)
    q = torch.randn(2, 4, 64, device="cuda")
    for kw in (dict(window=0), dict(window=-1), dict(sinks=3), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            ops.flash_decode_paged(q, *a, **kw)
    with pytest.raises(ValueError):
        ops.flash_decode_paged(q, *a[:5], None, window=4)
    with pytest.raises(ValueError):
        ops.flash_decode_paged(q, *a, window=4, page_lens=torch.zeros(2, 4, dtype=torch.int32,
                                                                      device="cuda"))
    with pytest.raises(ValueError):
        ops.flash_decode_paged(q, *a[:2], a[2][0, 0], a[3][0, 0], *a[4:], window=4)
    with pytest.raises(RuntimeError):
        ops.flash_decode_paged(q[:, :3], *a, window=4)
    with pytest.raises(RuntimeError):
        ops.flash_decode_paged(q.double(), *a, window=4)
    N = 5
    qt = torch.randn(2, 4, N, 64, device="cuda")
    kd = torch.randn(2, 2, N, 64, device="cuda")
    m = torch.ones(N, N, dtype=torch.bool, device="cuda")
    ok = ops.flash_decode_paged_tree(qt, kd, kd, m, *a)
    assert tuple(ok.shape) == (2, 4, N, 64)
    with pytest.raises(ValueError):
        ops.flash_decode_paged_tree(q, kd, kd, m, *a)
    with pytest.raises(ValueError):
        ops.flash_decode_paged_tree(qt, kd, kd, m, *a, window=N - 1)
    with pytest.raises(ValueError):
        ops.flash_decode_paged_tree(qt, kd, kd, m, *a, sinks=1)
    bad = [(qt, kd.half(), kd, m), (qt, kd, kd.half(), m), (qt, kd[:, :, :4], kd[:, :, :4], m),
           (qt, kd, kd, m[:4]), (qt, kd, kd, m.float()), (qt, kd, kd, m.cpu()),
           (qt, kd.cpu(), kd, m), (qt[..., :32], kd, kd, m), (qt[:1], kd, kd, m)]
    for args in bad:
        with pytest.raises(RuntimeError):
            ops.flash_decode_paged_tree(*args, *a)
    pad = torch.zeros(2, 2, N, 66, device="cuda")
    with pytest.raises(RuntimeError):
        ops.flash_decode_paged_tree(qt, pad[..., 1:65], kd, m, *a)    # rows off 16 bytes
    # Empty batches and heads are answered, not launched.
    assert ops.flash_decode_paged_tree(qt[:0], kd[:0], kd[:0], m, *a).numel() == 0
    assert ops.flash_decode_paged(q[:0], *a, window=3).numel() == 0
