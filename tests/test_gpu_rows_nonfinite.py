"""Windowed and tree attention where logits are not finite: a row whose visible logits are
all -infinity is NaN, as softmax gives it, and not the zero of a row that sees nothing; a
query that is not finite makes its own row NaN and leaves the others as they were, bit for
bit."""

import numpy as np
import pytest

from test_gpu_rows import _t, attend64, check, dense64, device_args, make_cache, visible

pytestmark = pytest.mark.gpu

INF = float("inf")


def attend(c, q, window=None, sinks=0, splits=0, kd=None, vd=None, mask=None):
    from flash_decode_int4 import ops
    if mask is None:
        return ops.flash_decode_paged(q, *device_args(c), c["group"], splits, window=window,
                                      sinks=sinks)
    return ops.flash_decode_paged_tree(q, kd, vd, mask, *device_args(c), c["group"], splits,
                                       window=window, sinks=sinks)


def drafts(c, N, seed=3):
    import torch
    g = torch.Generator().manual_seed(seed)
    shape = (c["B"], c["H"], N, c["D"])
    return (torch.randn(*shape, generator=g).cuda(),
            torch.randn(*shape, generator=g).to(c["v"].dtype).cuda())


def queries(c, Hq, N=0, query="float32", seed=4):
    import torch
    g = torch.Generator().manual_seed(seed)
    shape = (c["B"], Hq, N, c["D"]) if N else (c["B"], Hq, c["D"])
    return (0.1 * torch.randn(*shape, generator=g)).to(_t(query)).cuda()


@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("values,query", [("float32", "float32"), ("bfloat16", "bfloat16"),
                                          ("float16", "float32")])
@pytest.mark.parametrize("bad", [INF, -INF, float("nan")])
def test_a_query_that_is_not_finite(bad, values, query, splits):
    """Every key of channel 9 is positive: with an infinite query there all logits of the
    row are +infinity or all are -infinity. An empty sequence still gives zeros."""
    import torch
    c = make_cache(2, 3, 2, 64, [700, 90, 0], values, max_len=704)
    c["z"][..., 9] = -1
    q = queries(c, 4, query=query)
    want = attend(c, q, 400, 20, splits)
    q[:, 1, 9] = bad
    out = attend(c, q, 400, 20, splits)
    assert out[:2, 1].isnan().all() and not out[2].any()
    out[:2, 1] = want[:2, 1]
    assert torch.equal(out, want)


@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("nodes,Hq", [(5, 4), (13, 4), (40, 8)])
def test_a_tree_padded_with_nodes_that_are_not_finite(nodes, Hq, splits):
    """The last nodes of each sequence are padding: their queries and keys hold NaN and
    infinities, no other node sees them, and one of them sees nothing at all."""
    import torch
    c = make_cache(nodes, 2, 2, 64, [300, 0], "bfloat16")
    q = queries(c, Hq, nodes, "bfloat16")
    kd, vd = drafts(c, nodes)
    used = nodes - 3
    mask = torch.ones(2, nodes, nodes, dtype=torch.bool).tril()
    mask[:, used:] = False
    mask[:, used, used] = mask[:, used + 1, :2] = True
    mask = mask.cuda()
    want = attend(c, q, kd=kd, vd=vd, mask=mask, splits=splits)
    q[:, :, used] = INF
    q[:, :, used + 1] = float("nan")
    q[:, :, used + 2] = -INF
    kd[:, :, used] = float("nan")
    kd[:, :, used + 1:] = INF
    out = attend(c, q, kd=kd, vd=vd, mask=mask, splits=splits)
    assert torch.equal(out[:, :, :used], want[:, :, :used])
    assert out[:, :, used:used + 2].isnan().all() and out[0, :, used + 2].isnan().all()
    assert not out[1, :, used + 2].any()


@pytest.mark.parametrize("splits", [0, 1, 2, 5])
@pytest.mark.parametrize("values", ["float32", "float16", "bfloat16"])
def test_keys_of_minus_infinity(values, splits):
    """A zero-point of -infinity makes a channel's keys infinite, and with a negative query
    there every logit of the scale group -infinity: one such group weighs nothing, the
    output is that of the other keys; when all groups are so, the row is NaN."""
    import torch
    c = make_cache(6, 1, 2, 64, [640], values)
    window, sinks = 300, 10                      # groups 0 (sinks), 2, 3, 4
    q = queries(c, 4)
    q[..., 5] = -q[..., 5].abs() - 0.01
    c["z"][:, 0, 3, 5] = -INF
    out = attend(c, q, window, sinks, splits).double().cpu().numpy()
    k, v = dense64(c, 0)
    seen = visible(640, [0], window, sinks)
    seen[:, 384:512] = False
    k[0, 384:512] = 0
    want = attend64(q[0].double().cpu().numpy()[:, None], k, v, seen)[:, 0]
    finite = dict(c, z=np.where(np.isfinite(c["z"]), c["z"], 0))
    check(out[:, :2], want[None, :2], finite, q.double().cpu().numpy(), values=values)
    c["z"][:, 0, :, 5] = -INF
    out = attend(c, q, window, sinks, splits)
    assert out[:, :2].isnan().all() and out[:, 2:].isfinite().all()
    # (The groups between sinks and window are not read.)
    c["z"][:, 0, 0, 5] = 0
    out = attend(c, q, window, sinks, splits)
    assert out.isfinite().all()


@pytest.mark.parametrize("splits", [0, 1, 2])
def test_drafts_of_minus_infinity(splits):
    """Draft keys of -infinity: NaN where nothing else is seen, no weight beside others."""
    import torch
    c = make_cache(7, 2, 1, 128, [200, 0])
    N = 6
    q = queries(c, 2, N)
    q[..., 3] = q[..., 3].abs() + 0.01
    kd, vd = drafts(c, N)
    mask = torch.eye(N, dtype=torch.bool, device="cuda")
    mask[4, 3] = True
    mask[5] = False
    kd[:, :, 2, 3] = -INF
    kd[:, :, 4, 3] = -INF
    out = attend(c, q, kd=kd, vd=vd, mask=mask, splits=splits)
    assert out[0].isfinite().all()
    assert out[1, :, 2].isnan().all() and not out[1, :, 5].any()
    # (p v / p: the products of their bfloat16 terms round up to six times and leave out
    # three below 2^-24 of theirs, the sum of p and the quotient round once each.)
    assert (out[1, :, 4] / vd[1, :, 3].expand(2, -1) - 1).abs().max() <= 11 * 2.0 ** -24
    none = mask.clone()
    none[2] = False
    assert torch.equal(attend(c, q, kd=kd, vd=vd, mask=none, splits=splits)[0, :, 2],
                       out[0, :, 2])


@pytest.mark.parametrize("values,query", [("float32", "float32"), ("float16", "float32"),
                                          ("bfloat16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("D,nodes,used", [(64, 7, 3), (128, 40, 33), (256, 20, 11), (64, 150, 70)])
def test_values_of_drafts_that_no_node_sees(values, query, D, nodes, used):
    """Keys and values of padding drafts may be anything: NaN in them gives the bits that
    zeros give (a workgroup that had to go row by row would round otherwise)."""
    import torch
    c = make_cache(nodes, 2, 2, D, [300, 40], values)
    q = queries(c, 4, nodes, query)
    kd, vd = drafts(c, nodes)
    mask = torch.ones(2, nodes, nodes, dtype=torch.bool, device="cuda").tril()
    mask[:, :, used:] = False
    outs = []
    for fill in (0, float("nan"), INF):
        kd[:, :, used:] = fill
        vd[:, :, used:] = fill
        outs.append(attend(c, q, kd=kd, vd=vd, mask=mask))
    assert outs[0].isfinite().all()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("bad", [INF, float("nan")])
@pytest.mark.parametrize("values,query", [("float32", "float32"), ("bfloat16", "bfloat16"),
                                          ("float16", "float32")])
@pytest.mark.parametrize("D,splits", [(64, 0), (128, 1), (256, 3)])
def test_scales_that_are_not_finite(D, splits, values, query, bad):
    """A key scale of infinity or NaN in group 3 of one head of one sequence makes that
    head's rows NaN that see the group; other heads and sequences keep their bits, and nodes
    whose window begins behind the group their values."""
    import torch
    c = make_cache(D, 2, 2, D, [640, 600], values)
    q = queries(c, 4, query=query)
    want = attend(c, q, 300, 10, splits)
    N = 9
    qt = queries(c, 4, N, query)
    kd, vd = drafts(c, N)
    mask = torch.ones(N, N, dtype=torch.bool, device="cuda").tril()
    # Node i attends from 640 + i + 1 - 133 on: nodes 0 .. 3 see tokens of group 3 (384 ..
    # 511), the others none.
    tree = attend(c, qt, 133, 0, splits, kd, vd, mask)
    c["s"][0, 1, 3, 7] = bad
    out = attend(c, q, 300, 10, splits)
    assert out[0, 2:].isnan().all()
    assert torch.equal(out[0, :2], want[0, :2]) and torch.equal(out[1], want[1])
    out = attend(c, qt, 133, 0, splits, kd, vd, mask)
    assert out[0, 2:, :4].isnan().all()
    assert torch.equal(out[0, :2], tree[0, :2]) and torch.equal(out[1], tree[1])
    a, b = out[0, 2:, 4:].float(), tree[0, 2:, 4:].float()
    # (Row by row in float32 against the matrix cores: both within test_gpu_rows' bound of
    # the definition, 8 * 2^-24 A * 5 of single elements, and rounded once each.)
    A = (qt.abs().float().amax((0, 1, 2)) * torch.from_numpy(
        np.where(np.isfinite(c["s"]), c["s"], 0).max((0, 1, 2))
        * (15 + np.abs(c["z"]).max((0, 1, 2)))).cuda()).sum().item()
    eps = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}[query]
    p = 2.0 ** -17 if query == "bfloat16" else 2.0 ** -22
    vmax = max(1, b.abs().max().item())
    assert (a - b).abs().max() <= 2 * (8 * 2.0 ** -24 * A * 5 + 5 * p + eps * vmax)


@pytest.mark.parametrize("D,Hq", [(64, 4), (128, 16), (256, 4), (128, 4)])
@pytest.mark.parametrize("splits", [0, 1, 4])
def test_an_infinite_value_beside_a_query_that_is_not_finite(D, Hq, splits):
    """The workgroup goes row by row for the value and leaves the bad row out."""
    import torch
    c = make_cache(D, 1, 1, D, [500], "bfloat16")
    N = 5
    q = queries(c, Hq, N)
    kd, vd = drafts(c, N)
    mask = torch.ones(N, N, dtype=torch.bool, device="cuda").tril()
    q[:, 1, 2, 3] = INF
    c["v"][c["table"][0, 499 // 16], :, 499 % 16, 9] = INF
    vd[:, :, 4, 11] = -INF
    out = attend(c, q, 100, 2, splits, kd, vd, mask)
    assert out[:, 1, 2].isnan().all()
    out[:, 1, 2] = out[:, 0, 2]
    assert torch.isposinf(out[..., 9]).all() and torch.isneginf(out[:, :, 4, 11]).all()
    out[..., 9] = 0
    out[:, :, 4, 11] = 0
    assert out.isfinite().all()
