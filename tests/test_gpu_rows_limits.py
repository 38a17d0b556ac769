"""The windowed and tree attention, the multi-token write and the read at their limits:
pools past 4 GiB, lengths out of range, values near the end of float32, calls on two
streams, graphs that share a memory pool, and refusals that leave a cache as it was."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D, R, G = 128, 16, 128


def case(seed, B=2, H=2, lens=(700, 333), values="bfloat16", N=9, Hq=8):
    """A paged cache of random codes and one set of drafts, on the GPU."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, values)
    cols = -(-max(lens) // R)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    c = dict(kp=torch.randint(0, 256, (B * cols, H, R, D // 2), device="cuda", generator=g,
                              dtype=torch.uint8),
             v=randn(B * cols, H, R, D).to(dt),
             s=0.3 * torch.exp(0.4 * randn(B, H, -(-cols * R // G), D)),
             z=7.5 + randn(B, H, -(-cols * R // G), D),
             table=torch.randperm(B * cols, device="cuda", generator=g).int().view(B, cols),
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    t = dict(q=(0.1 * randn(B, Hq, N, D)).to(dt), kd=randn(B, H, N, D), vd=randn(B, H, N, D).to(dt),
             m=torch.ones(N, N, dtype=torch.bool, device="cuda").tril())
    return c, t


def args(c):
    return c["kp"], c["v"], c["s"], c["z"], c["table"], c["lens"]


def attend(c, t):
    from flash_decode_int4 import ops
    return (ops.flash_decode_paged_tree(t["q"], t["kd"], t["vd"], t["m"], *args(c), window=400,
                                        sinks=3),
            ops.flash_decode_paged_tree(t["q"], t["kd"], t["vd"], t["m"], *args(c)),
            ops.flash_decode_paged(t["q"][:, :, 0], *args(c), window=200, sinks=20))


def test_pages_past_4_gib():
    """The same pages at the bottom of a small pool and past 2^32 bytes of keys (2^34 of
    values): attention, write and read give the same bits."""
    import gc

    import torch
    from flash_decode_int4 import ops
    c, t = case(1, values="float16")
    used, H = c["kp"].shape[0], c["kp"].shape[1]
    first = (1 << 32) // (H * R * D // 2) + 5
    big = dict(c, s=c["s"].clone(), z=c["z"].clone(),
               kp=torch.empty(first + used, H, R, D // 2, dtype=torch.uint8, device="cuda"),
               v=torch.empty(first + used, H, R, D, dtype=torch.float16, device="cuda"),
               table=c["table"] + first)
    try:
        assert big["kp"].numel() > 1 << 32 and big["v"].numel() * 2 > 1 << 34
        big["kp"][first:] = c["kp"]
        big["v"][first:] = c["v"]
        for a, b in zip(attend(c, t), attend(big, t)):
            assert torch.equal(a, b)
        # 9 tokens onto lengths 700 - 40 and 333 - 40: into open groups, one of them new.
        c["lens"] -= 40
        out = []
        for x in (c, big):
            stage = torch.zeros(2, H, G, D, device="cuda")
            nxt = torch.zeros(2, dtype=torch.int32, device="cuda")
            stage[:] = torch.arange(G, device="cuda")[None, None, :, None] * 0.01
            ops.extend_int4_paged(t["kd"], t["vd"], torch.tensor([9, 5], dtype=torch.int32,
                                                                 device="cuda"),
                                  stage, x["kp"], x["v"], x["s"], x["z"], x["table"], x["lens"],
                                  nxt, G)
            assert nxt.tolist() == [669, 298]
            out.append((x["kp"][-used:].clone(), x["v"][-used:].clone(), x["s"].clone(),
                        x["z"].clone(), stage) +
                       tuple(ops.dequantize_int4_paged(*args(x)[:5], nxt, 100, 600)))
        for a, b in zip(*out):
            assert torch.equal(a, b)
    finally:
        del big
        gc.collect()
        torch.cuda.empty_cache()


def test_lengths_out_of_range():
    """Lengths past the capacity count as the capacity, negative ones as none."""
    import torch
    from flash_decode_int4 import ops
    c, t = case(2, lens=(704, 704))
    full = attend(c, t)
    kv = ops.dequantize_int4_paged(*args(c), 650, 100)
    c["lens"].fill_(2 ** 31 - 1)
    for a, b in zip(full, attend(c, t)):
        assert torch.equal(a, b)
    for a, b in zip(kv, ops.dequantize_int4_paged(*args(c), 650, 100)):
        assert torch.equal(a, b) and a[:, :, :54].any() and not a[:, :, 54:].any()
    c["lens"].zero_()
    none = attend(c, t)
    c["lens"].fill_(-(2 ** 31))
    for a, b in zip(none, attend(c, t)):
        assert torch.equal(a, b)
    assert none[0].any() and not none[2].any()
    assert not any(x.any() for x in ops.dequantize_int4_paged(*args(c), 0, 10))


@pytest.mark.parametrize("values", ["float32", "bfloat16"])
def test_values_near_the_end_of_float32(values):
    """A draft of 3e38 whose logit passes the shift of the one before it by less than the
    slack: the sum in that shift's units is beyond float32, the answer is not."""
    import torch
    from flash_decode_int4 import ops
    c, t = case(3, B=1, H=1, lens=(16,), values=values, N=80, Hq=1)
    c["lens"].zero_()
    t["q"].zero_()
    t["q"][..., 0] = 1
    t["kd"].zero_()
    t["kd"][:, :, 64, 0] = 4.5
    t["vd"].zero_()
    t["vd"][:, :, 0] = 1
    t["vd"][:, :, 64] = 3e38
    m = torch.zeros(80, 80, dtype=torch.bool, device="cuda")
    m[:, 0] = m[:, 64] = True
    out = ops.flash_decode_paged_tree(t["q"].float(), t["kd"], t["vd"], m, *args(c), num_splits=1)
    big = t["vd"][0, 0, 64, 0].double().item()
    want = big * np.exp(4.5) / (1 + np.exp(4.5))
    # The logit, the exponential and the quotient: a few float32 roundings.
    assert (out.double() / want - 1).abs().max().item() <= 16 * 2.0 ** -24


def test_two_streams_at_once():
    import torch
    cases = [case(4, lens=(700, 333)), case(5, lens=(500, 640), Hq=16)]
    want = [attend(*x) for x in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for x, s, g in zip(cases, streams, got):
            with torch.cuda.stream(s):
                g.append(attend(*x))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for outs in g:
            assert all(torch.equal(a, b) for a, b in zip(w, outs))


def test_two_graphs_of_one_pool():
    """Two captured graphs that share a memory pool (workspaces among it), replayed in
    turn with eager calls in between."""
    import torch
    cases = [case(6), case(7, lens=(512, 100), values="float32")]
    for x in cases:
        attend(*x)
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for x in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(attend(*x))
        pool = pool or graph.pool()
        graphs.append(graph)
    for i in range(4):
        for x, graph, out in zip(cases, graphs, outs):
            x[1]["q"].normal_(0, 0.1)
            x[0]["lens"].sub_(17)
            graph.replay()
            got = [o.clone() for o in out]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, attend(*x)))


def test_a_refused_step_leaves_the_cache():
    """What a windowed step() refuses is refused before the token is appended."""
    import torch
    from flash_decode_int4.vllm_integration import INT4PagedSequenceCache
    cache = INT4PagedSequenceCache(16, 2, 64, 2, 64, 16, 64)
    k = torch.randn(2, 2, 40, 64, device="cuda")
    cache.extend(k[:, :, :30], k[:, :, :30])
    cache.reserve(2, 4)
    q = torch.randn(2, 4, 64, device="cuda")
    for bad in (q[:, :3], q[:, :0], q[:1], q[..., :32], q[0], q.double(), q.cpu(),
                torch.randn(2, 4, 128, device="cuda")[..., ::2]):
        with pytest.raises(ValueError):
            cache.step(k[:, :, 30], k[:, :, 30], bad, window=8)
    for kw in (dict(window=0), dict(window=2 ** 31), dict(window=8, sinks=-1),
               dict(window=8, sinks=2 ** 31), dict(sinks=1)):
        with pytest.raises(ValueError):
            cache.step(k[:, :, 30], k[:, :, 30], q, **kw)
    with pytest.raises(TypeError):
        cache.step(k[:, :, 30], k[:, :, 30], q, window=8.5)
    assert cache.seq_lens.tolist() == [30, 30]
    out = cache.step(k[:, :, 30], k[:, :, 30], q, window=8)
    cache.sync_lengths()
    assert cache.seq_lens.tolist() == [31, 31] and cache.lengths()[:2].tolist() == [31, 31]
    assert torch.equal(out, cache.decode(q, window=8))


def test_read_takes_any_integer():
    import torch
    from flash_decode_int4.vllm_integration import INT4PagedSequenceCache
    cache = INT4PagedSequenceCache(16, 2, 64, 2, 64, 16, 64)
    k = torch.randn(2, 2, 40, 64, device="cuda")
    cache.extend(k, k)
    for a, b in zip(cache.read(2, 7), cache.read(2, np.int64(7))):
        assert torch.equal(a, b) and a.shape[2] == 33
    with pytest.raises(TypeError):
        cache.read(2, 1.5)
    with pytest.raises(ValueError):
        cache.read(2, torch.zeros(2, dtype=torch.int32, device="cuda"))


def test_a_host_index_is_not_captured():
    """Refused before anything reaches the stream, so the capture stays valid."""
    import torch
    from flash_decode_int4.vllm_integration import INT4PagedSequenceCache
    cache = INT4PagedSequenceCache(16, 2, 64, 2, 64, 16, 64)
    k = torch.randn(2, 2, 8, 64, device="cuda")
    n = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    cache.reserve(2, 32)
    cache.extend(k, k, n)
    cache.sync_lengths()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            cache.extend(k, k, n, [[0] * 8] * 2)
        cache.extend(k, k, n)
    before = cache.seq_lens.tolist()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert cache.seq_lens.tolist() == [before[0] + 2 * (i + 1), before[1] + i + 1]


@pytest.mark.parametrize("values,query,bits", [("float16", "float16", 21),
                                               ("bfloat16", "bfloat16", 21),
                                               ("float32", "float32", 29),
                                               ("bfloat16", "float32", 29)])
def test_outlier_channels(values, query, bits):
    """One channel of large queries and another of large key scales, the worst for
    products held relative to the largest of both. Such a product is off by at most half
    a unit U = 2^-bits max|q| max s (the units are powers of two, so one bit of 22 or 30
    goes), evenly spread: over D nibbles of up to 15 a logit's error has a standard
    deviation below U sqrt(D / 12) 15; six of them and the float32 steps of the logit and
    its constant (8 half steps of A, the largest sum |q| s (15 + |zp|)) bound it, twice
    that times the largest value the output's; the rest is the rounding of the
    probabilities (2^-17 at least) and of the output."""
    import torch
    c, t = case(8, values=values, N=5)
    dt = getattr(torch, query)
    c["s"][..., 17] *= 15
    c["z"][..., 17] = 7.5
    q = t["q"].float() * 0.3
    q[..., 90] *= 30
    t["q"] = q.to(dt)
    from flash_decode_int4 import ops
    out = ops.flash_decode_paged_tree(t["q"], t["kd"], t["vd"], t["m"], *args(c))
    worst = 0.0
    for b, n in enumerate(c["lens"].tolist()):
        pages = c["table"][b].long()
        raw = c["kp"][pages].permute(1, 0, 2, 3).reshape(2, -1, D // 2)[:, :n]
        nib = torch.stack([raw & 15, raw >> 4], -1).reshape(2, n, D).double()
        g = torch.arange(n, device="cuda") // G
        k = (nib - c["z"][b].double()[:, g]) * c["s"][b].double()[:, g]
        v = c["v"][pages].permute(1, 0, 2, 3).reshape(2, -1, D)[:, :n].double()
        k = torch.cat([k, t["kd"][b].double()], 1).repeat_interleave(4, 0).contiguous()
        v = torch.cat([v, t["vd"][b].double()], 1).repeat_interleave(4, 0).contiguous()
        x = torch.stack([t["q"][b, h].double() @ k[h].t().contiguous() for h in range(8)])
        x[:, :, n:].masked_fill_(~t["m"], float("-inf"))
        want = torch.softmax(x, -1) @ v
        worst = max(worst, (out[b].double() - want).abs().max().item())
        vmax = v.abs().max().item()
    qa, s = t["q"].double().abs(), c["s"].double()
    U = 2.0 ** -bits * qa.max().item() * s.max().item()
    A = (qa @ (s * (15 + c["z"].double().abs())).amax((0, 1, 2))).max().item()
    logit = 6 * 15 * (D / 12) ** 0.5 * U + 8 * 2.0 ** -24 * A
    half = torch.finfo(dt).eps / 2
    p = 2.0 ** -17 if query == "bfloat16" else 2.0 ** -22
    assert worst <= (2 * logit + p + half) * max(vmax, 5), (worst, logit)
