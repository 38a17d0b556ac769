"""Runs of tokens into the INT4 cache (chunks, accepted drafts) and back out of it: bit
for bit the grouped quantizer over the whole sequences, and its dequantization."""

import numpy as np
import pytest

from oracle import pack_int4, quantize_groups_ref

pytestmark = pytest.mark.gpu


def make(D=64, H=2, B=3, group=128, page_rows=16, values="float32", max_len=700, pages=None):
    from flash_decode_int4.vllm_integration import INT4PagedSequenceCache
    cols = -(-max_len // page_rows)
    return INT4PagedSequenceCache(pages or B * cols, H, D, B, max_len, page_rows, group, values)


def stream(rng, H, n, D):
    return rng.randn(H, n, D).astype(np.float32), rng.randn(H, n, D).astype(np.float32)


def expect(cache, streams, lens):
    """The cache holds the first lens[b] tokens of every stream."""
    import torch
    B, H, D, G, R = len(streams), cache.num_kv_heads, cache.head_dim, cache.group_rows, \
        cache.page_rows
    T = max(max(lens), 1)
    k = np.zeros((B, H, T, D), np.float32)
    for b, (kb, _) in enumerate(streams):
        k[b, :, :lens[b]] = kb[:, :lens[b]]
    q, s, z = quantize_groups_ref(k, np.asarray(lens), group_size=G)
    kp, vp = cache.k_pages.cpu().numpy(), cache.v_pages.cpu()
    sc, zc, table = cache.k_scale.cpu().numpy(), cache.k_zp.cpu().numpy(), \
        cache.page_table.cpu().numpy()
    stage = cache.k_stage.cpu().numpy()
    assert cache.seq_lens[:B].tolist() == list(lens)
    for b in range(B):
        n = lens[b]
        g = -(-n // G)
        np.testing.assert_array_equal(sc[b, :, :g], s[b, :, :g])
        np.testing.assert_array_equal(zc[b, :, :g], z[b, :, :g])
        v = torch.from_numpy(streams[b][1]).to(cache.v_pages.dtype)
        for t0 in range(0, n, R):
            m, page = min(R, n - t0), table[b, t0 // R]
            np.testing.assert_array_equal(kp[page, :, :m], pack_int4(q[b, :, t0:t0 + m]))
            assert torch.equal(vp[page, :, :m], v[:, t0:t0 + m])
        o = n // G * G
        np.testing.assert_array_equal(stage[b, :, :n - o], k[b, :, o:n])
    return q, s, z


def batch(streams, at, N):
    """Tokens at[b] .. at[b] + N - 1 of every stream (zeros past its end), [B, H, N, D]
    on the GPU."""
    import torch
    H, _, D = streams[0][0].shape
    out = np.zeros((2, len(streams), H, N, D), np.float32)
    for b, (s, a) in enumerate(zip(streams, at)):
        for i in (0, 1):
            x = s[i][:, a:a + N]
            out[i, b, :, :x.shape[1]] = x
    return tuple(torch.from_numpy(x).cuda() for x in out)


@pytest.mark.parametrize("D,group,page_rows,values", [
    (64, 128, 16, "float32"), (64, 64, 8, "bfloat16"), (128, 128, 32, "float16"),
    (128, 256, 1, "float32"), (256, 64, 64, "bfloat16"), (256, 256, 16, "float16")])
def test_extend_equals_whole_sequence_quantization(D, group, page_rows, values):
    rng = np.random.RandomState(D + group)
    B, H = 3, 2
    streams = [stream(rng, H, 1200, D) for _ in range(B)]
    cache = make(D, H, B, group, page_rows, values, max_len=1200)
    lens = [0, 0, 0]
    # Chunks and ragged counts: nothing, one token, up to a group's end, over it, over
    # several groups.
    for counts in ([5, 0, 1], [group - 5, 1, group - 1], [1, group, 2 * group + 3],
                   [0, 0, 0], [2 * group - 1, group - 2, 7]):
        N = max(max(counts), 1)
        k, v = batch(streams, lens, N)
        cache.extend(k, v, counts)
        lens = [n + c for n, c in zip(lens, counts)]
        expect(cache, streams, lens)
        assert list(cache.lengths()) == lens


def test_extend_continues_prefill_append_and_step():
    import torch
    rng = np.random.RandomState(3)
    B, H, D = 2, 2, 64
    streams = [stream(rng, H, 700, D) for _ in range(B)]
    cache = make(D, H, B, values="bfloat16")
    lens = [130, 250]
    k, v = batch(streams, [0, 0], 250)
    cache.prefill(k, v, lens)
    k, v = batch(streams, lens, 9)
    cache.extend(k, v)
    lens = [n + 9 for n in lens]
    expect(cache, streams, lens)
    k, v = batch(streams, lens, 1)
    cache.append(k[:, :, 0], v[:, :, 0])
    lens = [n + 1 for n in lens]
    cache.reserve(B, 20)
    q = torch.randn(B, 4, D, device="cuda")
    for _ in range(3):
        k, v = batch(streams, lens, 1)
        cache.step(k[:, :, 0], v[:, :, 0].bfloat16(), q, window=64, sinks=2)
        lens = [n + 1 for n in lens]
    k, v = batch(streams, lens, 17)
    cache.extend(k, v, [17, 3])
    lens = [lens[0] + 17, lens[1] + 3]
    expect(cache, streams, lens)
    cache.free(1)
    k, v = batch(streams, [lens[0], 0], 40)
    cache.extend(k, v, [2, 40])
    expect(cache, streams, [lens[0] + 2, 40])


@pytest.mark.parametrize("on_device", [False, True])
def test_extend_by_index(on_device):
    """The accepted path of a tree, the same new row for two tokens, rows in any order."""
    import torch
    rng = np.random.RandomState(11)
    B, H, D, N = 3, 2, 128, 12
    base = [stream(rng, H, 125, D) for _ in range(B)]
    drafts = [stream(rng, H, N, D) for _ in range(B)]
    cache = make(D, H, B, values="float16")
    lens = [125, 100, 0]
    k, v = batch(base, [0, 0, 0], 125)
    cache.prefill(k, v, lens)
    index = np.tile(np.arange(N), (B, 1))
    index[0, :4], index[1, :3], index[2, :12] = [0, 2, 7, 11], [5, 5, 1], rng.permutation(N)
    counts = [4, 3, 12]
    k, v = batch(drafts, [0, 0, 0], N)
    if on_device:
        cache.reserve(B, N)
        cache.extend(k, v, torch.tensor(counts, dtype=torch.int32, device="cuda"),
                     torch.from_numpy(index).int().cuda())
        cache.sync_lengths()
    else:
        cache.extend(k, v, counts, index)
    streams = [tuple(np.concatenate([base[b][i][:, :lens[b]], drafts[b][i][:, index[b, :c]]], 1)
                     for i in (0, 1)) for b, c in enumerate(counts)]
    now = [n + c for n, c in zip(lens, counts)]
    expect(cache, streams, now)
    assert list(cache.lengths()) == now


def test_extend_leaves_the_rest_alone():
    """Rows behind the sequences' ends, other sequences and other scale groups keep what
    they held; a sequence that takes nothing keeps its open group's bits."""
    import torch
    rng = np.random.RandomState(4)
    B, H, D = 3, 2, 64
    streams = [stream(rng, H, 400, D) for _ in range(B)]
    cache = make(D, H, B, max_len=400)
    k, v = batch(streams, [0] * 3, 300)
    cache.prefill(k, v, [300, 130, 77])
    cache.reserve(B, 60)
    cache.k_pages[cache.page_table[:, :].long().flatten()[::7]] |= 0
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scale, cache.k_zp,
                                  cache.k_stage, cache.page_table)]
    k, v = batch(streams, [300, 130, 77], 10)
    cache.extend(k, v, [7, 0, 0])
    table = before[5].long()
    touched = torch.zeros(cache.num_pages, 16, dtype=torch.bool, device="cuda")
    for t in range(256, 307):
        touched[table[0, t // 16], t % 16] = True
    for now, old in ((cache.k_pages, before[0]), (cache.v_pages, before[1])):
        same = (now == old).flatten(3).all(-1).all(1)
        assert same[~touched].all()
    assert torch.equal(cache.k_scale[1:], before[2][1:]) and torch.equal(cache.k_zp[1:],
                                                                         before[3][1:])
    assert torch.equal(cache.k_scale[0, :, :2], before[2][0, :, :2])
    assert torch.equal(cache.k_stage[1:], before[4][1:])
    assert torch.equal(cache.page_table, before[5])


def test_extend_that_does_not_fit_takes_nothing():
    """Device counts past the capacity, negative ones, more than there are, and corrupt
    lengths, through the raw entry point."""
    import torch
    from flash_decode_int4 import ops
    rng = np.random.RandomState(6)
    H, D = 1, 64
    cache = make(D, H, 6, max_len=256)
    streams = [stream(rng, H, 300, D) for _ in range(6)]
    k, v = batch(streams, [0] * 6, 256)
    cache.prefill(k, v, [250, 250, 250, 250, 256, 10])
    cache._grow_all((b, 256) for b in range(6))
    old = cache.seq_lens.clone()
    cache.seq_lens[3] = -7
    state = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scale, cache.k_stage)]
    k, v = batch(streams, [250] * 6, 20)
    counts = torch.tensor([7, -3, 6, 5, 1, 1000], dtype=torch.int32, device="cuda")
    nxt = torch.full((6,), -1, dtype=torch.int32, device="cuda")
    ops.extend_int4_paged(k, v, counts, cache.k_stage, cache.k_pages, cache.v_pages,
                          cache.k_scale, cache.k_zp, cache.page_table, cache.seq_lens, nxt)
    assert nxt.tolist() == [250, 250, 256, -7, 256, 30]
    for b in (0, 1, 3, 4):
        rows = cache.page_table[b].long()
        assert torch.equal(cache.k_pages[rows], state[0][rows])
        assert torch.equal(cache.v_pages[rows], state[1][rows])
        assert torch.equal(cache.k_scale[b], state[2][b])
        assert torch.equal(cache.k_stage[b], state[3][b])
    assert old.tolist()[0] == 250


def test_extend_refusals():
    import torch
    from flash_decode_int4 import ops
    cache = make(64, 2, 2, max_len=64, pages=6)
    k = torch.randn(2, 2, 8, 64, device="cuda")
    for bad in ((k[0], k[0]), (k[..., :32], k[..., :32]), (k, k[:, :, :4]),
                (k[:, :1], k[:, :1]), (torch.cat([k, k]), torch.cat([k, k]))):
        with pytest.raises(ValueError):
            cache.extend(*bad)
    with pytest.raises(TypeError):
        cache.extend(k.half(), k)
    for counts in ([1], [9, 1], [-1, 1], torch.tensor([1, 1], device="cuda")):
        with pytest.raises(ValueError):
            cache.extend(k, k, counts)
    with pytest.raises(ValueError):
        cache.extend(k, k, [2, 2], [[0, 9, 0, 0, 0, 0, 0, 0]] * 2)
    with pytest.raises(ValueError):
        cache.extend(k, k, [2, 2], [[0, 1]] * 2)
    with pytest.raises(RuntimeError):   # nothing reserved
        cache.extend(k, k, torch.tensor([1, 1], dtype=torch.int32, device="cuda"))
    assert cache.seq_lens.tolist() == [0, 0]
    big = torch.randn(2, 2, 60, 64, device="cuda")
    with pytest.raises(RuntimeError):   # out of pages
        cache.extend(big, big)
    with pytest.raises(ValueError):     # longer than a sequence may be
        cache.extend(torch.randn(2, 2, 65, 64, device="cuda"),
                     torch.randn(2, 2, 65, 64, device="cuda"), [65, 0])
    args = (cache.k_stage, cache.k_pages, cache.v_pages, cache.k_scale, cache.k_zp,
            cache.page_table)
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):   # lengths written over themselves
        ops.extend_int4_paged(k, k, n, *args, cache.seq_lens, cache.seq_lens)
    with pytest.raises(RuntimeError):
        ops.extend_int4_paged(k, k, n.long(), *args, cache.seq_lens, cache._lens_next)
    with pytest.raises(RuntimeError):
        ops.extend_int4_paged(k, k.half(), n, *args, cache.seq_lens, cache._lens_next)
    with pytest.raises(RuntimeError):
        ops.extend_int4_paged(k, k, n[:1], *args, cache.seq_lens, cache._lens_next)


# ---------------------------------------------------------------------------
# read
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("D,group,page_rows,values", [
    (64, 128, 16, "float32"), (128, 64, 8, "float16"), (256, 256, 1, "bfloat16"),
    (128, 128, 128, "bfloat16")])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_read_equals_dequantization(D, group, page_rows, values, dtype):
    import torch
    rng = np.random.RandomState(D)
    B, H = 3, 2
    streams = [stream(rng, H, 600, D) for _ in range(B)]
    lens = [600, 129, 0]
    cache = make(D, H, B, group, page_rows, values, max_len=601)
    k, v = batch(streams, [0] * 3, 600)
    cache.prefill(k, v, lens)
    q, s, z = expect(cache, streams, lens)
    dt = getattr(torch, dtype)
    kw, vw = torch.zeros(B, H, 600, D), torch.zeros(B, H, 600, D)
    for b in range(B):
        g = np.arange(lens[b]) // group
        sb, zb = s[b][:, g], z[b][:, g]
        kw[b, :, :lens[b]] = torch.from_numpy(q[b, :, :lens[b]].astype(np.float32) * sb - zb * sb)
        vw[b, :, :lens[b]] = torch.from_numpy(streams[b][1][:, :lens[b]]).to(
            cache.v_pages.dtype).float()
    kw, vw = kw.to(dt), vw.to(dt)
    for start, length in ((0, 600), (0, 1), (1, 77), (127, 2), (128, 300), (599, 1), (590, 40),
                          (600, 5), (5000, 3), (17, 0)):
        ko, vo = cache.read(B, start, length, dt)
        assert ko.dtype == vo.dtype == dt and tuple(ko.shape) == (B, H, length, D)
        ke, ve = torch.zeros(B, H, length, D, dtype=dt), torch.zeros(B, H, length, D, dtype=dt)
        m = max(0, min(600 - start, length))
        ke[:, :, :m], ve[:, :, :m] = kw[:, :, start:start + m], vw[:, :, start:start + m]
        assert torch.equal(ko.cpu(), ke) and torch.equal(vo.cpu(), ve)
    ko, vo = cache.read(B, dtype=dt)
    assert torch.equal(ko.cpu(), kw) and torch.equal(vo.cpu(), vw)
    # A start of its own for every sequence, out-of-range ones clamped to the pages.
    starts = torch.tensor([33, 128, -5], dtype=torch.int32, device="cuda")
    ko, vo = cache.read(B, starts, 50, dt)
    for b, a in enumerate([33, 128, 0]):
        assert torch.equal(ko[b].cpu(), kw[b, :, a:a + 50])
        assert torch.equal(vo[b].cpu(), vw[b, :, a:a + 50])


def test_read_refusals():
    import torch
    from flash_decode_int4 import ops
    cache = make()
    with pytest.raises(ValueError):
        cache.read(99)
    with pytest.raises(ValueError):
        cache.read(3, torch.zeros(3, dtype=torch.int32, device="cuda"))
    a = (cache.k_pages, cache.v_pages, cache.k_scale, cache.k_zp, cache.page_table,
         cache.seq_lens)
    for bad in ((-1, 4), (0, -4), (2 ** 31 - 1, 2 ** 31 - 1)):
        with pytest.raises(RuntimeError):
            ops.dequantize_int4_paged(*a, *bad)
    with pytest.raises(RuntimeError):
        ops.dequantize_int4_paged(*a, 0, 4, dtype=torch.float64)
    with pytest.raises(RuntimeError):
        ops.dequantize_int4_paged(*a, torch.zeros(3, dtype=torch.int64, device="cuda"), 4)
    assert ops.dequantize_int4_paged(*a, 0, 0)[0].numel() == 0


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def test_a_speculative_loop():
    """Prefill, then rounds of: attention of a drafted tree, its accepted path into the
    cache, a windowed step; the cache equals the accepted stream's quantization, the
    tree's outputs the attention over what read() gives back."""
    import torch
    rng = np.random.RandomState(5)
    B, H, Hq, D, N = 2, 2, 8, 64, 9
    cache = make(D, H, B, values="float32")
    streams = [list(stream(rng, H, n, D)) for n in (140, 60)]
    k = np.zeros((B, H, 140, D), np.float32)
    v = np.zeros_like(k)
    for b, s in enumerate(streams):
        k[b, :, :s[0].shape[1]], v[b, :, :s[0].shape[1]] = s
    cache.prefill(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), [140, 60])
    for r in range(6):
        n = cache.lengths()[:B]
        up = np.array([[rng.randint(-1, i) if i else -1 for i in range(N)] for _ in range(B)])
        mask = np.zeros((B, N, N), bool)
        for b in range(B):
            for i in range(N):
                if up[b, i] >= 0:
                    mask[b, i] = mask[b, up[b, i]]
                mask[b, i, i] = True
        kd, vd = (rng.randn(B, H, N, D).astype(np.float32) for _ in range(2))
        q = (rng.randn(B, Hq, N, D) * 2 / 8).astype(np.float32)
        out = cache.tree_attention(torch.from_numpy(q).cuda(), torch.from_numpy(kd).cuda(),
                                   torch.from_numpy(vd).cuda(), torch.from_numpy(mask).cuda())
        kr, vr = (t.double().cpu().numpy() for t in cache.read(B))
        leaf = [int(rng.randint(N)) for _ in range(B)]
        path = [np.nonzero(mask[b, leaf[b]])[0] for b in range(B)]
        for b in range(B):
            keys = np.concatenate([kr[b, :, :n[b]], kd[b]], 1)
            vals = np.concatenate([vr[b, :, :n[b]], vd[b]], 1)
            for h in range(Hq):
                for i in range(N):
                    at = np.concatenate([np.ones(n[b], bool), mask[b, i]])
                    x = keys[h // 4][at] @ q[b, h, i]
                    p = np.exp(x - x.max())
                    # (Logits of standard deviation 2 in float32: 1e-5 is 40 roundings
                    # of the largest, |x| about 8.)
                    np.testing.assert_allclose(out[b, h, i].cpu().numpy(),
                                               p @ vals[h // 4][at] / p.sum(), atol=4e-5)
        counts = [len(p) for p in path]
        index = np.zeros((B, N), np.int64)
        for b in range(B):
            index[b, :counts[b]] = path[b]
            streams[b] = [np.concatenate([s, d[b][:, path[b]]], 1)
                          for s, d in zip(streams[b], (kd, vd))]
        cache.extend(torch.from_numpy(kd).cuda(), torch.from_numpy(vd).cuda(), counts, index)
        kn, vn = (rng.randn(B, H, D).astype(np.float32) for _ in range(2))
        cache.reserve(B, 1)
        cache.step(torch.from_numpy(kn).cuda(), torch.from_numpy(vn).cuda(),
                   torch.from_numpy(q[:, :, 0]).cuda(), window=100, sinks=4)
        cache.sync_lengths()
        for b in range(B):
            streams[b] = [np.concatenate([s, x[b][:, None]], 1)
                          for s, x in zip(streams[b], (kn, vn))]
        expect(cache, streams, [s[0].shape[1] for s in streams])


def test_extend_with_device_counts_in_a_graph():
    """Tree attention, extend and a windowed step captured once: every replay appends
    what an eager cache appends, over scale groups' ends."""
    import torch
    rng = np.random.RandomState(8)
    B, H, D, N = 2, 2, 64, 6
    caches = [make(D, H, B) for _ in range(2)]
    k0 = torch.from_numpy(rng.randn(B, H, 120, D).astype(np.float32)).cuda()
    for c in caches:
        c.prefill(k0, k0, [120, 50])
        c.reserve(B, 100)
    kd, vd = torch.randn(B, H, N, D, device="cuda"), torch.randn(B, H, N, D, device="cuda")
    q = torch.randn(B, 4, N, D, device="cuda") * 0.2
    m = torch.ones(N, N, dtype=torch.bool, device="cuda").tril()
    counts = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    index = torch.arange(N, dtype=torch.int32, device="cuda").repeat(B, 1)
    kn, vn = torch.randn(B, H, D, device="cuda"), torch.randn(B, H, D, device="cuda")

    def body(c):
        a = c.tree_attention(q, kd, vd, m, window=64, sinks=2)
        c.extend(kd, vd, counts, index)
        return a, c.step(kn, vn, q[:, :, 0], window=64, sinks=2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(caches[0])
        body(caches[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = body(caches[0])
    for i in range(6):
        counts.copy_(torch.tensor([i, N - i], dtype=torch.int32))
        index.copy_(torch.stack([torch.randperm(N), torch.randperm(N)]).int())
        kd.normal_()
        kn.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, body(caches[1])):
            assert torch.equal(x, y)
        for name in ("k_pages", "v_pages", "k_scale", "k_zp", "seq_lens"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError):
            caches[0].extend(kd, vd, [1, 1])
        torch.zeros(1, device="cuda")
