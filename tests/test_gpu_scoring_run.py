"""A text fed through the cache in chunks and scored, as a serving or evaluation loop
does it: heads normed and rotated at the cache's lengths, chunks written, attended and
decoded with capped and biased scores, logits turned into log probabilities; against a
float64 model over the dequantized cache, token by token against chunks, and in graphs."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B, H, HQ, D, V = 3, 2, 8, 64, 997


def projections(seed, n, dtype="bfloat16"):
    """What a layer's projection gives for n tokens of every sequence, and an output
    projection to a vocabulary."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)
    qkv = torch.randn(B, n, HQ + 2 * H, D, device="cuda", generator=g).to(dt)
    return qkv, 0.1 * torch.randn(HQ * D, V, device="cuda", generator=g)


def setup(seed=0, max_len=400, values="bfloat16"):
    import torch
    from flash_decode_int4.vllm_integration import INT4PagedSequenceCache
    cache = INT4PagedSequenceCache(200, H, D, 4, max_len, value_dtype=values)
    g = torch.Generator(device="cuda").manual_seed(seed + 9)
    par = dict(inv=(10000.0 ** (-torch.arange(0, D, 2, device="cuda") / D)).float(),
               w=1 + 0.1 * torch.randn(D, device="cuda", generator=g),
               slopes=torch.exp2(-torch.arange(1.0, HQ + 1, device="cuda")))
    return cache, par


def split(qkv):
    x = qkv.transpose(1, 2)
    return x[:, :HQ], x[:, HQ:HQ + H], x[:, HQ + H:]


def feed(cache, par, qkv, counts=None, **kw):
    """One chunk: rotate, write, attend."""
    import torch
    q, k, v = split(qkv)
    q, k = cache.rotate(q, k, par["inv"], par["w"], par["w"], q_scale=D ** -0.5)
    cache.extend(k, v, counts)
    dev = None if counts is None else torch.as_tensor(counts).int().cuda()
    return cache.attend(q, dev, **kw)


def test_chunks_against_float64():
    """Prompts in ragged chunks; the outputs against attention over the cache as it was
    after each chunk, and the log probabilities against float64 log-softmax."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    cache, par = setup()
    lens = np.zeros(B, int)
    for step, counts in enumerate(([150, 70, 1], [33, 0, 129], [1, 1, 1])):
        n = max(counts)
        qkv, proj = projections(step, n)
        q0 = cache.seq_lens[:B].clone()
        q, k, v = split(qkv)
        qr, _ = cache.rotate(q, k, par["inv"], par["w"], par["w"], q_scale=D ** -0.5)
        out = feed(cache, par, qkv, counts, logit_cap=20.0, slopes=par["slopes"])
        lens += counts
        assert q0.cpu().tolist() == (lens - counts).tolist()
        assert cache.lengths()[:B].tolist() == lens.tolist()
        kd, vd = cache.read(B, 0, int(lens.max()))
        kd, vd, qd = kd.double().cpu().numpy(), vd.double().cpu().numpy(), qr.double().cpu().numpy()
        want = np.zeros(out.shape)
        for b in range(B):
            for i in range(counts[b]):
                p = lens[b] - counts[b] + i
                for h in range(HQ):
                    x = kd[b, h // 4, :p + 1] @ qd[b, h, i]
                    x = 20 * np.tanh(x / 20) - float(par["slopes"][h]) * (p - np.arange(p + 1))
                    w = np.exp(x - x.max())
                    want[b, h, i] = w @ vd[b, h // 4, :p + 1] / w.sum()
        got = out.double().cpu().numpy()
        # Roundings of the output, the weights (bfloat16 each) and the keys (2^-11 of their
        # products, of which a score has D): as squares, twice their sum.
        tol = 2 * (2 * 2.0 ** -8 + 2.0 ** -11 * 8)
        assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)
        logits = out.transpose(1, 2).reshape(B, n, HQ * D).float() @ proj
        tok = torch.randint(0, V, (B, n), device="cuda")
        tok[torch.arange(n, device="cuda")[None] >= torch.tensor(counts, device="cuda")[:, None]] = -1
        s = token_logprobs(logits, tok, top=3)
        ref = torch.log_softmax(logits.double(), -1)
        mine = ref.gather(2, tok.clamp(min=0)[..., None])[..., 0]
        assert (s.logprobs.double() - torch.where(tok < 0, 0.0, mine)).abs().max() < 1e-5
        assert (s.entropy.double() + (ref.exp() * ref).sum(-1)).abs().max() < 1e-5
        assert torch.equal(s.top_ids, logits.sort(dim=-1, descending=True, stable=True)
                           .indices[..., :3])


def test_single_tokens_of_a_loop():
    """step() with a cap and a bias is append() and decode() with them, and decode() is
    attend() of one query."""
    import torch
    a, par = setup()
    b, _ = setup()
    qkv, _ = projections(1, 140)
    for c in (a, b):
        feed(c, par, qkv, [140, 77, 128])
    a.reserve(B, 6)
    for step in range(6):
        qkv, _ = projections(10 + step, 1)
        kw = dict(logit_cap=15.0, slopes=par["slopes"])
        if step % 2:
            kw.update(window=50, sinks=2)
        if step == 4:
            kw.pop("slopes")
        q, k, v = split(qkv)
        q, k = a.rotate(q, k, par["inv"], par["w"], par["w"], q_scale=D ** -0.5)
        got = a.step(k[:, :, 0], v[:, :, 0].contiguous(), q[:, :, 0], **kw)
        b.append(k[:, :, 0], v[:, :, 0].contiguous())
        assert torch.equal(got, b.decode(q[:, :, 0], **kw))
        assert torch.equal(got, b.attend(q, **kw)[:, :, 0])
    a.sync_lengths()
    assert a.lengths().tolist() == b.lengths().tolist()


def test_a_chunk_is_its_tokens():
    """Queries of one chunk give what they give one by one over the cache that holds the
    chunk (the same keys: nothing is written in between), to the roundings of two ways."""
    import torch
    cache, par = setup()
    qkv, _ = projections(2, 200)
    out = feed(cache, par, qkv, [200, 150, 60], logit_cap=20.0)
    q, k, v = split(qkv)
    lens = cache.seq_lens.clone()
    cache.seq_lens[:B] = 0
    qr, _ = cache.rotate(q, k, par["inv"], par["w"], par["w"], q_scale=D ** -0.5)
    for i in (0, 59, 149):
        at = torch.tensor([i + 1, i + 1, min(i, 59) + 1], dtype=torch.int32, device="cuda")
        cache.seq_lens[:B] = at
        one = cache.attend(torch.stack([qr[b, :, int(at[b]) - 1] for b in range(B)])[:, :, None],
                           logit_cap=20.0)
        for b in range(B):
            ref = out[b, :, int(at[b]) - 1].double()
            err = (one[b, :, 0].double() - ref).norm()
            assert err <= 2 * (2 * 2.0 ** -8 + 2.0 ** -11 * 8) * ref.norm()
    cache.seq_lens.copy_(lens)


def test_a_loop_in_graphs():
    """A chunk and a step captured, replayed with the program's own work between."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    a, par = setup()
    b, _ = setup()
    for c in (a, b):
        feed(c, par, projections(3, 100)[0], [100, 60, 3])
    qkv, proj = projections(4, 9)
    one, _ = projections(5, 1)
    counts = torch.zeros(B, dtype=torch.int32, device="cuda")
    tok = torch.randint(0, V, (B, 9), device="cuda")

    def work(c):
        q, k, v = split(qkv)
        q, k = c.rotate(q, k, par["inv"], par["w"], par["w"], q_scale=D ** -0.5)
        c.extend(k, v, counts)
        chunk = c.attend(q, counts, logit_cap=20.0, slopes=par["slopes"])
        q, k, v = split(one)
        q, k = c.rotate(q, k, par["inv"], par["w"], par["w"], q_scale=D ** -0.5)
        step = c.step(k[:, :, 0], v[:, :, 0].contiguous(), q[:, :, 0], logit_cap=20.0,
                      window=70)
        score = token_logprobs(chunk.transpose(1, 2).reshape(B, 9, HQ * D).float() @ proj, tok, 4)
        return chunk, step, score.logprobs, score.entropy, score.top_ids

    for c in (a, b):
        c.reserve(B, 60)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(a)
    for r in range(4):
        counts.copy_(torch.tensor([9 - r, 2 * r, r]))
        qkv.copy_(projections(20 + r, 9)[0])
        one.copy_(projections(30 + r, 1)[0])
        graph.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        want = work(b)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(a.seq_lens, b.seq_lens) and torch.equal(a.k_scale[:B], b.k_scale[:B])


def test_refused_calls_leave_the_cache():
    import torch
    cache, par = setup()
    feed(cache, par, projections(6, 20)[0])
    cache.reserve(B, 3)
    q, k, v = split(projections(7, 1)[0])
    k, v, q = k[:, :, 0].float(), v[:, :, 0].contiguous(), q[:, :, 0]
    lens, pages = cache.seq_lens.clone(), cache.k_pages.clone()
    for kw in (dict(logit_cap=0.0), dict(logit_cap=float("nan")), dict(slopes=par["slopes"][:3]),
               dict(slopes=par["slopes"].half()), dict(slopes=[0.5] * HQ),
               dict(logit_cap=3.0, sinks=2), dict(logit_cap=3.0, window=0)):
        with pytest.raises(ValueError):
            cache.step(k, v, q, **kw)
    with pytest.raises(ValueError):
        cache.step(k, v, q[:, :3], logit_cap=3.0)
    with pytest.raises(ValueError):
        cache.rotate(*split(projections(7, 1)[0])[:2][::-1], par["inv"])
    assert torch.equal(cache.seq_lens, lens) and torch.equal(cache.k_pages, pages)
