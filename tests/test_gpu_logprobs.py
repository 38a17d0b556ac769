"""Log probabilities of given tokens, entropies and alternatives, against float64.

Tolerances, derived. With d = x - m rounded once (2^-24 of |d|, and the capped logit before
it to 2^-22 of the cap), e = exp(d) is off by 2^-24 * 1.45 |d| + 2^-22 of itself. The sum of e
adds the roundings of its additions, along chains of at most 600 terms in a thread and a
tree: their mean, weighted with e, stays below (600 + 20) * 2^-24 in the worst case
and sqrt of that for independent ones; 64 * 2^-24 holds both kinds here, where the terms
are positive and unordered. So log l is off by at most (64 + 1.45 * 30) * 2^-24 (terms
with |d| > 30 weigh nothing), a log probability by that and two roundings of its own
size, and the entropy, a mean of d with weights e / l, by the same relative to its
mean |d| plus that of log l.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def make(shape, vocab, dtype, seed=0, spread=2.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + vocab)
    x = (torch.randn(*shape, vocab, device="cuda", generator=g) * spread).to(
        getattr(torch, dtype))
    tok = torch.randint(0, vocab, shape, device="cuda", generator=g)
    return x, tok


def oracle(x, tok, top, cap=None):
    raw = x.double().cpu().numpy().reshape(-1, x.shape[-1])
    t = tok.cpu().numpy().reshape(-1)
    y = raw if cap is None else cap * np.tanh(raw / cap)
    m = y.max(1, keepdims=True)
    d = y - m
    e = np.exp(d)
    l = e.sum(1)
    with np.errstate(invalid="ignore"):
        ent = np.log(l) - np.where(e > 0, e * d, 0.0).sum(1) / l
    lse = m[:, 0] + np.log(l)
    rows = np.arange(len(t))
    lp = np.where(t < 0, 0.0, y[rows, np.maximum(t, 0)] - lse)
    ids = np.argsort(-raw, axis=1, kind="stable")[:, :top]
    return lp, ent, np.take_along_axis(y, ids, 1) - lse[:, None], ids, np.abs(m[:, 0])


def check(out, x, tok, top=0, cap=None):
    lead = tuple(x.shape[:-1])
    lp, ent, tl, ids, m = oracle(x, tok, top, cap)
    base = (64 + 45) * U + 2.0 ** -22 * (cap or 0.0) + 4 * U * (m + 30)
    for got, want in ((out.logprobs, lp), (out.entropy, ent)):
        assert tuple(got.shape) == lead
        g = got.double().cpu().numpy().reshape(-1)
        tol = base + 4 * U * np.abs(want) + (base * np.abs(ent) if want is ent else 0.0)
        assert (np.abs(g - want) <= tol).all(), (np.abs(g - want) / tol).max()
    assert tuple(out.top_ids.shape) == lead + (top,)
    assert (out.top_ids.cpu().numpy().reshape(len(lp), top) == ids).all()
    g = out.top_logprobs.double().cpu().numpy().reshape(len(lp), top)
    assert (np.abs(g - tl) <= base[:, None] + 4 * U * np.abs(tl)).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4097, 32000, 50021])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_sizes(vocab, top, dtype):
    from flash_decode_int4.quality import token_logprobs
    top = min(top, vocab)
    x, tok = make((3,), vocab, dtype)
    check(token_logprobs(x, tok, top), x, tok, top)


@pytest.mark.parametrize("rows,vocab", [(1, 128000), (1, 200003), (7, 128001), (300, 9001),
                                        (1200, 777)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cap", [None, 30.0])
def test_rows_and_caps(rows, vocab, dtype, cap):
    from flash_decode_int4.quality import token_logprobs
    x, tok = make((rows,), vocab, dtype, spread=6.0)
    check(token_logprobs(x, tok, 7, logit_cap=cap), x, tok, 7, cap)
    check(token_logprobs(x, tok, 0, logit_cap=cap), x, tok, 0, cap)


def test_views_and_shapes():
    import torch
    from flash_decode_int4.quality import token_logprobs
    x, tok = make((4, 6), 515, "bfloat16")
    for view, ids in ((x[:, :-1], tok[:, 1:]), (x[1:, ::2], tok[1:, ::2]),
                      (x.transpose(0, 1), tok.transpose(0, 1)), (x[0], tok[0]),
                      (x[0, 0], tok[0, 0]), (x[:, :, 3:], tok.clamp(max=511)),
                      (x.view(2, 2, 6, 515), tok.view(2, 2, 6)),
                      (x.view(2, 2, 6, 515)[:, :, 1:], tok.view(2, 2, 6)[:, :, 1:]),
                      (x[:1].expand(4, 6, 515), tok), (x[..., ::2], tok.clamp(max=257)),
                      (x, tok.int())):
        check(token_logprobs(view, ids, 5), view, ids, 5)
    e = token_logprobs(x[:0], tok[:0], 3)
    assert tuple(e.logprobs.shape) == (0, 6) and tuple(e.top_ids.shape) == (0, 6, 3)
    assert torch.equal(token_logprobs(x, tok).logprobs, token_logprobs(x, tok, 5).logprobs)


def test_ties_go_to_the_lowest_index():
    import torch
    from flash_decode_int4.quality import token_logprobs
    x = torch.zeros(2, 5000, device="cuda")
    x[1, 100::7] = 2.0
    x[1, 4999] = 3.0
    x[0, ::2] = -0.0
    out = token_logprobs(x, torch.zeros(2, dtype=torch.long, device="cuda"), 64)
    assert out.top_ids[0].tolist() == list(range(64))
    assert out.top_ids[1].tolist() == [4999] + list(range(100, 100 + 7 * 63, 7))
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(0, 6, (50, 3001), device="cuda", generator=g).half()
    out = token_logprobs(x, torch.zeros(50, dtype=torch.long, device="cuda"), 64)
    want = x.float().sort(dim=1, descending=True, stable=True).indices[:, :64]
    assert torch.equal(out.top_ids, want)


@pytest.mark.parametrize("order", ["rising", "falling"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sorted_rows(order, dtype):
    """Every element of a rising row is a new largest one."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    x = torch.linspace(-9, 9, 70001, device="cuda").to(getattr(torch, dtype))
    x = torch.stack([x, x.flip(0)]) if order == "rising" else torch.stack([x.flip(0), x])
    tok = torch.tensor([70000, 3], device="cuda")
    check(token_logprobs(x, tok, 64), x, tok, 64)


def test_infinities_and_nan():
    import torch
    from flash_decode_int4.quality import token_logprobs
    inf, nan = float("inf"), float("nan")
    x, tok = make((8,), 3000, "float32")
    x[0, ::3] = -inf
    tok[0] = 0
    x[1, 17] = inf
    x[2, 2900] = nan
    x[3] = -inf
    x[4, 1:] = -inf
    tok[4] = 0
    x[5, 5:] = -inf
    x[6] = torch.finfo(torch.float32).min
    out = token_logprobs(x, tok, 6)
    assert out.logprobs[0] == -inf and torch.isfinite(out.entropy[0])
    for r in (1, 2, 3):
        assert torch.isnan(out.logprobs[r]) and torch.isnan(out.entropy[r])
    assert out.top_ids[1, 0] == 17 and out.top_ids[2, 0] == 2900
    assert out.top_ids[3].tolist() == list(range(6))
    assert out.logprobs[4] == 0 and out.entropy[4] == 0
    assert out.top_logprobs[4, 0] == 0 and (out.top_logprobs[4, 1:] == -inf).all()
    assert sorted(out.top_ids[5].tolist()) == list(range(6)) and out.top_ids[5, 5] == 5
    assert abs(float(out.entropy[6]) - np.log(3000)) < 1e-4
    check(type(out)(*[t[7:] for t in out]), x[7:], tok[7:], 6)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("vocab", [5, 999, 33001])
def test_small_caps_and_masked_logits(vocab, dtype):
    """Logits of -infinity stay masked under a cap that would make them count, and nothing
    behind a row does."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    x, tok = make((9,), vocab, dtype)
    check(token_logprobs(x, tok, 4, logit_cap=0.5), x, tok, 4, 0.5)
    x[:, 2::3] = -float("inf")
    tok[:] = 1
    out = token_logprobs(x, tok, 3, logit_cap=0.5)
    kept = [i for i in range(vocab) if i % 3 != 2]
    part = x[:, kept].contiguous()
    lp, ent, tl, ids, m = oracle(part, tok, 3, 0.5)
    base = (64 + 45) * U + 2.0 ** -22 * 0.5 + 4 * U * 31
    for got, want in ((out.logprobs, lp), (out.entropy, ent)):
        g = got.double().cpu().numpy()
        assert (np.abs(g - want) <= 2 * base + 4 * U * np.abs(want) + base * np.abs(ent)).all()
    assert (out.top_ids.cpu().numpy() == np.asarray(kept)[ids]).all()
    assert (token_logprobs(x, tok + 1, 0, logit_cap=0.5).logprobs == -float("inf")).all()


def test_places_without_a_token():
    import torch
    from flash_decode_int4.quality import token_logprobs
    x, tok = make((6,), 100, "float16")
    tok[0], tok[1], tok[2], tok[3] = -1, -100, 100, 2 ** 40
    out = token_logprobs(x, tok, 1)
    assert out.logprobs[:2].tolist() == [0.0, 0.0] and torch.isnan(out.logprobs[2:4]).all()
    assert torch.isfinite(out.logprobs[4:]).all() and torch.isfinite(out.entropy).all()


def test_streams_and_a_graph():
    import torch
    from flash_decode_int4.quality import token_logprobs
    for rows, vocab in ((2, 128000), (300, 2000)):
        x, tok = make((rows,), vocab, "bfloat16")
        want = token_logprobs(x, tok, 9)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = token_logprobs(x, tok, 9)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = token_logprobs(x, tok, 9)
        for step in range(3):
            x.copy_(make((rows,), vocab, "bfloat16", seed=step)[0])
            graph.replay()
            now = [t.clone() for t in out]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(now, token_logprobs(x, tok, 9)))


def test_refused():
    import torch
    from flash_decode_int4.quality import token_logprobs
    x, tok = make((4,), 100, "float32")
    for error, args in ((ValueError, (x, tok[:3])), (ValueError, (x, tok, -1)),
                        (ValueError, (x, tok, 65)), (ValueError, (x[:, :9], tok, 10)),
                        (TypeError, (x.double(), tok)), (TypeError, (x, tok.float())),
                        (TypeError, (x.cpu().numpy(), tok)), (ValueError, (x, tok, 0, 0.0)),
                        (ValueError, (x, tok, 0, float("nan"))), (RuntimeError, (x.cpu(), tok)),
                        (RuntimeError, (x, tok.cpu()))):
        with pytest.raises(error):
            token_logprobs(*args)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("rows,vocab", [(4, 700), (4, 20011), (300, 9001)])
@pytest.mark.parametrize("cap", [None, 2.0])
def test_alternatives_with_infinities(rows, vocab, dtype, cap):
    """+infinity is the largest logit, behind NaN alone."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    x, tok = make((rows,), vocab, dtype)
    inf = float("inf")
    x[0, vocab // 2] = inf
    x[1, 5::3] = inf
    x[2, 9] = float("nan")
    x[2, vocab - 2] = inf
    x[3, 1::2] = -inf
    x[3, 8] = inf
    raw = x.double().cpu().numpy()
    raw[2, 9] = 2e300                      # above infinity for the order
    order = np.where(np.isposinf(raw), 1e300, raw)
    want = np.argsort(-order, axis=1, kind="stable")
    for top in (1, 2, 33, 64):
        out = token_logprobs(x, tok, top, logit_cap=cap)
        assert (out.top_ids.cpu().numpy() == want[:, :top]).all()
        assert torch.isnan(out.top_logprobs[:3]).all() and torch.isnan(out.logprobs[:4]).all()


def test_expanded_rows():
    from flash_decode_int4.quality import token_logprobs
    x, _ = make((2, 3, 1), 515, "float32")
    _, tok = make((2, 3, 4), 515, "float32")
    for view, ids in ((x.expand(2, 3, 4, 515), tok), (x[:, :1].expand(2, 3, 4, 515), tok),
                      (x[:, 0].expand(2, 4, 515), tok[:, 0]), (x[0, :1, 0].expand(4, 515), tok[0, 0])):
        check(token_logprobs(view, ids, 3), view, ids, 3)
