"""A text fed through the INT4 cache in chunks and scored, as measurable cases.

Three operators around the paged INT4 key/value cache:

  attend  queries of the last tokens of every sequence (a chunk of a prompt, or one
          token) over the cache that holds them: causal, with a window and sinks or a
          prefix that all of them see; scores capped by a tanh, or lowered by the distance
  rotate  the norm of every query and key head and the position rotation, from a
          projection's output to the queries and float32 keys that the cache takes
  score   log probabilities of given tokens, the entropy of every row, and the most
          likely alternatives

The plain form is elementary torch in float32 (angles in float64); with `own` set the
same inputs go through the framework's entry points. Inputs are made on the GPU from the
seed alone; lengths and counts belong to the case, so that a case's work is a number.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "int4-kv-cache-quantization-cuda-triton-pallas_amd")

_DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _attend(name, batch, kv_heads, q_heads, head_dim, tokens, new, values, query, ragged=False,
            window=0, sinks=0, prefix=0, cap=0.0, bias=False, page_rows=16, group_rows=128):
    """`tokens` are in the cache, the last `new` of them are the queries'. ragged: fewer of
    both in some sequences. 0: no window, no prefix, no cap."""
    return dict(name=name, kind="attend", batch=batch, kv_heads=kv_heads, q_heads=q_heads,
                head_dim=head_dim, tokens=tokens, new=new, values=values, query=query,
                ragged=ragged, window=window, sinks=sinks, prefix=prefix, cap=cap, bias=bias,
                page_rows=page_rows, group_rows=group_rows)


def _rotate(name, batch, new, kv_heads, q_heads, head_dim, rotary, dtype, norm=True,
            interleaved=False, start=1000):
    """Rows of one fused projection [batch, new, (q_heads + 2 kv_heads) * head_dim], at
    positions from about `start`."""
    return dict(name=name, kind="rotate", batch=batch, new=new, kv_heads=kv_heads,
                q_heads=q_heads, head_dim=head_dim, rotary=rotary, dtype=dtype, norm=norm,
                interleaved=interleaved, start=start)


def _score(name, rows, vocab, dtype, top, cap=0.0, padded=False):
    """padded: some rows have no token (its number is negative)."""
    return dict(name=name, kind="score", rows=rows, vocab=vocab, dtype=dtype, top=top, cap=cap,
                padded=padded)


def listed():
    return [
        # The smallest call: one token of one sequence with capped scores (latency).
        _attend("attend_one_small", 1, 4, 4, 64, 500, 1, "float32", "float32", cap=30.0),
        # A decode step of a model with capped scores, long contexts, 16 bits.
        _attend("attend_one_cap_bf16", 16, 8, 32, 128, 16384, 1, "bfloat16", "bfloat16",
                cap=50.0),
        # A decode step with a distance bias, a kv-head for every head, every length.
        _attend("attend_one_bias_f16", 24, 16, 16, 128, 6000, 1, "float16", "float16",
                ragged=True, bias=True),
        # A chunk of a prompt over a long context: the chunked prefill of a server.
        _attend("attend_chunk_bf16", 8, 8, 32, 128, 8192, 1024, "bfloat16", "bfloat16"),
        # A local layer of a model with capped scores: wide heads, odd and ragged chunks.
        _attend("attend_window_d256_f16", 6, 4, 8, 256, 5000, 700, "float16", "float16",
                ragged=True, window=1024, sinks=4, cap=50.0),
        # A prefix that every token sees (an instruction), then text; float32 throughout.
        _attend("attend_prefix_f32", 3, 4, 8, 64, 1500, 333, "float32", "float32", ragged=True,
                prefix=1300),
        # One token of every sequence of a batch, norms on (latency).
        _rotate("rotate_one", 16, 1, 8, 32, 128, 128, "bfloat16"),
        # Prompts of a batch, norms on, far positions.
        _rotate("rotate_prompt_bf16", 8, 2048, 8, 32, 128, 128, "bfloat16", start=100000),
        # A quarter of the channels rotated, neighbours paired, no norm, float16, odd sizes.
        _rotate("rotate_part_f16", 5, 777, 4, 20, 256, 64, "float16", norm=False,
                interleaved=True),
        # What a decode step's answer carries: few rows, the five most likely tokens (latency).
        _score("score_step_f32", 4, 32000, "float32", 5),
        # The log likelihood of a text: every row of a window, no alternatives.
        _score("score_text_bf16", 2048, 128000, "bfloat16", 0, padded=True),
        # Alternatives of every row, an odd vocabulary, capped.
        _score("score_top_f16", 777, 50021, "float16", 20, cap=30.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over the listed ranges, every type, head layout,
    page and group size in use."""
    kind = rng.choice(["attend", "attend", "attend", "rotate", "score"])
    most = {"bytes": 0, "flops": 0}
    for c in listed():
        if c["kind"] == kind:
            w = work(c)
            most = {k: max(most[k], w[k]) for k in most}
    while True:
        case = dict(kind=kind)
        if kind == "attend":
            kv = rng.choice([1, 2, 4, 8, 8, 16])
            values = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
            tokens = _log_int(rng, 100, 16000)
            form = rng.choice(["plain", "window", "prefix"])
            case.update(batch=_log_int(rng, 1, 24), kv_heads=kv,
                        q_heads=kv * rng.choice([1, 1, 2, 4, 4, 7, 8]),
                        head_dim=rng.choice([64, 128, 128, 256]), tokens=tokens,
                        new=1 if rng.random() < 0.4 else _log_int(rng, 2, min(tokens, 1500)),
                        values=values, query=rng.choice([values, values, "float32", "bfloat16"]),
                        ragged=rng.random() < 0.5, window=0, sinks=0, prefix=0,
                        cap=rng.choice([0.0, 30.0, 50.0]), bias=rng.random() < 0.35,
                        page_rows=rng.choice([16, 16, 16, 32, 64]),
                        group_rows=rng.choice([128, 128, 64, 256]))
            if form == "window":
                case["window"] = _log_int(rng, 32, 6000)
                case["sinks"] = rng.choice([0, 1, 4, 100])
            elif form == "prefix":
                case["prefix"] = rng.randint(1, tokens)
        elif kind == "rotate":
            kv = rng.choice([1, 2, 4, 8, 16])
            d = rng.choice([64, 128, 128, 256])
            case.update(batch=_log_int(rng, 1, 32),
                        new=1 if rng.random() < 0.3 else _log_int(rng, 2, 4000), kv_heads=kv,
                        q_heads=kv * rng.choice([1, 2, 4, 5, 8]), head_dim=d,
                        rotary=rng.choice([d, d, d // 2, d // 4]),
                        dtype=rng.choice(["float32", "float16", "bfloat16", "bfloat16"]),
                        norm=rng.random() < 0.6, interleaved=rng.random() < 0.4,
                        start=rng.choice([0, 1000, 100000]))
        else:
            case.update(rows=_log_int(rng, 1, 4000), vocab=_log_int(rng, 1000, 200000),
                        dtype=rng.choice(["float32", "float16", "bfloat16"]),
                        top=rng.choice([0, 0, 1, 5, 20, 50]),
                        cap=rng.choice([0.0, 0.0, 30.0]), padded=rng.random() < 0.5)
        w = work(case)
        # (A case costs its inputs too, and the plain form a score of every pair.)
        if kind == "attend" and (_pool_bytes(case) > 8e8 or case["batch"] * case["q_heads"]
                                 * case["new"] * case["tokens"] > 2.2e9):
            continue
        if all(w[k] <= most[k] for k in most):
            return case


def _lengths(case):
    """int64 [B] tokens in the cache, and [B] queries of each sequence (its last tokens)."""
    B, T, N = case["batch"], case["tokens"], case["new"]
    if not case["ragged"]:
        return np.full(B, T, np.int64), np.full(B, N, np.int64)
    rng = np.random.RandomState(B * 7919 + T)
    lens = rng.randint(max(1, T // 32), T + 1, size=B).astype(np.int64)
    cnt = rng.randint(max(1, N // 4), N + 1, size=B).astype(np.int64)
    cnt[0] = N
    return lens, np.minimum(cnt, lens)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _inv_freq(rotary):
    j = torch.arange(0, rotary, 2, dtype=torch.float64)
    return (10000.0 ** (-j / rotary)).float().cuda()


def _prepare_attend(case, g):
    """A cache in use (random physical pages) and the queries of its last tokens, scaled."""
    B, H, D, R, G = (case["batch"], case["kv_heads"], case["head_dim"], case["page_rows"],
                     case["group_rows"])
    lens, cnt = _lengths(case)
    cols = -(-int(lens.max()) // R)
    groups = -(-cols * R // G)
    pages = B * cols
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(B, cols)
    codes = torch.empty(2, pages, H, R, D // 2, dtype=torch.uint8, device="cuda")
    for i in range(2):
        x = torch.randn(pages, H, R, D // 2, generator=g, device="cuda")
        codes[i] = x.mul_(2.8).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
    k_pages = codes[0] | (codes[1] << 4)
    # Channels of unlike spread; the scales of a channel differ little between groups.
    spread = torch.exp(0.5 * _randn(g, 1, H, 1, D))
    wobble = 1 + 0.1 * torch.rand(B, H, groups, D, generator=g, device="cuda")
    st = dict(k_pages=k_pages, v_pages=_randn(g, pages, H, R, D, dtype=_DT[case["values"]]),
              k_scale=(0.37 * spread * wobble).contiguous(),
              k_zp=7.5 + 0.7 * _randn(g, B, H, groups, D), table=table, group_rows=G,
              lens=torch.as_tensor(lens, dtype=torch.int32).cuda(),
              counts=torch.as_tensor(cnt, dtype=torch.int32).cuda(),
              window=case["window"], sinks=case["sinks"], cap=case["cap"], prefix=None,
              slopes=None)
    q = _randn(g, B, case["q_heads"], case["new"], D) * (2.0 / math.sqrt(D))
    st["query"] = q.to(_DT[case["query"]])
    if case["prefix"]:
        st["prefix"] = torch.as_tensor(np.minimum(case["prefix"], lens),
                                       dtype=torch.int32).cuda()
    if case["bias"]:
        h = torch.arange(1, case["q_heads"] + 1, device="cuda", dtype=torch.float32)
        st["slopes"] = torch.exp2(-8.0 * h / case["q_heads"])
    return st


def _prepare_rotate(case, g):
    B, N, H, Hq, D = (case["batch"], case["new"], case["kv_heads"], case["q_heads"],
                      case["head_dim"])
    dt = _DT[case["dtype"]]
    qkv = _randn(g, B, N, Hq + 2 * H, D, dtype=dt).transpose(1, 2)
    st = dict(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + H], inv_freq=_inv_freq(case["rotary"]),
              interleaved=case["interleaved"], scale=1.0 / math.sqrt(D), eps=1e-6,
              q_weight=None, k_weight=None)
    st["positions"] = (case["start"] + torch.randint(0, 500, (B,), generator=g,
                                                     device="cuda")).int()
    if case["norm"]:
        st["q_weight"] = 1 + 0.1 * _randn(g, D)
        st["k_weight"] = 1 + 0.1 * _randn(g, D)
    return st


def _prepare_score(case, g):
    R, V = case["rows"], case["vocab"]
    # A few likely tokens in every row above a wide floor.
    x = 2.5 * torch.randn(R, V, generator=g, device="cuda")
    x.scatter_add_(1, torch.randint(0, V, (R, 8), generator=g, device="cuda"),
                   8.0 * torch.rand(R, 8, generator=g, device="cuda"))
    st = dict(logits=x.to(_DT[case["dtype"]]), top=case["top"], cap=case["cap"])
    best = st["logits"].float().argmax(1)
    other = torch.randint(0, V, (R,), generator=g, device="cuda")
    tokens = torch.where(torch.rand(R, generator=g, device="cuda") < 0.5, best, other)
    if case["padded"]:
        tokens[torch.rand(R, generator=g, device="cuda") < 0.1] = -100
    st["tokens"] = tokens
    return st


_PREPARE = {"attend": _prepare_attend, "rotate": _prepare_rotate, "score": _prepare_score}


def prepare(case, seed):
    return dict(kind=case["kind"], **_PREPARE[case["kind"]](case, _gen(seed)))


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

def _seen(lens, counts, N, T, window, sinks, prefix):
    """bool [B, N, T]: the cached tokens that each query sees; and [B, N] positions."""
    dev = lens.device
    i = torch.arange(N, device=dev)[None]
    n, c = lens.long()[:, None], counts.long()[:, None]
    pos = n - c + i
    t = torch.arange(T, device=dev)[None, None]
    seen = t <= pos[:, :, None]
    if window:
        seen = seen & ((t < sinks) | (t > pos[:, :, None] - window))
    if prefix is not None:
        seen = seen | (t < prefix.long()[:, None, None])
    return seen & (t < n[:, :, None]) & (i < c)[:, :, None], pos


def _dense(st):
    """Keys (dequantized) and values of all pages as float32 [B, H, T, D], zeros behind a
    sequence's end."""
    kp, vp, table, G = st["k_pages"], st["v_pages"], st["table"].long(), st["group_rows"]
    B, cols = table.shape
    H, R, D = vp.shape[1:]
    raw = kp[table].permute(0, 2, 1, 3, 4).reshape(B, H, cols * R, D // 2)
    codes = torch.stack([raw & 15, raw >> 4], -1).flatten(-2).float()
    s = st["k_scale"].repeat_interleave(G, 2)[:, :, :cols * R]
    z = st["k_zp"].repeat_interleave(G, 2)[:, :, :cols * R]
    v = vp[table].permute(0, 2, 1, 3, 4).reshape(B, H, cols * R, D).float()
    there = torch.arange(cols * R, device=kp.device)[None] < st["lens"].long()[:, None]
    there = there[:, None, :, None]
    return torch.where(there, codes * s - z * s, 0.0), torch.where(there, v, 0.0)


def _plain_attend(st):
    q = st["query"]
    B, Hq, N, D = q.shape
    k, v = _dense(st)
    H, T = k.shape[1:3]
    seen, pos = _seen(st["lens"], st["counts"], N, T, st["window"], st["sinks"], st["prefix"])
    x = torch.matmul(q.float().reshape(B, H, -1, D), k.transpose(2, 3))
    x = x.reshape(B, H, Hq // H, N, T)
    if st["cap"]:
        x = st["cap"] * torch.tanh(x / st["cap"])
    if st["slopes"] is not None:
        far = (pos[:, :, None] - torch.arange(T, device=q.device)).abs().float()
        x = x - st["slopes"].view(1, H, -1, 1, 1) * far[:, None, None]
    x = torch.where(seen[:, None, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.where(seen[:, None, None], torch.exp(x - m), 0.0)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(B, H, -1, T), v).reshape(B, H, Hq // H, N, D)
    out = out / torch.where(total > 0, total, 1.0)
    return out.reshape(B, Hq, N, D).to(q.dtype)


def _plain_rotate(st):
    B, Hq, N, D = st["q"].shape
    f = st["inv_freq"]
    R = 2 * f.shape[0]
    pos = st["positions"].long()[:, None] + torch.arange(N, device=f.device)
    angle = pos.double()[..., None] * f.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + st["eps"]) * w
        rot, rest = y[..., :R], y[..., R:]
        if st["interleaved"]:
            a, b = rot[..., 0::2], rot[..., 1::2]
            rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = rot[..., :R // 2], rot[..., R // 2:]
            rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.cat([rot, rest], -1))
    return (out[0] * st["scale"]).to(st["q"].dtype), out[1]


def _plain_score(st):
    raw = st["logits"].float()
    x = raw if not st["cap"] else st["cap"] * torch.tanh(raw / st["cap"])
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1)
    lse = m[:, 0] + torch.log(total)
    entropy = torch.log(total) - (e * torch.where(e > 0, x - m, 0.0)).sum(-1) / total
    tok = st["tokens"]
    mine = x.gather(1, tok.clamp(min=0)[:, None])[:, 0] - lse
    out = [torch.where(tok >= 0, mine, 0.0), entropy]
    if st["top"]:
        ids = raw.sort(dim=1, descending=True, stable=True).indices[:, :st["top"]]
        out += [x.gather(1, ids) - lse[:, None], ids]
    return out


_PLAIN = {"attend": _plain_attend, "rotate": _plain_rotate, "score": _plain_score}


def _entry_points():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from flash_decode_int4 import ops, quality
    return ops, quality


def run(st):
    kind = st["kind"]
    if not own:
        return _PLAIN[kind](st)
    ops, quality = _entry_points()
    if kind == "attend":
        return ops.flash_attend_paged(
            st["query"], st["k_pages"], st["v_pages"], st["k_scale"], st["k_zp"], st["table"],
            st["lens"], counts=st["counts"], group_rows=st["group_rows"],
            window=st["window"] or None, sinks=st["sinks"], prefix_lens=st["prefix"],
            logit_cap=st["cap"] or None, slopes=st["slopes"])
    if kind == "rotate":
        return ops.norm_rotary(st["q"], st["k"], st["positions"], st["inv_freq"],
                               q_weight=st["q_weight"], k_weight=st["k_weight"], eps=st["eps"],
                               q_scale=st["scale"], interleaved=st["interleaved"])
    out = quality.token_logprobs(st["logits"], st["tokens"], top=st["top"],
                                 logit_cap=st["cap"] or None)
    return [out.logprobs, out.entropy] + ([out.top_logprobs, out.top_ids] if st["top"] else [])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _size(dt):
    return 4 if dt == "float32" else 2


def _pool_bytes(case):
    D = case["head_dim"]
    return (case["batch"] * case["kv_heads"] * case["tokens"]
            * (D // 2 + D * _size(case["values"])))


def _runs(case, n, c):
    """The cached tokens that the last c tokens of n see, as ranges [begin, end), and the
    number of (query, token) pairs."""
    W, S, P = case["window"], case["sinks"], min(case["prefix"], n)
    pos = np.arange(n - c, n, dtype=np.int64)
    low = np.maximum(pos - W + 1, 0) if W else np.zeros(c, np.int64)
    head = np.minimum(S, pos + 1) if W else np.zeros(c, np.int64)
    head = np.maximum(head, P)
    pairs = int((head + np.maximum(pos + 1 - np.maximum(low, head), 0)).sum())
    end = max(n, P)
    first = int(low.min())
    front = int(head.max())
    return ([(0, end)] if front >= first else [(0, front), (first, end)]), pairs


def work(case):
    if case["kind"] == "attend":
        lens, cnt = _lengths(case)
        B, H, Hq, D = case["batch"], case["kv_heads"], case["q_heads"], case["head_dim"]
        R, G = case["page_rows"], case["group_rows"]
        nbytes = Hq * D * _size(case["query"]) * (int(cnt.sum()) + B * case["new"]) + 8 * B
        pairs = 0
        for n, c in zip(lens.tolist(), cnt.tolist()):
            runs, p = _runs(case, n, c)
            pairs += p
            for begin, end in runs:
                if end <= begin:
                    continue
                nbytes += H * (end - begin) * (D // 2 + D * _size(case["values"]))
                nbytes += H * (-(-end // G) - begin // G) * D * 8
                nbytes += (-(-end // R) - begin // R) * 4
        return dict(bytes=nbytes, flops=4 * Hq * D * pairs)
    if case["kind"] == "rotate":
        rows = case["batch"] * case["new"]
        H, Hq, D, es = case["kv_heads"], case["q_heads"], case["head_dim"], _size(case["dtype"])
        return dict(bytes=rows * D * (2 * Hq * es + H * (es + 4)),
                    flops=rows * (Hq + H) * (3 * case["rotary"] + (4 * D if case["norm"] else 0)))
    R, V = case["rows"], case["vocab"]
    return dict(bytes=R * (V * _size(case["dtype"]) + 16 + 12 * case["top"]), flops=5 * R * V)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _sequence64(st, b, n, H, D):
    """float64 keys and values [H, n, D] of sequence b."""
    R, G = st["k_pages"].shape[2], st["group_rows"]
    pages = st["table"][b, :-(-n // R)].long()
    raw = st["k_pages"][pages].permute(1, 0, 2, 3).reshape(H, -1, D // 2)[:, :n]
    q = torch.empty(H, n, D, dtype=torch.float64, device=raw.device)
    q[..., 0::2] = raw % 16
    q[..., 1::2] = raw // 16
    for g0 in range(0, n, G):
        q[:, g0:g0 + G] -= st["k_zp"][b, :, g0 // G].double()[:, None]
        q[:, g0:g0 + G] *= st["k_scale"][b, :, g0 // G].double()[:, None]
    v = st["v_pages"][pages].permute(1, 0, 2, 3).reshape(H, -1, D)[:, :n].double()
    return q, v


def _exact_attend(case, st):
    lens, cnt = _lengths(case)
    B, H, Hq, D, N = (case["batch"], case["kv_heads"], case["q_heads"], case["head_dim"],
                      case["new"])
    per, W, cap = Hq // H, case["window"], case["cap"]
    out = torch.zeros(B, Hq, N, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, c = int(lens[b]), int(cnt[b])
        k, v = _sequence64(st, b, n, H, D)
        t = torch.arange(n, device="cuda")[None]
        at = torch.arange(n - c, n, device="cuda")[:, None]
        hidden = t > at
        if W:
            hidden |= (t >= case["sinks"]) & (at - t >= W)
        if case["prefix"]:
            hidden &= t >= min(case["prefix"], n)
        for h in range(Hq):
            x = st["query"][b, h, :c].double() @ k[h // per].T
            if cap:
                x = torch.tanh(x / cap) * cap
            if case["bias"]:
                x = x - st["slopes"][h].double() * (at - t).abs()
            w = torch.softmax(x.masked_fill_(hidden, -math.inf), -1)
            out[b, h, :c] = w @ v[h // per]
    return out


def _exact_rotate(case, st):
    R, N = case["rotary"], case["new"]
    out = []
    for x, w, scale in ((st["q"], st["q_weight"], st["scale"]), (st["k"], st["k_weight"], 1.0)):
        y = x.double()
        if case["norm"]:
            y = y / (y.square().mean(-1, keepdim=True) + st["eps"]).sqrt() * w.double()
        at = st["positions"].double()[:, None] + torch.arange(N, device="cuda").double()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           at[:, None, :, None] * st["inv_freq"].double())
        first = slice(0, R, 2) if case["interleaved"] else slice(0, R // 2)
        second = slice(1, R, 2) if case["interleaved"] else slice(R // 2, R)
        pair = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
        y = y.clone()
        y[..., first], y[..., second] = pair.real, pair.imag
        out.append(y * scale)
    return tuple(out)


def _exact_score(case, st):
    raw = st["logits"].double()
    x = torch.tanh(raw / case["cap"]) * case["cap"] if case["cap"] else raw
    logp = torch.log_softmax(x, -1)
    tok = st["tokens"]
    mine = logp.gather(1, tok.clamp(min=0)[:, None])[:, 0]
    out = [torch.where(tok < 0, torch.zeros_like(mine), mine), -(logp.exp() * logp).sum(-1)]
    if case["top"]:
        # (Among equal logits the places do not matter for the values.)
        best = raw.topk(case["top"], dim=1).values
        best = torch.tanh(best / case["cap"]) * case["cap"] if case["cap"] else best
        out += [best - torch.logsumexp(x, -1, keepdim=True), None]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"attend": _exact_attend, "rotate": _exact_rotate,
            "score": _exact_score}[case["kind"]](case, st)
