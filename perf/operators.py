"""Attention over part of the INT4 cache and over drafted tokens, and the writes and
reads of runs of tokens, as measurable cases.

Four operators on the paged INT4 key/value cache:

  window  one query token per sequence over the first `sinks` and the last
          `window` tokens of the cache
  tree    a tree of drafted tokens per sequence over the cache (all of it, or
          sinks and a window) and over the drafts that each of them descends from
  extend  several tokens per sequence into the cache (all of a chunk, or the
          accepted path of a tree), and the scale groups that this touched read
          back as values
  read    a range of every sequence's tokens back as dense keys and values

The plain form is elementary torch in float32; with `own` set the same inputs go
through the framework's entry points. Inputs are made on the GPU from the seed
alone; lengths, counts and trees belong to the case, so that a case's work is a
number. Keys are INT4 codes as normal keys give them, their scales differing
between channels and groups; queries are N(0, 1) * 2 / sqrt(D) (no softmax scale
is applied, so a caller scales the query).
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

def _attend(name, kind, batch, kv_heads, q_heads, head_dim, tokens, nodes=1, window=0, sinks=0,
            ragged=False, values="float32", query="float32", chain=False, page_rows=16,
            group_rows=128):
    """window 0: the whole cache. chain: the drafts follow one another (a chunk of
    a prompt); otherwise every sequence has a random tree."""
    return dict(name=name, kind=kind, batch=batch, kv_heads=kv_heads, q_heads=q_heads,
                head_dim=head_dim, tokens=tokens, nodes=nodes, window=window, sinks=sinks,
                ragged=ragged, values=values, query=query, chain=chain, page_rows=page_rows,
                group_rows=group_rows)


def _write(name, batch, kv_heads, head_dim, tokens, new, path, ragged=False, values="float32",
           page_rows=16, group_rows=128):
    """path: between none and all of `new` drafts are accepted, by index, inside the
    open scale group; otherwise a whole chunk of `new` tokens from a group's start."""
    return dict(name=name, kind="extend", batch=batch, kv_heads=kv_heads, head_dim=head_dim,
                tokens=tokens, new=new, path=path, ragged=ragged, values=values,
                page_rows=page_rows, group_rows=group_rows)


def _read(name, batch, kv_heads, head_dim, tokens, start, length, out, ragged=False,
          values="float32", page_rows=16, group_rows=128):
    return dict(name=name, kind="read", batch=batch, kv_heads=kv_heads, head_dim=head_dim,
                tokens=tokens, start=start, length=length, out=out, ragged=ragged,
                values=values, page_rows=page_rows, group_rows=group_rows)


def listed():
    return [
        # The smallest call: one sequence, four heads, a short window (latency).
        _attend("window_small", "window", 1, 4, 4, 64, 500, window=128, sinks=4),
        # A chat model's sliding-window layer late in a long context, 16 bits.
        _attend("window_gqa_bf16", "window", 16, 8, 32, 128, 16384, window=4096, sinks=4,
                values="bfloat16", query="bfloat16"),
        # One query per head, float32 values, the headline's layout in a window.
        _attend("window_mha_f32", "window", 8, 32, 32, 128, 4000, window=1024, sinks=16),
        # Continuous batching: every length, some shorter than the window; wide heads.
        _attend("window_ragged_d256_f16", "window", 24, 4, 16, 256, 9000, window=1000, sinks=64,
                ragged=True, values="float16", query="float16"),
        # The smallest tree: five drafts of one short sequence.
        _attend("tree_small", "tree", 1, 4, 8, 64, 300, nodes=5),
        # Sixteen drafts a sequence over long contexts: a decode step that verifies.
        _attend("tree_gqa_bf16", "tree", 8, 8, 32, 128, 8192, nodes=16, values="bfloat16",
                query="bfloat16"),
        # Ragged lengths, an odd tree, eight heads per kv-head, within a window.
        _attend("tree_window_f16", "tree", 16, 8, 64, 128, 4096, nodes=21, window=1500, sinks=4,
                ragged=True, values="float16", query="float16"),
        # The last chunk of a prompt: a chain of 100 tokens, float32 throughout.
        _attend("tree_chain_f32", "tree", 4, 8, 16, 128, 3000, nodes=100, ragged=True,
                chain=True),
        # Accepted drafts of a batch into their open groups (latency, small writes).
        _write("extend_accepted_bf16", 16, 8, 128, 2000, 8, True, ragged=True,
               values="bfloat16"),
        # A chunk of a prompt for every sequence, ending in a partial group.
        _write("extend_chunk_f16", 8, 8, 128, 2048, 1000, False, values="float16"),
        # A few hundred tokens from the middle of ragged sequences, as float32.
        _read("read_ragged_f32", 6, 4, 64, 3000, 333, 700, "float32", ragged=True),
        # Whole long sequences to 16 bits (for a dense kernel, or to move the cache).
        _read("read_all_bf16", 8, 8, 128, 8192, 0, 8192, "bfloat16", values="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes log-uniform over the listed ranges, every type, head
    layout, page and group size in use."""
    most = {}
    for c in listed():
        w = work(c)
        most["bytes"] = max(most.get("bytes", 0), w["bytes"])
        most["flops"] = max(most.get("flops", 0), w["flops"])
    while True:
        kind = rng.choice(["window", "window", "tree", "tree", "tree", "extend", "read"])
        kv = rng.choice([1, 2, 4, 8, 8, 16, 32])
        values = rng.choice(["float32", "float16", "bfloat16"])
        case = dict(kind=kind, batch=_log_int(rng, 1, 32), kv_heads=kv,
                    head_dim=rng.choice([64, 128, 128, 256]), tokens=_log_int(rng, 100, 16000),
                    ragged=rng.random() < 0.5, values=values,
                    page_rows=rng.choice([16, 16, 16, 32, 64]),
                    group_rows=rng.choice([128, 128, 64, 256]))
        if kind in ("window", "tree"):
            case["q_heads"] = kv * (rng.choice([1, 1, 2, 4, 4, 7, 8]) if kv <= 16 else 1)
            case["query"] = rng.choice([values, values, "float32"])
            case["nodes"] = _log_int(rng, 1, 128) if kind == "tree" else 1
            case["chain"] = kind == "tree" and rng.random() < 0.3
            case["sinks"] = rng.choice([0, 1, 4, 16, 100])
            if kind == "window" or rng.random() < 0.4:
                case["window"] = max(_log_int(rng, 32, 6000), case["nodes"])
            else:
                case["window"] = case["sinks"] = 0
        elif kind == "extend":
            case["path"] = rng.random() < 0.5
            case["new"] = _log_int(rng, 1, 40) if case["path"] else _log_int(rng, 20, 2000)
        else:
            case["out"] = rng.choice(["float32", values])
            case["start"] = rng.choice([0, rng.randint(0, case["tokens"] // 2)])
            case["length"] = _log_int(rng, 1, case["tokens"] - case["start"])
        w = work(case)
        # (A case costs its inputs too: caches far larger than what is attended over.)
        if (w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]
                and _pool_bytes(case) <= 6e8):
            return case


def _lengths(case):
    """int64 [B] tokens in the cache before the call."""
    B, T, G = case["batch"], case["tokens"], case["group_rows"]
    if case["ragged"]:
        rng = np.random.RandomState(B * 7919 + T)
        lens = rng.randint(max(1, T // 64), T + 1, size=B)
    else:
        lens = np.full(B, T)
    lens = lens.astype(np.int64)
    if case["kind"] == "extend":
        # A pass is repeated on the same state, so no staged row that it reads is
        # overwritten by a later group's: accepted drafts stay inside the open group,
        # chunks begin with one.
        if case["path"]:
            lens -= np.maximum(lens % G + case["new"] - G, 0)
            lens = np.maximum(lens, 0)
        else:
            lens -= lens % G
    return lens


def _counts(case):
    """int64 [B] tokens that an extend takes of each sequence's new ones."""
    B, N = case["batch"], case["new"]
    if not case["path"]:
        return np.full(B, N, np.int64)
    cnt = np.random.RandomState(B * 31 + N).randint(0, N + 1, size=B).astype(np.int64)
    cnt[0] = max(cnt[0], 1)
    return cnt


def _parents(case):
    """int64 [B, N]: the node each draft follows (an earlier one), or -1 for the cache."""
    B, N = case["batch"], case["nodes"]
    if case["chain"]:
        return np.tile(np.arange(-1, N - 1), (B, 1))
    rng = np.random.RandomState(B * 131 + N)
    back = rng.randint(1, 6, size=(B, N))
    return np.maximum(np.arange(N)[None] - back, -1)


def _tree(case):
    """bool [B, N, N]: the drafts that draft i sees (its ancestors and itself)."""
    B, N = case["batch"], case["nodes"]
    up = _parents(case)
    mask = np.zeros((B, N, N), bool)
    for i in range(N):
        has = up[:, i] >= 0
        mask[has, i] = mask[has, up[has, i]]
        mask[:, i, i] = True
    return mask


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _capacity(case):
    extra = case.get("new", 0)
    return int(_lengths(case).max()) + extra


def _cache(case, g):
    """A cache in use: random physical pages, codes and values, and its lengths."""
    B, H, D, R, G = (case["batch"], case["kv_heads"], case["head_dim"], case["page_rows"],
                     case["group_rows"])
    lens = _lengths(case)
    cols = -(-_capacity(case) // R)
    groups = -(-cols * R // G)
    pages = B * cols
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(B, cols)
    codes = torch.empty(2, pages, H, R, D // 2, dtype=torch.uint8, device="cuda")
    for i in range(2):
        x = torch.randn(pages, H, R, D // 2, generator=g, device="cuda")
        codes[i] = x.mul_(2.8).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
    k_pages = codes[0] | (codes[1] << 4)
    spread = torch.exp(0.5 * _randn(g, 1, H, 1, D))
    wobble = 1 + 0.1 * torch.rand(B, H, groups, D, generator=g, device="cuda")
    k_scale = (0.37 * spread * wobble).contiguous()
    k_zp = 7.5 + 0.7 * _randn(g, B, H, groups, D)
    v_pages = _randn(g, pages, H, R, D, dtype=_DT[case["values"]])
    return dict(k_pages=k_pages, v_pages=v_pages, k_scale=k_scale, k_zp=k_zp, table=table,
                lens=torch.as_tensor(lens, dtype=torch.int32).cuda(), group_rows=G)


def prepare(case, seed):
    kind = case["kind"]
    g = _gen(seed)
    st = dict(kind=kind, **_cache(case, g))
    B, H, D = case["batch"], case["kv_heads"], case["head_dim"]
    vdt = _DT[case["values"]]
    if kind in ("window", "tree"):
        N = case["nodes"]
        q = _randn(g, B, case["q_heads"], N, D) * (2.0 / math.sqrt(D))
        st.update(query=q.to(_DT[case["query"]]), window=case["window"], sinks=case["sinks"])
        if kind == "window":
            st["query"] = st["query"][:, :, 0]
            return st
        # Drafts as their layer gives them: float32 keys, values of the cache's type.
        st.update(k_draft=_randn(g, B, H, N, D), v_draft=_randn(g, B, H, N, D, dtype=vdt),
                  mask=torch.from_numpy(_tree(case)).cuda())
        return st
    if kind == "extend":
        N, G = case["new"], case["group_rows"]
        st.update(k_new=_randn(g, B, H, N, D), v_new=_randn(g, B, H, N, D, dtype=vdt),
                  k_stage=_randn(g, B, H, G, D),
                  counts=torch.as_tensor(_counts(case), dtype=torch.int32).cuda(),
                  lens_next=torch.zeros(B, dtype=torch.int32, device="cuda"),
                  index=None)
        if case["path"]:
            # An accepted path: increasing indices into the drafts.
            order = torch.rand(B, N, generator=g, device="cuda").argsort(1)
            n = torch.arange(N, device="cuda")
            taken = n[None] < st["counts"][:, None]
            st["index"] = torch.where(taken, order, N).sort(1).values.clamp(max=N - 1).int()
        # What is read back: the rows of the groups that the call touches.
        st["first"] = (st["lens"] // G * G).to(torch.int32)
        st["rows"] = int((_lengths(case) % G + _counts(case)).max())
        return st
    st.update(start=case["start"], length=case["length"], out=_DT[case["out"]])
    return st


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

def _tokens(st, pos, dtype=torch.float32):
    """Keys (dequantized, float32) and values (float32) of tokens pos [B, n] (in range)
    as [B, H, n, D]."""
    kp, vp, G = st["k_pages"], st["v_pages"], st["group_rows"]
    R = kp.shape[2]
    page = st["table"].long().gather(1, pos // R)
    row = pos % R
    b = kp[page, :, row]                                   # [B, n, H, D/2]
    codes = torch.stack([b & 15, b >> 4], -1).flatten(-2).float().transpose(1, 2)
    grp = (pos // G)[:, None, :, None].expand(-1, kp.shape[1], -1, codes.shape[-1])
    s, z = st["k_scale"].gather(2, grp), st["k_zp"].gather(2, grp)
    return codes * s - z * s, vp[page, :, row].transpose(1, 2).float()


def _softmax_values(logits, seen, v):
    """softmax over the seen places, times v; a row that sees nothing is zero."""
    logits = torch.where(seen, logits, -math.inf)
    m = logits.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(logits - m), 0.0)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _plain_attend(st):
    tree = st["kind"] == "tree"
    q = st["query"] if tree else st["query"][:, :, None]
    B, Hq, N, D = q.shape
    H = st["k_pages"].shape[1]
    n = st["lens"].long()
    W, S = st["window"], st["sinks"]
    cap = st["table"].shape[1] * st["k_pages"].shape[2]
    # Node i is the last token of the sequence that it sees: the cached tokens and then
    # its drafts (a plain decode's query is itself the last token of the cache).
    own_tokens = st["mask"].sum(-1) if tree else torch.zeros(B, 1, dtype=torch.long,
                                                             device=q.device)
    if W:
        at = torch.arange(W, device=q.device)[None] + (n - W)[:, None]
        first = torch.arange(S, device=q.device)[None].expand(B, S)
        pos = torch.cat([first, at], 1)
        lower = (n[:, None] + own_tokens - W)[:, :, None]
        sink = (torch.arange(S + W, device=q.device) < S)[None, None]
        p = pos[:, None]
        seen = torch.where(sink, p < n[:, None, None],
                           (p >= lower) & (p >= S) & (p >= 0)).expand(B, N, -1)
        pos = pos.clamp(0, cap - 1)
    else:
        pos = torch.arange(cap, device=q.device)[None].expand(B, cap)
        seen = (pos < n[:, None])[:, None].expand(B, N, -1)
    k, v = _tokens(st, pos)
    # Rows behind a sequence's end hold whatever the pool holds.
    used = seen.any(1)[:, None, :, None]
    v = torch.where(used, v, 0.0)
    qg = q.float().reshape(B, H, -1, D)
    if tree:
        k = torch.cat([k, st["k_draft"]], 2)
        v = torch.cat([v, st["v_draft"].float()], 2)
        seen = torch.cat([seen, st["mask"]], 2)
    logits = torch.matmul(qg, k.transpose(2, 3)).reshape(B, H, Hq // H, N, -1)
    out = _softmax_values(logits, seen[:, None, None], v[:, :, None])
    out = out.reshape(B, Hq, N, D).to(q.dtype)
    return out if tree else out[:, :, 0]


def _plain_extend(st):
    kp, vp, G = st["k_pages"], st["v_pages"], st["group_rows"]
    B, H, N, D = st["k_new"].shape
    R, dev = kp.shape[2], kp.device
    n, cnt = st["lens"].long(), st["counts"].long()
    first, rows = st["first"].long(), st["rows"]
    k_new, v_new = st["k_new"], st["v_new"]
    if st["index"] is not None:
        take = st["index"].long()[:, None, :, None].expand(B, H, N, D)
        k_new, v_new = k_new.gather(2, take), v_new.gather(2, take)
    # Rows r of the touched groups: staged ones, then the new ones.
    r = torch.arange(-(-rows // G) * G, device=dev)[None]
    old = (n - first)[:, None]
    valid = r < old + cnt[:, None]
    staged = st["k_stage"][:, :, r[0] % G]
    src = (r - old).clamp(0, N - 1)[:, None, :, None].expand(B, H, r.shape[1], D)
    k = torch.where((r < old)[:, None, :, None], staged, k_new.gather(2, src))
    keep = valid[:, None, :, None]
    grouped = (B, H, -1, G, D)
    mn = torch.where(keep, k, math.inf).reshape(grouped).amin(3)
    mx = torch.where(keep, k, -math.inf).reshape(grouped).amax(3)
    s = torch.clamp(mx - mn, min=1e-8) / torch.full((), 15.0, device=dev)
    z = -mn / s
    step, low = s.repeat_interleave(G, 2), mn.repeat_interleave(G, 2)
    codes = torch.round((k - low) / step).clamp(0, 15).to(torch.uint8)
    packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
    # To the pages, the scales and the staging rows; only rows that exist.
    b, at = torch.nonzero(valid & (cnt > 0)[:, None], as_tuple=True)
    tok = first[b] + at
    page = st["table"].long()[b, tok // R]
    kp[page, :, tok % R] = packed[b, :, at]
    fresh = at >= old[b, 0]
    fb, fat, ftok, fpage = b[fresh], at[fresh], tok[fresh], page[fresh]
    vp[fpage, :, ftok % R] = v_new[fb, :, fat - old[fb, 0]]
    heads = at % G == 0
    st["k_scale"][b[heads], :, tok[heads] // G] = s[b[heads], :, at[heads] // G]
    st["k_zp"][b[heads], :, tok[heads] // G] = z[b[heads], :, at[heads] // G]
    end = old[:, 0] + cnt
    is_open = fresh & (at >= (end // G * G)[b])
    st["k_stage"][b[is_open], :, at[is_open] % G] = k[b[is_open], :, at[is_open]]
    st["lens_next"].copy_((n + cnt).int())
    return _plain_read(st, first, st["rows"], st["lens_next"].long(), torch.float32)


def _plain_read(st, first, length, lens, dtype):
    cap = st["table"].shape[1] * st["k_pages"].shape[2]
    pos = first[:, None] + torch.arange(length, device=first.device)[None]
    there = (pos < lens[:, None])[:, None, :, None]
    k, v = _tokens(st, pos.clamp(max=cap - 1))
    return torch.where(there, k, 0.0).to(dtype), torch.where(there, v, 0.0).to(dtype)


def _entry_points():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from flash_decode_int4 import ops
    return ops


def run(st):
    kind = st["kind"]
    if own:
        ops = _entry_points()
        cache = (st["k_pages"], st["v_pages"], st["k_scale"], st["k_zp"], st["table"])
        if kind == "window":
            return ops.flash_decode_paged(st["query"], *cache, st["lens"], st["group_rows"],
                                          window=st["window"], sinks=st["sinks"])
        if kind == "tree":
            return ops.flash_decode_paged_tree(st["query"], st["k_draft"], st["v_draft"],
                                               st["mask"], *cache, st["lens"],
                                               st["group_rows"], window=st["window"] or None,
                                               sinks=st["sinks"])
        if kind == "read":
            return ops.dequantize_int4_paged(*cache, st["lens"], st["start"], st["length"],
                                             st["group_rows"], dtype=st["out"])
        ops.extend_int4_paged(st["k_new"], st["v_new"], st["counts"], st["k_stage"], *cache,
                              st["lens"], st["lens_next"], st["group_rows"], index=st["index"])
        k, v = ops.dequantize_int4_paged(*cache, st["lens_next"], st["first"], st["rows"],
                                         st["group_rows"], dtype=torch.float32)
    else:
        if kind in ("window", "tree"):
            return _plain_attend(st)
        if kind == "read":
            first = torch.full_like(st["lens"], st["start"]).long()
            return _plain_read(st, first, st["length"], st["lens"].long(), st["out"])
        k, v = _plain_extend(st)
    return dict(k=k, v=v, k_scale=st["k_scale"], k_zp=st["k_zp"], stage=st["k_stage"],
                lens=st["lens_next"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _size(dt):
    return 4 if dt == "float32" else 2


def _pool_bytes(case):
    D = case["head_dim"]
    return (case["batch"] * case["kv_heads"] * _capacity(case)
            * (D // 2 + D * _size(case["values"])))


def _cached_bytes(case, begin, end):
    """Codes, values, scales and table entries of cached tokens [begin, end)."""
    if end <= begin:
        return 0
    H, D, R, G = case["kv_heads"], case["head_dim"], case["page_rows"], case["group_rows"]
    per = D // 2 + D * _size(case["values"])
    return (H * ((end - begin) * per + (-(-end // G) - begin // G) * D * 8)
            + (-(-end // R) - begin // R) * 4)


def work(case):
    kind, lens = case["kind"], _lengths(case)
    B, H, D, G = case["batch"], case["kv_heads"], case["head_dim"], case["group_rows"]
    veb = _size(case["values"])
    if kind in ("window", "tree"):
        Hq, N, W, S = case["q_heads"], case["nodes"], case["window"], case["sinks"]
        nbytes = 2 * B * Hq * N * D * _size(case["query"]) + 4 * B
        if kind == "tree":
            seen = _tree(case).sum(-1)
            nbytes += B * (H * N * D * (4 + veb) + N * N)
        else:
            seen = np.zeros((B, 1), np.int64)
        pairs = int(seen.sum())
        for b, n in enumerate(lens.tolist()):
            if not W:
                nbytes += _cached_bytes(case, 0, n)
                pairs += N * n
                continue
            low = np.clip(n + seen[b] - W, 0, n)
            first = int(low.min())
            sinks = min(S, first)
            nbytes += _cached_bytes(case, 0, sinks) + _cached_bytes(case, first, n)
            pairs += int((n - low + np.minimum(S, low)).sum())
        return dict(bytes=nbytes, flops=4 * Hq * D * pairs)
    if kind == "extend":
        cnt = _counts(case)
        old = lens % G
        touched = np.where(cnt > 0, old + cnt, 0)
        groups = int((-(-touched // G)).sum())
        stage = int(np.where(cnt > 0, np.minimum(cnt, (old + cnt) % G), 0).sum())
        staged = int(np.where(cnt > 0, old, 0).sum())
        rows = int(touched.sum())
        nbytes = H * D * (int(cnt.sum()) * (4 + 2 * veb) + (staged + stage) * 4 + groups * 8)
        nbytes += H * rows * (D // 2)
        # Read back: codes, values and scales of the touched rows, as float32.
        back = int(((old + cnt)).sum())
        nbytes += H * (back * (D // 2 + D * veb) + int((-(-(old + cnt) // G)).sum()) * D * 8)
        nbytes += 2 * B * H * _read_back_rows(case) * D * 4
        return dict(bytes=nbytes, flops=H * D * (6 * rows + 3 * back))
    nbytes = 2 * B * H * case["length"] * D * _size(case["out"])
    rows = 0
    for n in lens.tolist():
        end = min(n, case["start"] + case["length"])
        nbytes += _cached_bytes(case, case["start"], end) + 4
        rows += max(0, end - case["start"])
    return dict(bytes=nbytes, flops=3 * H * D * rows)


def _read_back_rows(case):
    """Rows that an extend's read-back returns per sequence."""
    return int((_lengths(case) % case["group_rows"] + _counts(case)).max())


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _sequence64(st, b, n, H, D):
    """float64 keys and values [H, n, D] of the first n tokens of sequence b."""
    R, G = st["k_pages"].shape[2], st["group_rows"]
    pages = st["table"][b, :-(-n // R)].long()
    raw = st["k_pages"][pages].permute(1, 0, 2, 3).reshape(H, -1, D // 2)[:, :n]
    q = torch.empty(H, n, D, dtype=torch.float64, device=raw.device)
    q[..., 0::2] = raw % 16
    q[..., 1::2] = raw // 16
    for g0 in range(0, n, G):
        g = g0 // G
        q[:, g0:g0 + G] -= st["k_zp"][b, :, g].double()[:, None]
        q[:, g0:g0 + G] *= st["k_scale"][b, :, g].double()[:, None]
    v = st["v_pages"][pages].permute(1, 0, 2, 3).reshape(H, -1, D)[:, :n].double()
    return q, v


def exact(case, seed):
    st = prepare(case, seed)
    kind, lens = case["kind"], _lengths(case)
    B, H, D, G = case["batch"], case["kv_heads"], case["head_dim"], case["group_rows"]
    if kind == "read":
        n1 = case["start"] + case["length"]
        k = torch.zeros(B, H, case["length"], D, dtype=torch.float64, device="cuda")
        v = torch.zeros_like(k)
        for b in range(B):
            kb, vb = _sequence64(st, b, int(lens[b]), H, D)
            kb, vb = kb[:, case["start"]:n1], vb[:, case["start"]:n1]
            k[b, :, :kb.shape[1]], v[b, :, :vb.shape[1]] = kb, vb
        return k, v
    if kind == "extend":
        # Codes next to a border have no value in 64 bits; scales and zero-points have.
        cnt = _counts(case)
        s, z = st["k_scale"].double(), st["k_zp"].double()
        v = torch.zeros(B, H, _read_back_rows(case), D, dtype=torch.float64, device="cuda")
        for b in range(B):
            n, c = int(lens[b]), int(cnt[b])
            first, old = n // G * G, n % G
            if old:
                v[b, :, :old] = _sequence64(st, b, n, H, D)[1][:, first:]
            if not c:
                continue
            pick = (st["index"][b, :c].long() if st["index"] is not None
                    else torch.arange(c, device="cuda"))
            keys = torch.cat([st["k_stage"][b, :, :old], st["k_new"][b][:, pick]], 1).double()
            v[b, :, old:old + c] = st["v_new"][b][:, pick].double()
            for g0 in range(0, old + c, G):
                x = keys[:, g0:g0 + G]
                low, high = x.amin(1), x.amax(1)
                sg = torch.clamp(high - low, min=float(np.float32(1e-8))) / 15.0
                s[b, :, (first + g0) // G], z[b, :, (first + g0) // G] = sg, -low / sg
        return dict(k=None, v=v, k_scale=s, k_zp=z, stage=None, lens=None)
    N, W, S, Hq = case["nodes"], case["window"], case["sinks"], case["q_heads"]
    per = Hq // H
    out = torch.zeros(B, Hq, N, D, dtype=torch.float64, device="cuda")
    tree = _tree(case) if kind == "tree" else None
    q = st["query"] if kind == "tree" else st["query"][:, :, None]
    for b in range(B):
        n = int(lens[b])
        k, v = _sequence64(st, b, n, H, D)
        t = np.arange(n)
        see = np.ones((N, n), bool)
        if W:
            mine = tree[b].sum(-1) if kind == "tree" else np.zeros(1, np.int64)
            see = (t[None] < S) | (t[None] >= n + mine[:, None] - W)
        if kind == "tree":
            see = np.concatenate([see, tree[b]], 1)
            k = torch.cat([k, st["k_draft"][b].double()], 1)
            v = torch.cat([v, st["v_draft"][b].double()], 1)
        hidden = torch.from_numpy(~see).cuda()
        for h in range(H):
            qh = q[b, h * per:(h + 1) * per].double().reshape(per * N, D)
            x = (qh @ k[h].T).reshape(per, N, -1).masked_fill(hidden, -math.inf)
            w = torch.softmax(x, -1)
            out[b, h * per:(h + 1) * per] = torch.matmul(w, v[h])
    return out if kind == "tree" else out[:, :, 0]
