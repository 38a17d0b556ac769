"""What the host knows of a sequence cache's lengths when tokens were appended by counts on
the device or by graph replays."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D, H = 64, 2


def make(num_pages=64, max_seqs=2, max_seq_len=512):
    from flash_decode_int4.vllm_integration import INT4PagedSequenceCache
    return INT4PagedSequenceCache(num_pages, H, D, max_seqs, max_seq_len, 16, 64)


def tokens(n, B=2, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(B, H, n, D, device="cuda", generator=g)


def test_a_reservation_holds_what_was_accepted():
    """64 tokens are reserved; every round drafts 16 and accepts two: 24 rounds and then
    some fit (a count of 16 a round would end at the fourth)."""
    import torch
    cache = make()
    cache.reserve(2, 64)
    k = tokens(16)
    n = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    for _ in range(24):
        cache.extend(k, k, n)
    # 48 and 24 tokens: sixteen more could be taken, seventeen could not.
    q = torch.randn(2, H, D, device="cuda")
    cache.extend(k, k, torch.tensor([15, 3], dtype=torch.int32, device="cuda"))
    cache.step(k[:, :, 0], k[:, :, 0], q)
    with pytest.raises(RuntimeError, match="reserve"):
        cache.step(k[:, :, 0], k[:, :, 0], q)
    with pytest.raises(RuntimeError, match="reserve"):
        cache.extend(k, k, n)
    assert cache.seq_lens.tolist() == [64, 28] and cache.lengths().tolist() == [64, 28]
    cache.reserve(2, 16)
    cache.extend(k, k, n)
    assert cache.seq_lens.tolist() == [66, 29]


def test_in_a_capture_the_count_of_the_host_stands():
    """Nothing is read from the device while a graph is captured."""
    import torch
    cache = make()
    cache.reserve(2, 32)
    k = tokens(16)
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache.extend(k, k, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.extend(k, k, n)
        with pytest.raises(RuntimeError, match="reserve"):
            cache.extend(k, k, n)
    n.fill_(3)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert cache.seq_lens.tolist() == [3 * i + 3] * 2


@pytest.mark.parametrize("how", ["extend", "append", "reserve", "read"])
def test_replays_after_a_sync_are_seen(how):
    """Replays of a captured extend move the lengths after the host last read them: a call
    that maps pages or counts tokens on the host starts from the device's."""
    import torch
    cache = make()
    k = tokens(16)
    n = torch.tensor([16, 9], dtype=torch.int32, device="cuda")
    cache.extend(k, k)
    cache.reserve(2, 160)
    cache.extend(k, k, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.extend(k, k, n)
    cache.sync_lengths()
    for _ in range(8):
        graph.replay()
    used = [16 + 16 * 9, 16 + 9 * 9]
    big = tokens(70, seed=1)
    if how == "extend":
        cache.extend(big, big)
        new, want = 70, big
    elif how == "append":
        cache.append(k[:, :, 0], k[:, :, 0])
        new, want = 1, k[:, :, :1]
    elif how == "reserve":
        cache.reserve(2, 70)
        cache.extend(big, big, torch.full((2,), 70, dtype=torch.int32, device="cuda"))
        cache.sync_lengths()
        new, want = 70, big
    else:
        new, want = 0, None
    assert cache.read(2)[0].shape[2] == used[0] + new
    assert cache.seq_lens.tolist() == cache.lengths().tolist() == [u + new for u in used]
    pages = cache.page_table.cpu().numpy()
    held = [pages[b, i] for b in range(2) for i in range(-(-(used[b] + new) // 16))]
    assert len(set(held)) == len(held)
    for b in range(2):
        v = cache.read(2)[1][b, :, used[b]:used[b] + new]
        assert want is None or torch.equal(v, want[b, :, :new])
