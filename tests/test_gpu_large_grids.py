"""More rows than one launch has threads for (2^32 - 1): log probabilities of 17 million rows, the
rotation of 67 million heads. The tail of a large call against a call of the tail alone, bit by
bit (a row's result depends on the row and its alignment)."""

import pytest

pytestmark = pytest.mark.gpu


def test_rows_of_logits():
    import torch
    from flash_decode_int4.quality import token_logprobs
    rows, vocab = (1 << 24) + 1003, 3
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(rows, vocab, device="cuda", generator=g)
    tok = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    out = token_logprobs(x, tok, 2)
    ref = torch.log_softmax(x.double(), -1)
    # (Four logits below 6 in size: a handful of roundings of numbers below 16.)
    assert float((out.logprobs - ref.gather(1, tok[:, None])[:, 0]).abs().max()) < 16 * 2.0 ** -20
    assert torch.equal(out.top_ids, x.sort(dim=1, descending=True, stable=True).indices[:, :2])
    for at in (slice(0, 300), slice(rows - 1503, rows)):
        # (Four rows on: the order of a row's sums goes by where it lies between 16 bytes.)
        assert at.start % 4 == 0
        part = token_logprobs(x[at].repeat(2, 1), tok[at].repeat(2), 2)
        for a, b in zip(out, part):
            assert bool(torch.equal(a[at], b[:len(a[at])]))


@pytest.mark.parametrize("R,N,Hq,H", [(2, (1 << 21) + 77, 31, 1),         # a wave a head
                                      (64, (1 << 26) + 77, 1, 1)])        # a wave a token
def test_heads(R, N, Hq, H):
    import torch
    from flash_decode_int4 import ops
    D = 64
    q = torch.empty(1, Hq, N, D, dtype=torch.bfloat16, device="cuda").normal_()
    k = torch.empty(1, H, N, D, dtype=torch.bfloat16, device="cuda").normal_()
    inv = (10000.0 ** (-torch.arange(0, R, 2, device="cuda") / R)).float()
    start = torch.tensor([5], dtype=torch.int32, device="cuda")
    w = torch.rand(D, device="cuda")
    a = ops.norm_rotary(q, k, start, inv, w, w)
    for at in (0, N // 2, N - 1000):
        b = ops.norm_rotary(q[:, :, at:at + 1000], k[:, :, at:at + 1000], start + at, inv, w, w)
        for x, y in zip(a, b):
            assert bool(torch.equal(x[:, :, at:at + 1000], y))


def test_packed_and_dequantized_elements():
    import torch
    from flash_decode_int4 import ops
    C, rows = 128, (1 << 26) + 1003                 # 2^33 values, 2^32 bytes of them
    q = torch.empty(rows, C, dtype=torch.uint8, device="cuda").random_(0, 16)
    p = ops.pack_int4_device(q)
    for at in (slice(0, 1000), slice(rows // 2, rows // 2 + 1000), slice(rows - 2000, rows)):
        assert bool(torch.equal(p[at], q[at, 0::2] | q[at, 1::2] << 4))
    del q
    s, z = (torch.rand(C, device="cuda") for _ in range(2))
    x = ops.dequantize_int4(p, s, z, packed=True)
    assert tuple(x.shape) == (rows, C)
    for at in (slice(0, 1000), slice(rows // 2, rows // 2 + 1000), slice(rows - 2000, rows)):
        assert bool(torch.equal(x[at], ops.dequantize_int4(p[at].contiguous(), s, z, packed=True)))
