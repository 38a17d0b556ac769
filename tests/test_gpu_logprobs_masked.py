"""Log probabilities of rows whose masked logits are the type's lowest value, of huge logits,
and of rows with many NaN. The oracle and its tolerances are test_gpu_logprobs.py's: no term
of the derivation there depends on how far a logit lies below the largest."""

import numpy as np
import pytest

from test_gpu_logprobs import check, make

pytestmark = pytest.mark.gpu


def masked(rows, vocab, dtype, value, kept, seed=0):
    """Rows of `value` but for the logits that `kept(row)` names."""
    import torch
    x, tok = make((rows,), vocab, dtype, seed=seed)
    y = torch.full_like(x, value)
    for r in range(rows):
        at = torch.as_tensor(sorted(kept(r)), device="cuda")
        y[r, at] = x[r, at]
        tok[r] = at[r % len(at)]
    return y, tok


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(3, 1000), (3, 70001), (300, 1003), (300, 20011)])
@pytest.mark.parametrize("top", [0, 3, 20])
def test_masks_of_the_lowest_value(rows, vocab, dtype, top):
    """A few allowed tokens of a vocabulary, in one and in several segments of a row's
    threads, of 1024 and of 256 threads."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    low = torch.finfo(getattr(torch, dtype)).min
    for value in (low, low / 4):
        x, tok = masked(rows, vocab, dtype, value,
                        lambda r: {(7 * r + 1) % vocab, vocab // 2, (13 * r + 5) % vocab,
                                   vocab - 1 - r, vocab - 2})
        check(token_logprobs(x, tok, top), x, tok, top)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("tail", [1, 8, 990])
def test_a_masked_part_of_a_row(tail, rows, dtype):
    """Behind or before usual logits, some masked ones (one thread's at the least)."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    low = torch.finfo(getattr(torch, dtype)).min
    for vocab in (1000, 40000):
        for part in (slice(vocab - tail, vocab), slice(0, tail)):
            kept = set(range(vocab)) - set(range(vocab)[part])
            x, tok = make((rows,), vocab, dtype)
            x[:, part] = low
            tok[:] = min(kept)
            check(token_logprobs(x, tok, 2), x, tok, 2)
            # Masked so, a cap lets them count.
            check(token_logprobs(x, tok, 2, logit_cap=5.0), x, tok, 2, 5.0)


@pytest.mark.parametrize("rows,vocab", [(3, 700), (300, 20011)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_huge_logits(rows, vocab, dtype):
    """One logit far above all: probability one, an entropy of zero."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    for size in (2e31, 1e38, float(torch.finfo(getattr(torch, dtype)).max)):
        x, tok = make((rows,), vocab, dtype)
        at = (torch.arange(rows, device="cuda") * 37 + 11) % vocab
        x[torch.arange(rows, device="cuda"), at] = size
        out = token_logprobs(x, at, 1)
        assert not out.logprobs.any() and not out.entropy.any()
        assert torch.equal(out.top_ids[:, 0], at) and not out.top_logprobs.any()


@pytest.mark.parametrize("rows,vocab", [(3, 700), (3, 5000), (300, 5000), (2, 40000)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_nan_at_the_front_of_many_candidates(rows, vocab, dtype):
    """NaN first, ties to the lowest index, also where a row has more NaN or equal logits
    than are ranked at once."""
    import torch
    from flash_decode_int4.quality import token_logprobs
    nan = float("nan")
    tok = torch.zeros(rows, dtype=torch.long, device="cuda")
    for seen, first in ((slice(None), []), (slice(0, 1), [0]), ([0, 17, vocab - 1], [0, 17, vocab - 1]),
                        (slice(1, None, 2), list(range(1, vocab, 2)))):
        x = torch.zeros(rows, vocab, device="cuda", dtype=getattr(torch, dtype))
        x[:, seen] = nan
        rest = [i for i in range(200) if i not in set(first[:200])]
        want = (first + rest)[:64]
        for top in (1, 5, 64):
            out = token_logprobs(x, tok, top)
            assert (out.top_ids.cpu().numpy() == np.array(want[:top])).all()
            assert torch.isnan(out.top_logprobs).all() and torch.isnan(out.entropy).all()
