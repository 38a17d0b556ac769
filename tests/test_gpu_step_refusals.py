"""A step that is refused leaves the cache and its reservation as they were: nothing is
appended, and the steps reserved before are still there."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B, H, HQ, D = 2, 2, 4, 64


def setup():
    import torch
    from flash_decode_int4.vllm_integration import INT4PagedSequenceCache
    cache = INT4PagedSequenceCache(40, H, D, B, 256, value_dtype="float32")
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(B, H, 30, D, device="cuda", generator=g) for _ in range(2))
    cache.extend(k, v)
    cache.reserve(B, 2)          # (Two of a page's sixteen: 32 tokens.)
    one = [torch.randn(B, h, D, device="cuda", generator=g) for h in (H, H, HQ)]
    return cache, one


PATHS = [dict(), dict(num_splits=2), dict(window=9), dict(logit_cap=5.0), dict(logit_cap=5.0, window=9)]


@pytest.mark.parametrize("path", PATHS, ids=str)
def test_refused_steps_leave_the_cache(path):
    import torch
    cache, (k, v, q) = setup()
    names = ("seq_lens", "k_pages", "v_pages", "k_scale", "k_zp", "k_stage", "_lens_next")
    before = {n: getattr(cache, n).clone() for n in names}
    bad = [((k, v, q), dict(num_splits="two")), ((k, v, q), dict(num_splits=[3])),
           ((k.half(), v, q), {}), ((k, v.half(), q), {}), ((k, v[:, :1], q), {}),
           ((k, v, q.double()), {}), ((k, v, q[:, :3]), {}), ((k, v, q[:1]), {})]
    if path:
        bad += [((k, v, torch.randn(B, HQ, 2 * D, device="cuda")[..., ::2]), {}),
                ((k, v, q.cpu()), {}), ((k, v, q.unsqueeze(2)), {})]
    for args, kw in bad:
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            cache.step(*args, **{**path, **kw})
        for n in names:
            same = bool(torch.equal(getattr(cache, n), before[n]))
            assert same, (n, kw)
    # Both steps that were reserved are still there, and not one more.
    for _ in range(2):
        assert torch.isfinite(cache.step(k, v, q, **path)).all()
    with pytest.raises(RuntimeError):
        cache.step(k, v, q, **path)
    cache.sync_lengths()
    assert cache.lengths()[:B].tolist() == [32, 32]
    assert np.array_equal(cache.seq_lens.cpu().numpy(), [32, 32])
