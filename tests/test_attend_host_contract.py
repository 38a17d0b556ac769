"""What the C entry points of the cached-chunk attention, the head norms with rotation and
the token log probabilities refuse: every rejected call returns hipErrorInvalidValue
before any device work, so these run without a GPU (no pointer is followed)."""

import ctypes

import pytest

from flash_decode_int4 import capi
from test_rows_host_contract import BAD_CACHES, INVALID, P, cache


def attend(c, q=P, qt=capi.K_BF16, B=2, Hq=8, N=5, counts=P, prefix=None, w=0, s=0, cap=0.0,
           slopes=None, out=P, ot=capi.K_BF16, splits=0, ws=P, wsb=1 << 40):
    return capi.load().fdi4_attend_paged(q, qt, B, Hq, N, Hq * 5 * 128, 5 * 128, 128,
                                         ctypes.byref(c), ctypes.byref(
                                             capi.AttendOptions(counts, prefix, slopes, w, s, cap)),
                                         out, ot, splits, ws, wsb, None)


def rotary(q=P, k=P, dt=capi.K_BF16, B=2, N=3, Hq=8, H=2, D=128, pos=P, pb=1, pt=0, inv=P, R=128,
           qw=P, kw=P, wd=capi.K_F32, eps=1e-6, qo=P, ko=P):
    return capi.load().fdi4_norm_rotary(q, k, dt, B, N, Hq, H, D, 4096, 512, 128, 4096, 512, 128,
                                        pos, pb, pt, ctypes.byref(
                                            capi.RotaryOptions(inv, qw, kw, wd, R, 0, eps, 1.0,
                                                               1.0)), qo, ko, None)


def logprobs(x=P, dt=capi.K_BF16, outer=2, inner=3, vocab=1000, tok=P, cap=0.0, top=5, lp=P,
             en=P, tl=P, ti=P):
    return capi.load().fdi4_token_logprobs(x, dt, outer, inner, 3000, 1000, vocab, tok,
                                           ctypes.byref(capi.LogprobOptions(top, cap)), lp, en,
                                           tl, ti, None)


@pytest.mark.parametrize("bad", BAD_CACHES + [dict(seq_lens=None), dict(pages_per_group=3),
                                              dict(max_pages=(1 << 26) + 1)], ids=str)
def test_caches_refused(bad):
    assert attend(cache(**bad)) == INVALID


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(qt=5), dict(B=0), dict(B=-1), dict(B=70000), dict(Hq=0), dict(Hq=7),
    dict(N=0), dict(N=-2), dict(N=1 << 28), dict(N=1 << 30), dict(w=-1), dict(s=-1), dict(s=3),
    dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(counts=P + 2),
    dict(prefix=P + 1), dict(slopes=P + 2), dict(out=None), dict(ot=-1),
    dict(splits=4, ws=None), dict(splits=4, wsb=100), dict(splits=4, ws=P + 8)], ids=str)
def test_attend_refused(kw):
    assert attend(cache(), **kw) == INVALID


def test_attend_workspace():
    lib, c = capi.load(), cache()

    def size(B, Hq, N, w, s, splits, c=c):
        return lib.fdi4_attend_workspace_bytes(
            B, Hq, N, capi.K_BF16, ctypes.byref(capi.AttendOptions(None, None, None, w, s, 0.0)), splits,
            ctypes.byref(c) if c else None)

    assert size(2, 8, 5, 0, 0, 1) == 0
    need = size(2, 8, 5, 0, 0, 4)
    assert need >= 2 * 8 * 5 * 4 * (128 * 4 + 16)
    assert attend(c, splits=4, wsb=need - 1) == INVALID
    for args in ((0, 8, 5, 0, 0, 4), (2, 7, 5, 0, 0, 4), (2, 8, 0, 0, 0, 4), (2, 8, 5, -1, 0, 4),
                 (2, 8, 5, 0, -1, 4), (2, 8, 1 << 30, 0, 0, 4)):
        assert size(*args) == 0
    assert size(2, 8, 5, 0, 0, 4, None) == 0
    assert lib.fdi4_attend_workspace_bytes(2, 8, 5, capi.K_BF16, None, 4, ctypes.byref(c)) == 0


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(k=None), dict(dt=3), dict(B=-1), dict(N=-1), dict(Hq=0), dict(H=0),
    dict(Hq=70000), dict(D=96), dict(pos=None), dict(pos=P + 2), dict(inv=None), dict(inv=P + 1),
    dict(R=0), dict(R=130), dict(R=63), dict(wd=9), dict(qw=P + 2), dict(kw=P + 1),
    dict(eps=-1e-6), dict(eps=float("nan")), dict(qo=None), dict(ko=None), dict(qo=P + 8),
    dict(ko=P + 4), dict(q=P + 1), dict(B=1 << 20, N=1 << 20), dict(B=60000, N=60000)], ids=str)
def test_rotary_refused(kw):
    assert rotary(**kw) == INVALID


def test_options_are_needed():
    lib, c = capi.load(), cache()
    assert lib.fdi4_attend_paged(P, capi.K_BF16, 2, 8, 5, 5120, 640, 128, ctypes.byref(c), None, P,
                                 capi.K_BF16, 0, P, 1 << 40, None) == INVALID
    assert lib.fdi4_norm_rotary(P, P, 0, 2, 3, 8, 2, 128, 0, 0, 0, 0, 0, 0, P, 1, 0, None, P, P,
                                None) == INVALID
    assert lib.fdi4_token_logprobs(P, 0, 2, 3, 3000, 1000, 1000, P, None, P, P, P, P,
                                   None) == INVALID


def test_nothing_to_do():
    assert rotary(B=0, q=None) == 0 and rotary(N=0, qo=None) == 0
    assert logprobs(outer=0, x=None) == 0 and logprobs(inner=0, lp=None) == 0


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(x=P + 1), dict(dt=4), dict(outer=-1), dict(inner=-1), dict(vocab=0),
    dict(tok=None), dict(tok=P + 4), dict(cap=-2.0), dict(cap=float("nan")), dict(top=-1),
    dict(top=65), dict(top=9, vocab=8), dict(lp=None), dict(en=None), dict(tl=None),
    dict(ti=None), dict(ti=P + 4), dict(outer=1 << 20, inner=1 << 20)], ids=str)
def test_logprobs_refused(kw):
    assert logprobs(**kw) == INVALID
