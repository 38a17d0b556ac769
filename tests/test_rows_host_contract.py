"""What the C entry points of the windowed and tree attention, the multi-token write and
the read refuse: every rejected call returns hipErrorInvalidValue before any device
work, so these run without a GPU (no pointer is followed)."""

import ctypes

import pytest

from flash_decode_int4 import capi

INVALID = 1
P = 1 << 20     # a 16-byte aligned address that nothing reads


def cache(**kw):
    c = capi.PagedCache()
    vals = dict(k_pages=P, k_page_stride=2 * 16 * 64, k_head_stride=16 * 64, k_row_stride=64,
                v_pages=P, v_dtype=capi.V_F16, v_page_stride=2 * 16 * 128,
                v_head_stride=16 * 128, v_row_stride=128, k_scale=P, k_zp=P,
                s_batch_stride=2 * 8 * 128, s_head_stride=8 * 128, s_group_stride=128,
                s_page_stride=0, page_table=P, pt_batch_stride=64, seq_lens=P, page_lens=None,
                pl_batch_stride=0, num_kv_heads=2, head_dim=128, page_rows=16,
                pages_per_group=8, max_pages=64, num_pages=200)
    vals.update(kw)
    for k, v in vals.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [dict(k_pages=None), dict(v_pages=None), dict(k_scale=None), dict(k_zp=None),
              dict(head_dim=96), dict(page_rows=0), dict(pages_per_group=0), dict(num_pages=0),
              dict(k_row_stride=32), dict(v_row_stride=64), dict(v_dtype=7),
              dict(k_pages=P + 4), dict(v_pages=P + 8), dict(k_scale=P + 4),
              dict(max_pages=1 << 30), dict(s_page_stride=128, pages_per_group=1),
              dict(page_lens=P)]


def window(c, q=P, qt=capi.K_F16, B=2, Hq=8, qb=1024, qh=128, w=64, s=4, out=P, ot=capi.K_F16,
           splits=0, ws=P, wsb=1 << 40, lens_out=None):
    return capi.load().fdi4_decode_window(q, qt, B, Hq, qb, qh, ctypes.byref(c), w, s, out, ot,
                                          splits, ws, wsb, lens_out, None)


def tree(c, q=P, qt=capi.K_F16, B=2, Hq=8, N=5, kd=P, vd=P, kdn=128, vdn=128, mask=P, w=0, s=0,
         out=P, ot=capi.K_F16, splits=0, ws=P, wsb=1 << 40):
    return capi.load().fdi4_decode_tree(q, qt, B, Hq, N, 8 * 5 * 128, 5 * 128, 128, kd,
                                        2 * 5 * 128, 5 * 128, kdn, vd, 2 * 5 * 128, 5 * 128, vdn,
                                        mask, 25, 5, ctypes.byref(c), w, s, out, ot, splits, ws,
                                        wsb, None)


def extend(c, k=P, v=P, B=2, N=5, counts=P, kr=128, vr=128, stage=P, G=128, nxt=2 * P):
    return capi.load().fdi4_extend_paged(k, 1280, 640, kr, v, 1280, 640, vr, B, N, counts, None,
                                         0, stage, 2 * 128 * 128, 128 * 128, 128, G,
                                         ctypes.byref(c), nxt, None)


def read(c, B=2, start=None, start0=0, n=10, k=P, v=P, kr=128, vr=128, dt=capi.K_F32):
    return capi.load().fdi4_read_paged(ctypes.byref(c), B, start, start0, n, k, 2 * 10 * 128,
                                       10 * 128, kr, v, 2 * 10 * 128, 10 * 128, vr, dt, None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: "-".join(f"{k}={v}" for k, v in
                                                                   d.items()))
def test_caches_refused(bad):
    c = cache(**bad)
    assert window(c) == INVALID
    assert tree(c) == INVALID
    assert read(c) == INVALID
    if "page_lens" not in bad:
        assert extend(c) == INVALID


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(qt=5), dict(B=0), dict(B=-1), dict(B=70000), dict(Hq=0), dict(Hq=7),
    dict(w=0), dict(w=-3), dict(s=-1), dict(out=None), dict(ot=9), dict(lens_out=P),
    dict(lens_out=P + 2)])
def test_window_refused(kw):
    assert window(cache(), **kw) == INVALID


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(qt=-1), dict(N=0), dict(N=capi.MAX_NODES + 1), dict(Hq=3), dict(kd=None),
    dict(vd=None), dict(mask=None), dict(kd=P + 4), dict(vd=P + 8), dict(kdn=130), dict(vdn=132),
    dict(w=4), dict(w=-1), dict(s=2), dict(w=64, s=-1), dict(out=None), dict(ot=3)])
def test_tree_refused(kw):
    assert tree(cache(), **kw) == INVALID


@pytest.mark.parametrize("kw", [
    dict(k=None), dict(v=None), dict(k=P + 4), dict(v=P + 4), dict(B=-1), dict(N=-1),
    dict(counts=None), dict(stage=None), dict(kr=130), dict(vr=130), dict(G=96), dict(G=64),
    dict(nxt=None), dict(nxt=P), dict(nxt=P + 4), dict(N=2 ** 31 - 1)])
def test_extend_refused(kw):
    assert extend(cache(), **kw) == INVALID


@pytest.mark.parametrize("kw", [
    dict(B=-1), dict(start0=-1), dict(n=-1), dict(k=None), dict(v=None), dict(k=P + 4),
    dict(v=P + 8), dict(kr=130), dict(vr=130), dict(dt=4), dict(start0=2 ** 31 - 5, n=2),
    dict(n=2 ** 31 - 1)])
def test_read_refused(kw):
    assert read(cache(), **kw) == INVALID


def test_workspace_refused_when_too_small():
    lib = capi.load()
    c = cache(max_pages=4096, pt_batch_stride=4096, s_head_stride=512 * 128,
              s_batch_stride=2 * 512 * 128)
    need = lib.fdi4_decode_rows_workspace_bytes(2, 8, 5, 0, 0, 4, ctypes.byref(c))
    if need:
        assert tree(c, splits=4, wsb=need - 1) == INVALID
        assert tree(c, splits=4, ws=None) == INVALID
        assert tree(c, splits=4, ws=P + 8) == INVALID


def test_python_arguments_refused():
    from flash_decode_int4 import ops
    for args in ((None, 1), (0, 0), (-4, 0), (5, -1)):
        with pytest.raises(ValueError):
            ops._check_window(*args)
    with pytest.raises(ValueError):
        ops._check_window(7, 0, 8)
    ops._check_window(None, 0)
    ops._check_window(8, 100, 8)


@pytest.mark.parametrize("bad", [
    dict(max_pages=(1 << 26) + 1), dict(k_page_stride=1 << 32), dict(k_page_stride=-1024),
    dict(v_page_stride=1 << 31), dict(v_page_stride=-1024), dict(s_group_stride=1 << 32),
    dict(s_group_stride=-128)],
    ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_sizes_beyond_the_attentions_32_bits_refused(bad):
    c = cache(**bad)
    assert window(c) == INVALID
    assert tree(c) == INVALID


def test_python_windows_beyond_32_bits_refused():
    from flash_decode_int4 import ops
    for args in ((2 ** 31, 0), (8, 2 ** 31)):
        with pytest.raises(ValueError):
            ops._check_window(*args)
    for args in ((8.5, 0), (8, 1.0)):
        with pytest.raises(TypeError):
            ops._check_window(*args)
