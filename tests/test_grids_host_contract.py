"""Calls of more workgroups than a launch has threads for (2^32 - 1 along a dimension) are
refused before any device work (no pointer is followed)."""

import pytest

from test_attend_host_contract import attend
from test_rows_host_contract import INVALID, cache


@pytest.mark.parametrize("kw", [
    dict(B=65535, Hq=64, N=1, splits=16),          # few rows: 67 million workgroups of 256
    dict(B=65535, Hq=64, N=40, splits=4),          # many: 17 million of 512
    dict(B=1, Hq=64, N=1100000, splits=2)], ids=str)     # 70 million rows to merge
def test_attend(kw):
    assert attend(cache(num_kv_heads=64), wsb=1 << 50, **kw) == INVALID


def test_reads():
    import ctypes

    from flash_decode_int4 import capi
    from test_rows_host_contract import P
    c = cache(num_kv_heads=512)
    assert capi.load().fdi4_read_paged(
        ctypes.byref(c), 65535, None, 0, 1, P, 512 * 128, 128, 128, P, 512 * 128, 128, 128,
        capi.K_F32, None) == INVALID
