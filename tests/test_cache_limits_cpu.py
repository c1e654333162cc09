"""Limits of the paged MX cache's entry points, checked before anything touches a device."""
import ctypes

import pytest
from test_cache_cpu import make_args, make_cache


@pytest.mark.parametrize("sizes", [dict(pages=(1 << 31) - 1, kv_heads=2, page_size=16),
                                   dict(pages=1 << 16, kv_heads=32, page_size=1 << 12),
                                   dict(pages=(1 << 20) + 1, kv_heads=1, page_size=1 << 12),
                                   dict(pages=(1 << 31) - 1, kv_heads=65535, page_size=(1 << 31) - 16)], ids=str)
def test_more_rows_than_32_bits_number_are_refused(mxk, sizes):
    """No query tokens: what is not refused is nothing to do."""
    lib, args = mxk.load(), make_args(mxk, heads=sizes["kv_heads"], tokens=0)
    status = lib.mxk_cache_attention(ctypes.byref(make_cache(mxk, **sizes)), ctypes.byref(args), None)
    assert status == mxk.ERR_UNSUPPORTED


@pytest.mark.parametrize("sizes", [dict(pages=1 << 20, kv_heads=1, page_size=1 << 12),
                                   dict(pages=1 << 15, kv_heads=32, page_size=1 << 12)], ids=str)
def test_as_many_rows_as_32_bits_number_are_not(mxk, sizes):
    lib, args = mxk.load(), make_args(mxk, heads=sizes["kv_heads"], tokens=0)
    assert lib.mxk_cache_attention(ctypes.byref(make_cache(mxk, **sizes)), ctypes.byref(args), None) == mxk.OK
