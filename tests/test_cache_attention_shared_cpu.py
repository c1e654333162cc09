"""Refusals of mxk_cache_attention_shared: bad arguments come back as MXK_ERR_INVALID or
MXK_ERR_UNSUPPORTED before anything touches a device."""
import ctypes

import pytest

from test_cache_cpu import BAD_ATTENTION, BAD_CACHE, BUF, make_args, make_cache, ref


def call(mxk, cache=None, args=None, none=False, **kw):
    f = dict(groups=1, cu_groups=BUF, prefix_lens=BUF, max_prefix=64)
    f.update(kw)
    prefixes = None if none else ref(mxk.Prefixes(**f))
    return mxk.load().mxk_cache_attention_shared(ref(cache or make_cache(mxk)), ref(args or make_args(mxk)), prefixes, None)


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches_are_refused(mxk, bad):
    assert call(mxk, cache=make_cache(mxk, **bad)) == mxk.ERR_INVALID


@pytest.mark.parametrize("bad", BAD_ATTENTION, ids=str)
def test_bad_attention_is_refused(mxk, bad):
    assert call(mxk, args=make_args(mxk, **bad)) == mxk.ERR_INVALID
    assert b"cache_attention_shared" in mxk.load().mxk_last_error()


@pytest.mark.parametrize("bad", [dict(none=True), dict(groups=-1), dict(groups=1 << 30), dict(max_prefix=-1),
                                 dict(cu_groups=None), dict(prefix_lens=None), dict(cu_groups=BUF + 2),
                                 dict(prefix_lens=BUF + 1)], ids=str)
def test_bad_prefixes_are_refused(mxk, bad):
    assert call(mxk, **bad) == mxk.ERR_INVALID
    assert b"cache_attention_shared" in mxk.load().mxk_last_error()


def test_windows_and_sizes_are_refused(mxk):
    assert call(mxk, args=make_args(mxk, window=64)) == mxk.ERR_INVALID
    assert call(mxk, args=make_args(mxk, tokens=1 << 29, heads=4)) == mxk.ERR_INVALID
    assert call(mxk, cache=make_cache(mxk, head_dim=96)) == mxk.ERR_UNSUPPORTED
    assert mxk.load().mxk_cache_attention_shared(ctypes.byref(make_cache(mxk)), None, None, None) == mxk.ERR_INVALID


def test_nothing_to_do(mxk):
    assert call(mxk, args=make_args(mxk, tokens=0, q=mxk.Rows(), out=mxk.Rows(), cu_q=None), cu_groups=None) == mxk.OK
