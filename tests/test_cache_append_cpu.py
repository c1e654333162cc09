"""Refusals of mxk_cache_append: bad arguments come back as MXK_ERR_INVALID before anything
touches a device."""
import ctypes

import pytest

BUF = 0x7f0000000000  # a plausible, aligned address; nothing here reads it


def make_cache(mxk, **kw):
    f = dict(bits=8, kv_heads=2, head_dim=128, page_size=64, pages=10, k_values=BUF, k_scales=BUF, v_values=BUF,
             v_scales=BUF)
    f.update(kw)
    return mxk.Cache(**f)


def make_args(mxk, **kw):
    rows = mxk.Rows(BUF, 512, 128)
    f = dict(dtype=mxk.BF16, heads=4, tokens=3, q=rows, q_out=rows, k=rows, v=rows, slots=BUF, positions=BUF,
             cos_sin=BUF, table_rows=100, rot_dim=128, interleaved=0)
    f.update(kw)
    return mxk.Append(**f)


def call(mxk, cache, args):
    return mxk.load().mxk_cache_append(ctypes.byref(cache), None if args is None else ctypes.byref(args), None)


BAD = [dict(dtype=3), dict(dtype=-1), dict(heads=-1), dict(heads=65536), dict(tokens=-1), dict(rot_dim=0),
       dict(rot_dim=-16), dict(rot_dim=24), dict(rot_dim=144), dict(table_rows=-1), dict(slots=None),
       dict(positions=None), dict(cos_sin=None), dict(slots=BUF + 4), dict(positions=BUF + 4), dict(cos_sin=BUF + 8)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_bad_arguments_are_refused(mxk, bad):
    assert call(mxk, make_cache(mxk), make_args(mxk, **bad)) == mxk.ERR_INVALID
    assert b"cache_append" in mxk.load().mxk_last_error()


@pytest.mark.parametrize("side", ["q", "q_out", "k", "v"])
@pytest.mark.parametrize("at", [None, BUF + 1])
def test_bad_rows_are_refused(mxk, side, at):
    assert call(mxk, make_cache(mxk), make_args(mxk, **{side: mxk.Rows(at, 512, 128)})) == mxk.ERR_INVALID


@pytest.mark.parametrize("bad", [dict(bits=5), dict(head_dim=48), dict(page_size=40), dict(pages=0),
                                 dict(k_values=BUF + 8)], ids=str)
def test_bad_caches_are_refused(mxk, bad):
    assert call(mxk, make_cache(mxk, **bad), make_args(mxk)) == mxk.ERR_INVALID


def test_null_arguments_and_nothing_to_do(mxk):
    assert call(mxk, make_cache(mxk), None) == mxk.ERR_INVALID
    assert mxk.load().mxk_cache_append(None, ctypes.byref(make_args(mxk)), None) == mxk.ERR_INVALID
    nothing = make_args(mxk, tokens=0, slots=None, positions=None, cos_sin=None, q=mxk.Rows(), q_out=mxk.Rows(),
                        k=mxk.Rows(), v=mxk.Rows())
    assert call(mxk, make_cache(mxk), nothing) == mxk.OK
