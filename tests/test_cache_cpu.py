"""Refusals of the paged MX cache's entry points: bad arguments come back as
MXK_ERR_INVALID / MXK_ERR_UNSUPPORTED before anything touches a device."""
import ctypes

import pytest

BUF = 0x7f0000000000  # a plausible, aligned address; nothing here reads it


def ref(x):
    return ctypes.byref(x)


def make_cache(mxk, **kw):
    f = dict(bits=8, kv_heads=2, head_dim=128, page_size=64, pages=10, k_values=BUF, k_scales=BUF, v_values=BUF,
             v_scales=BUF)
    f.update(kw)
    return mxk.Cache(**f)


def make_args(mxk, **kw):
    rows = mxk.Rows(BUF, 512, 128)
    f = dict(dtype=mxk.BF16, heads=4, tokens=3, seqs=2, max_q=2, max_kv=100, q=rows, cu_q=BUF, page_table=BUF,
             page_table_stride=2, kv_lens=BUF, scale=0.1, causal=1, window=0, out=rows, lse=None)
    f.update(kw)
    return mxk.Attention(**f)


BAD_CACHE = [dict(bits=5), dict(bits=0), dict(head_dim=0), dict(head_dim=48), dict(head_dim=544), dict(page_size=0),
             dict(page_size=8), dict(page_size=40), dict(kv_heads=0), dict(kv_heads=70000), dict(pages=0),
             dict(pages=-3), dict(pages=1 << 31), dict(k_values=None), dict(v_scales=None), dict(k_values=BUF + 8),
             dict(v_scales=BUF + 1)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_cache_is_refused(mxk, bad):
    lib = mxk.load()
    c = make_cache(mxk, **bad)
    rows = mxk.Rows(BUF, 256, 128)
    for st in (lib.mxk_cache_write(ref(c), mxk.BF16, 1, ref(rows), ref(rows), BUF, None),
               lib.mxk_cache_read(ref(c), mxk.BF16, 1, BUF, ref(rows), ref(rows), None),
               lib.mxk_cache_attention(ref(c), ref(make_args(mxk)), None)):
        assert st == mxk.ERR_INVALID
        assert lib.mxk_last_error()


def test_bad_moves_are_refused(mxk):
    lib = mxk.load()
    c = make_cache(mxk)
    rows, none, odd = (ref(mxk.Rows(at, 256, 128)) for at in (BUF, None, BUF + 1))
    for args in ((3, 1, rows, rows, BUF), (-1, 1, rows, rows, BUF), (mxk.F16, -1, rows, rows, BUF),
                 (mxk.F16, 1, none, rows, BUF), (mxk.F16, 1, rows, none, BUF), (mxk.F16, 1, rows, rows, None),
                 (mxk.F16, 1, odd, rows, BUF), (mxk.F32, 1, rows, ref(mxk.Rows(BUF + 2, 256, 128)), BUF),
                 (mxk.F16, 1, rows, rows, BUF + 4), (mxk.F16, 1, None, rows, BUF)):
        dtype, tokens, k, v, slots = args
        assert lib.mxk_cache_write(ref(c), dtype, tokens, k, v, slots, None) == mxk.ERR_INVALID
        assert lib.mxk_cache_read(ref(c), dtype, tokens, slots, k, v, None) == mxk.ERR_INVALID
    assert lib.mxk_cache_write(None, mxk.F16, 1, rows, rows, BUF, None) == mxk.ERR_INVALID
    # nothing to do: no pointer is looked at
    assert lib.mxk_cache_write(ref(c), mxk.F16, 0, None, None, None, None) == mxk.OK
    assert lib.mxk_cache_read(ref(c), mxk.F16, 0, None, None, None, None) == mxk.OK


BAD_ATTENTION = [dict(dtype=0), dict(dtype=7), dict(heads=0), dict(heads=3), dict(heads=-2), dict(tokens=-1),
                 dict(tokens=1 << 30), dict(seqs=-1), dict(max_q=-1), dict(max_kv=-1), dict(max_q=1 << 30),
                 dict(max_kv=1 << 31), dict(window=-1), dict(window=5, causal=0), dict(scale=float("nan")),
                 dict(scale=float("inf")), dict(cu_q=None), dict(page_table=None), dict(kv_lens=None),
                 dict(cu_q=BUF + 2), dict(lse=BUF + 2), dict(page_table_stride=1)]


@pytest.mark.parametrize("bad", BAD_ATTENTION, ids=str)
def test_bad_attention_is_refused(mxk, bad):
    assert mxk.load().mxk_cache_attention(ref(make_cache(mxk)), ref(make_args(mxk, **bad)), None) == mxk.ERR_INVALID


def test_bad_attention_rows_are_refused(mxk):
    lib, c = mxk.load(), make_cache(mxk)
    for rows in (mxk.Rows(None, 512, 128), mxk.Rows(BUF + 1, 512, 128)):
        assert lib.mxk_cache_attention(ref(c), ref(make_args(mxk, q=rows)), None) == mxk.ERR_INVALID
        assert lib.mxk_cache_attention(ref(c), ref(make_args(mxk, out=rows)), None) == mxk.ERR_INVALID
    assert lib.mxk_cache_attention(ref(c), None, None) == mxk.ERR_INVALID


@pytest.mark.parametrize("dim", [32, 96, 160, 256])
def test_other_head_dims_are_unsupported(mxk, dim):
    st = mxk.load().mxk_cache_attention(ref(make_cache(mxk, head_dim=dim)), ref(make_args(mxk)), None)
    assert st == mxk.ERR_UNSUPPORTED


@pytest.mark.parametrize("nothing", [dict(tokens=0), dict(seqs=0), dict(max_q=0)], ids=str)
def test_no_queries_is_nothing_to_do(mxk, nothing):
    args = make_args(mxk, q=mxk.Rows(None, 0, 0), out=mxk.Rows(None, 0, 0), cu_q=None, page_table=None, kv_lens=None,
                     **nothing)
    assert mxk.load().mxk_cache_attention(ref(make_cache(mxk)), ref(args), None) == mxk.OK


def test_binding_refuses_host_and_misshapen_tensors(mxk):
    import torch
    u8 = torch.uint8
    k, s = torch.zeros(3, 2, 16, 64, dtype=u8), torch.zeros(3, 2, 16, 2, dtype=u8)
    for bits in (5, 8):  # no such format; host tensors
        with pytest.raises(mxk.MxkInvalidArgument):
            mxk.PagedCache(k, s, k, s, bits)
    with pytest.raises(mxk.MxkInvalidArgument):
        mxk.PagedCache(k[0], s[0], k[0], s[0], 8)
