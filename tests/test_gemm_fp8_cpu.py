"""Refusals of the E4M3 quantiser and products: bad arguments come back as MXK_ERR_INVALID
before anything touches a device."""
import pytest

BUF = 0x7f0000000000  # a plausible, aligned address; nothing here reads it


def quantize(mxk, **kw):
    f = dict(dtype=mxk.BF16, rows=3, k=64, x=BUF, row_stride=64, block_rows=1, values=BUF, scales=BUF)
    f.update(kw)
    return mxk.load().mxk_quantize_fp8(*f.values(), None)


def gemm(mxk, **kw):
    f = dict(dtype=mxk.BF16, m=3, n=5, k=64, a=BUF, a_scales=BUF, b=BUF, b_scales=BUF, out=BUF, out_stride=5)
    f.update(kw)
    return mxk.load().mxk_gemm_fp8(*f.values(), None)


def linear(mxk, **kw):
    f = dict(dtype=mxk.BF16, m=3, n=5, k=64, x=BUF, x_stride=64, b=BUF, b_scales=BUF, out=BUF, out_stride=5)
    f.update(kw)
    return mxk.load().mxk_linear_fp8(*f.values(), None)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(k=-16), dict(k=40), dict(k=1 << 30),
                                 dict(block_rows=0), dict(block_rows=64), dict(x=None), dict(values=None),
                                 dict(scales=None), dict(x=BUF + 1), dict(values=BUF + 8), dict(scales=BUF + 2),
                                 dict(rows=1 << 50), dict(rows=1 << 24, block_rows=128)], ids=str)
def test_bad_quantisations_are_refused(mxk, bad):
    assert quantize(mxk, **bad) == mxk.ERR_INVALID
    assert b"quantize_fp8" in mxk.load().mxk_last_error()


BAD = [dict(dtype=3), dict(dtype=-1), dict(m=-1), dict(n=-1), dict(k=-16), dict(k=24), dict(m=1 << 30),
       dict(n=1 << 30, out_stride=1 << 30), dict(k=1 << 30), dict(b=None), dict(b_scales=None), dict(out=None),
       dict(b=BUF + 8), dict(b_scales=BUF + 2), dict(out=BUF + 1), dict(out_stride=4), dict(out_stride=-5)]


@pytest.mark.parametrize("bad", BAD + [dict(a=None), dict(a_scales=None), dict(a=BUF + 8), dict(a_scales=BUF + 1)], ids=str)
def test_bad_products_are_refused(mxk, bad):
    assert gemm(mxk, **bad) == mxk.ERR_INVALID
    assert b"gemm_fp8" in mxk.load().mxk_last_error()


@pytest.mark.parametrize("bad", BAD + [dict(x=None), dict(x=BUF + 1)], ids=str)
def test_bad_layers_are_refused(mxk, bad):
    assert linear(mxk, **bad) == mxk.ERR_INVALID
    assert b"linear_fp8" in mxk.load().mxk_last_error()


def test_nothing_to_do(mxk):
    assert quantize(mxk, rows=0, x=None, values=None, scales=None) == mxk.OK
    assert quantize(mxk, k=0, x=None, values=None, scales=None) == mxk.OK
    for size in (dict(m=0), dict(n=0)):
        assert gemm(mxk, **size, a=None, a_scales=None, b=None, b_scales=None, out=None) == mxk.OK
        assert linear(mxk, **size, x=None, b=None, b_scales=None, out=None) == mxk.OK
