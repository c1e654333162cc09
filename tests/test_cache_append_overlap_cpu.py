"""mxk_cache_append writes no queries to rows that lie over each other; reading such is fine."""
import pytest
from test_cache_append_cpu import BUF, call, make_args, make_cache


def rows(mxk, token_stride, head_stride):
    return mxk.Rows(BUF, token_stride, head_stride)


@pytest.mark.parametrize("token_stride,head_stride", [(0, 128), (512, 0), (0, 0), (64, 128), (512, 127), (-64, 128), (512, -1)])
def test_rows_over_each_other_are_refused(mxk, token_stride, head_stride):
    over = rows(mxk, token_stride, head_stride)
    for args in (dict(q=over, q_out=over), dict(q_out=over)):
        assert call(mxk, make_cache(mxk), make_args(mxk, **args)) == mxk.ERR_INVALID
        assert b"overlap" in mxk.load().mxk_last_error()
