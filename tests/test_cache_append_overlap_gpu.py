"""Broadcast queries: rotated to rows of their own, refused in place."""
import pytest
from test_cache_append_gpu import table

pytestmark = pytest.mark.gpu


def test_broadcast_queries(torch_cuda, mxk):
    torch = torch_cuda
    tokens, heads = 5, 4
    cache = mxk.PagedCache.empty(2, 16, 2, 64, 8)
    q = torch.randn(1, heads, 64, device="cuda").half()
    k, v = (torch.randn(1, 1, 64, device="cuda").half().expand(tokens, 2, 64) for _ in range(2))
    cos_sin, at = table(torch, 64, 64), torch.arange(tokens, device="cuda")
    whole, out = q.repeat(tokens, 1, 1), torch.empty(tokens, heads, 64, device="cuda").half()
    mxk.cache_append(cache, q.expand(tokens, -1, -1), k, v, at, cos_sin, at, q_out=out)
    got = cache.k_values.clone(), cache.v_values.clone()
    for t in (cache.k_values, cache.v_values):
        t.zero_()
    want = whole.clone()
    mxk.cache_append(cache, want, k.contiguous(), v.contiguous(), at, cos_sin, at)
    assert torch.equal(out, want) and torch.equal(cache.k_values, got[0]) and torch.equal(cache.v_values, got[1])
    for bad in (dict(q=q.expand(tokens, -1, -1)), dict(q=whole, q_out=out[:1].expand(tokens, -1, -1)),
                dict(q=whole, q_out=out[:, :1].expand(-1, heads, -1))):
        with pytest.raises(mxk.MxkInvalidArgument):
            mxk.cache_append(cache, k=k, v=v, positions=at, cos_sin=cos_sin, slots=at, **bad)
    # one token, one head: any strides
    one = torch.empty(1, 1, 64, device="cuda").half()
    mxk.cache_append(cache, q[:, :1], k[:1], v[:1], at[:1], cos_sin, at[:1], q_out=one.as_strided((1, 1, 64), (0, 0, 1)))
    assert torch.equal(one, want[:1, :1])
