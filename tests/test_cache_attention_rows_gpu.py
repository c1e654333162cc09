"""cache_attention_shared with first rows that do not ascend."""
import pytest

pytestmark = pytest.mark.gpu


def test_first_rows_that_do_not_ascend(torch_cuda, mxk):
    """cu_q that goes up and down, so that more sequences have a token than there are tokens: their
    lengths together are beyond 31 bits, and all of them say the same of row 0.  No list or
    workspace is left."""
    torch = torch_cuda
    seqs, heads, tokens = 1 << 17, 4096, 1 << 16
    cache = mxk.PagedCache.empty(1, 1024, heads, 64, 8)
    for t in (cache.k_values, cache.v_values):
        t.random_(0, 100)
    for t in (cache.k_scales, cache.v_scales):
        t.fill_(120)
    i32 = dict(dtype=torch.int32, device="cuda")
    cu = torch.arange(seqs + 1, **i32) % 2
    table = torch.zeros(seqs, tokens // 1024, **i32)
    q = torch.randn(2, heads, 64, device="cuda", dtype=torch.bfloat16)
    out, want = torch.full_like(q, 77.0), torch.full_like(q, 77.0)
    mxk.cache_attention_shared(cache, q, cu, table, torch.full((seqs,), tokens, **i32), torch.tensor([0, seqs], **i32),
                               torch.tensor([128], **i32), out, max_q=1, max_kv=tokens, max_prefix=tokens)
    mxk.cache_attention(cache, q, torch.tensor([0, 1], **i32), table[:1], torch.full((1,), tokens, **i32), want, max_q=1,
                        max_kv=tokens)
    torch.cuda.synchronize()
    # both within half a step of bfloat16 of values that differ by 2^-10 of their sizes at most
    assert (out[0].float() - want[0].float()).norm() <= 2.0 ** -7 * want[0].float().norm()
    assert (out[1] == 77.0).all()
