"""Which calls of cache_attention_shared share, by the sizes and bounds that they are given, and
that both ways give the same.  A call that shares launches attention_merge, others do not."""
import numpy as np
import pytest
from test_cache_attention_gpu import check
from test_cache_attention_shared_gpu import attend, build

pytestmark = pytest.mark.gpu


def shares(torch, mxk, b, **kw):
    """The call's result, and whether it shared."""
    mxk.profile_enable()
    out, lse = attend(torch, mxk, b, **kw)
    names = mxk.profile_read()
    mxk.profile_enable(False)
    shared = "attention_merge" in names
    assert shared == ("attention_parts" in names) and ("attention_join" in names) != shared
    return out, lse, shared


def ordinary(torch, mxk, b):
    out = torch.full_like(b["q"], 77.0)
    mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], out, max_q=max(b["q_lens"]), max_kv=max(b["kv_lens"]))
    return out


# (heads, key heads, features, sequences, new tokens each, prefix of the call that does not, of the one that does)
AROUND = [
    (32, 32, 64, 2, 1, 8192, 12288),     # up to 32 rows a key head: a sequence's pass is saved
    (8, 8, 128, 40, 1, 896, 1024),       # single tokens
    (8, 2, 128, 8, 40, 5120, 8192),      # rows of two tiles each
    (8, 2, 128, 5, 70, 4096, 8320),      # rows that are converted for
    (4, 2, 128, 4, 600, 8192, 17024),    # the same, long chunks
]


@pytest.mark.parametrize("heads,kv_heads,dim,seqs,new,below,above", AROUND)
@pytest.mark.parametrize("bits", [8, 4])
def test_tight_bounds_on_both_sides(torch_cuda, mxk, bits, heads, kv_heads, dim, seqs, new, below, above):
    torch, g = torch_cuda, np.random.default_rng(1)
    for prefix in (below, above):
        b = build(torch, mxk, g, [(prefix, prefix, [(new, new + 5 * i) for i in range(seqs)])], heads, kv_heads, dim, 64, bits,
                  "bfloat16")
        out, lse, shared = shares(torch, mxk, b, tight=True)
        assert shared == (prefix == above)
        check(torch, b, out, lse)
        if not shared:
            assert torch.equal(out, ordinary(torch, mxk, b))


@pytest.mark.parametrize("heads,seqs,new,prefix", [(32, 2, 64, 16384), (32, 8, 2048, 1024), (32, 4, 2048, 4096),
                                                   (32, 64, 128, 512)])
def test_long_chunks_do_not_share_short_prefixes(torch_cuda, mxk, heads, seqs, new, prefix):
    """What sharing saves is less than the rows' way through float32; or one row tile a sequence."""
    torch = torch_cuda
    cache = mxk.PagedCache.empty(prefix // 64 + seqs * (new // 64), 64, 8, 128, 8)
    for t in (cache.k_values, cache.v_values):
        t.random_(0, 100)
    for t in (cache.k_scales, cache.v_scales):
        t.fill_(120)
    own, i32 = new // 64, dict(dtype=torch.int32, device="cuda")
    table = torch.cat([torch.arange(prefix // 64).expand(seqs, -1),
                       prefix // 64 + torch.arange(seqs * own).view(seqs, own)], 1).to(**i32).contiguous()
    q = torch.randn(seqs * new, heads, 128, device="cuda", dtype=torch.bfloat16)
    b = dict(cache=cache, q=q, cu=torch.arange(seqs + 1, **i32) * new, table=table, kv=torch.full((seqs,), prefix + new, **i32),
             q_lens=[new] * seqs, kv_lens=[prefix + new] * seqs, groups=torch.tensor([0, seqs], **i32),
             prefixes=torch.tensor([prefix], **i32), most=prefix)
    out, _, shared = shares(torch, mxk, b, tight=True, lse=False)
    assert not shared and torch.equal(out, ordinary(torch, mxk, b))


@pytest.mark.parametrize("most", [128, 200, 256, 511, 640, 5000])
def test_prefixes_are_cut_at_their_bound(torch_cuda, mxk, most):
    """Many sequences, so that 128 tokens are worth it."""
    torch, g = torch_cuda, np.random.default_rng(2)
    b = build(torch, mxk, g, [(640, 640, [(1, 1 + i % 40) for i in range(200)])], 32, 32, 64, 16, 8, "bfloat16")
    out, lse, shared = shares(torch, mxk, b, max_prefix=most, max_kv=680)
    assert shared
    check(torch, b, out, lse)


@pytest.mark.parametrize("bits,dim,dtype", [(8, 128, "bfloat16"), (6, 64, "float16"), (4, 128, "float16")])
def test_long_chunks_as_the_ordinary_call(torch_cuda, mxk, bits, dim, dtype):
    """Up to 2048 new tokens a sequence, several groups, beside single tokens, with bounds that
    make the call share: within the tolerance of the definition, as the ordinary call is."""
    torch, g = torch_cuda, np.random.default_rng(3)
    groups = [(1024, 1024, [(2048, 2100), (1, 70), (700, 701)]), (384, 384, [(333, 400), (1, 1), (513, 513)])]
    b = build(torch, mxk, g, groups, 4, 2, dim, 64, bits, dtype)
    out, lse, shared = shares(torch, mxk, b)
    assert shared
    check(torch, b, out, lse)
    other = ordinary(torch, mxk, b)
    check(torch, b, other, None)
    assert not torch.equal(out, other)


def test_results_do_not_depend_on_timing(torch_cuda, mxk):
    """Chunks of single tokens are taken from a counter: again, and on two streams at once."""
    torch, g = torch_cuda, np.random.default_rng(4)
    made = [build(torch, mxk, g, [(512, 512, [(1, 1 + 97 * i % 1500) for i in range(n)])], 16, 4, 128, 32, bits, "bfloat16")
            for n, bits in ((50, 8), (70, 4))]
    want = [shares(torch, mxk, b) for b in made]
    assert all(shared for _, _, shared in want)
    # without any wait between the calls
    streams = [torch.cuda.Stream() for _ in made]
    got = [[torch.full_like(b["q"], 77.0) for _ in range(20)] for b in made]
    tables = []
    for b in made:
        width = 1 + 4096 * 400 // 32
        tables.append(torch.nn.functional.pad(b["table"], (0, width - b["table"].shape[1])))
    torch.cuda.synchronize()
    for i in range(20):
        for b, table, stream, outs in zip(made, tables, streams, got):
            mxk.cache_attention_shared(b["cache"], b["q"], b["cu"], table, b["kv"], b["groups"], b["prefixes"], outs[i], max_q=1,
                                       max_kv=4096 * 400, max_prefix=4096 * 400, stream=stream)
    torch.cuda.synchronize()
    for b, outs, (out, _, _) in zip(made, got, want):
        check(torch, b, outs[0], None)
        assert all(torch.equal(o, outs[0]) for o in outs)
