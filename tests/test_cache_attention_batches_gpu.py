"""Attention over the paged MX cache: batches whose sequences differ much, bounds far
above the lengths, and what such calls take in memory."""
import numpy as np
import pytest
from test_cache_attention_gpu import attend, build, check

pytestmark = pytest.mark.gpu


def widened(torch, b, max_kv):
    """The batch with a page table for max_kv tokens a sequence; what lies past a
    sequence's pages is any number."""
    table = torch.full((b["table"].shape[0], -(-max_kv // b["cache"].page_size)), -7, dtype=torch.int32, device="cuda")
    table[:, :b["table"].shape[1]] = b["table"]
    return dict(b, table=table)


@pytest.mark.parametrize("max_kv", [2048, 1 << 20])
def test_one_long_chunk_beside_many_decoding_sequences(torch_cuda, mxk, max_kv):
    """Few row tiles in all, though 256 sequences of the longest chunk over the longest
    cache would have more key tiles than can be numbered."""
    torch, g = torch_cuda, np.random.default_rng(41)
    q_lens = [1] * 256
    q_lens[77] = 2000
    kv_lens = [int(x) for x in g.integers(1, 200, 256)]
    kv_lens[77] = 2040
    b = widened(torch, build(torch, mxk, g, q_lens, kv_lens, 16, 2, 64, 128, 8, "bfloat16"), max_kv)
    check(torch, b, *attend(torch, mxk, b, max_kv=max_kv))


def test_unused_entries_at_the_end(torch_cuda, mxk):
    """A batch padded with sequences whose row range is empty or runs backwards."""
    torch, g = torch_cuda, np.random.default_rng(42)
    b = build(torch, mxk, g, [1, 40, 300], [100, 90, 400], 4, 2, 64, 32, 8, "bfloat16")
    want = attend(torch, mxk, b)
    cu = torch.cat([b["cu"], torch.tensor([0, 0, 0], dtype=torch.int32, device="cuda")])
    padded = dict(b, cu=cu, kv=torch.nn.functional.pad(b["kv"], (0, 3)),
                  table=torch.nn.functional.pad(b["table"], (0, 0, 0, 3)))
    got = attend(torch, mxk, padded)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_overlapping_rows_stay_inside(torch_cuda, mxk):
    """Row ranges that overlap, so that there is far more work than the query tokens
    make: nothing outside the output is written."""
    torch, g = torch_cuda, np.random.default_rng(43)
    n, seqs = 1, 4000
    b = build(torch, mxk, g, [n], [64], 2, 2, 64, 16, 8, "bfloat16")
    cu = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    cu[1::2] = n
    over = dict(b, cu=cu, table=b["table"].expand(seqs, -1).contiguous(), kv=b["kv"].expand(seqs).contiguous())
    out = torch.full((n + 2, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    attend(torch, mxk, over, lse=False, out=out[1:1 + n])
    assert (out[0] == 5.0).all() and (out[-1] == 5.0).all()


def launched(torch, mxk, call):
    """Names of the kernels that a call launches."""
    mxk.profile_enable(True)
    mxk.profile_read()
    call()
    names = {n for n, _ in mxk.profile_read().items()}
    mxk.profile_enable(False)
    return names


@pytest.mark.parametrize("max_kv", [8192, 32768])
def test_memory_goes_by_the_chunks_there_are(torch_cuda, mxk, max_kv):
    """One prompt chunk beside 63 decoding sequences: room is made for the sequences that
    can be converted, not for all of them, and the chunk has the kernel it has alone."""
    torch, g = torch_cuda, np.random.default_rng(44)
    q_lens, kv_lens = [1] * 64, [int(x) for x in g.integers(1, 300, 64)]
    q_lens[20], kv_lens[20] = 300, 700
    b = widened(torch, build(torch, mxk, g, q_lens, kv_lens, 32, 8, 128, 64, 8, "bfloat16"), max_kv)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    mxk.release_workspace()
    free = torch.cuda.mem_get_info()[0]
    names = launched(torch, mxk, lambda: attend(torch, mxk, b, max_kv=max_kv))
    taken = free - torch.cuda.mem_get_info()[0]
    assert "attention_ready" in names
    # 363 query tokens of 4 rows: at most five sequences of more than 256 rows
    assert taken <= 5 * 8 * max_kv * 128 * 4 * 1.05 + (128 << 20), f"{taken >> 20} MB"
    mxk.release_workspace()
    check(torch, b, *attend(torch, mxk, b, max_kv=max_kv))


@pytest.mark.parametrize("bits,dim", [(8, 128), (4, 64)])
def test_long_chunks_among_short_ones(torch_cuda, mxk, bits, dim):
    """Converted tiles are numbered by the sequences that have them."""
    torch, g = torch_cuda, np.random.default_rng(45)
    q_lens = [1, 300, 0, 2, 150, 260, 5, 0, 500, 1] + [1] * 40 + [270]
    kv_lens = [n + int(x) for n, x in zip(q_lens, g.integers(0, 500, len(q_lens)))]
    b = build(torch, mxk, g, q_lens, kv_lens, 4, 2, dim, 32, bits, "bfloat16")
    for kw in (dict(), dict(window=140), dict(causal=False)):
        check(torch, b, *attend(torch, mxk, b, **kw), **kw)


@pytest.mark.parametrize("q_lens", [[3], [2, 0, 70, 1], [300, 300]])
def test_nothing_cached_and_no_pages(torch_cuda, mxk, q_lens):
    """max_kv of zero needs no page table: zeros and -inf."""
    torch = torch_cuda
    cache = mxk.PagedCache.empty(2, 16, 2, 64, 8)
    seqs, tokens = len(q_lens), sum(q_lens)
    q = torch.randn(tokens, 4, 64, device="cuda").to(torch.bfloat16)
    out, lse = torch.full_like(q, 3.0), torch.full((tokens, 4), 3.0, device="cuda")
    cu = torch.tensor([0] + list(np.cumsum(q_lens)), dtype=torch.int32, device="cuda")
    mxk.cache_attention(cache, q, cu, torch.empty(seqs, 0, dtype=torch.int32, device="cuda"),
                        torch.zeros(seqs, dtype=torch.int32, device="cuda"), out, max_q=max(q_lens), max_kv=0, lse=lse)
    torch.cuda.synchronize()
    assert (out == 0).all() and (lse == -float("inf")).all()


@pytest.mark.parametrize("q_lens,kv_lens", [([300], [700]), ([400, 1, 90], [1000, 50, 300])])
def test_a_cache_too_long_to_be_converted(torch_cuda, mxk, q_lens, kv_lens):
    """Where the bounds ask for more than 4 GB of converted tiles, chunks of any length go
    through the packed kernel."""
    torch, g = torch_cuda, np.random.default_rng(46)
    max_kv = (1 << 20) + 128
    b = widened(torch, build(torch, mxk, g, q_lens, kv_lens, 32, 8, 128, 128, 8, "bfloat16"), max_kv)
    torch.cuda.synchronize()
    names = launched(torch, mxk, lambda: attend(torch, mxk, b, max_kv=max_kv))
    assert "attention_tiles" in names and "attention_ready" not in names
    check(torch, b, *attend(torch, mxk, b, max_kv=max_kv))


@pytest.mark.parametrize("max_q", [64, 512])
def test_a_graph_for_chunks_replayed_with_one_token(torch_cuda, mxk, max_q):
    """One sequence, captured for chunks, whose kernels then see a single row."""
    torch, g = torch_cuda, np.random.default_rng(47)
    b = build(torch, mxk, g, [max_q], [1500], 8, 2, 128, 64, 8, "bfloat16")
    out, lse = torch.empty_like(b["q"]), torch.empty(max_q, 8, device="cuda")
    attend(torch, mxk, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], out, max_q=max_q, max_kv=1500, lse=lse)
    for n in (1, 3, 60):
        b["cu"].copy_(torch.tensor([0, n], dtype=torch.int32))
        b["q_lens"] = [n]
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        check(torch, b, out, lse)
        assert (out[n:] == 9.0).all()
