"""Attention over the paged MX cache: what a row does not see does not change it,
whatever magnitudes and bytes lie there."""
import numpy as np
import pytest
from test_cache_attention_gpu import attend, build, check

pytestmark = pytest.mark.gpu


def poison(b, i, tokens, byte=0xff):
    """Fills the elements and scales of some tokens of sequence i with a byte."""
    c = b["cache"]
    slots = b["slots"][i][tokens]
    for t in (c.k_values, c.k_scales, c.v_values, c.v_scales):
        t[slots // c.page_size, :, slots % c.page_size] = byte


@pytest.mark.parametrize("bits", [8, 6, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len,window", [(1, 37), (5, 150), (40, 131), (300, 77), (300, 300)])
def test_what_lies_before_every_window(torch_cuda, mxk, bits, dim, q_len, window):
    """Slots before the first row's window, whose pages a program may have given to
    others, hold NaNs and scale bytes of 255: the result is that of a clean cache, bit
    for bit."""
    torch, g = torch_cuda, np.random.default_rng(21)
    l = 900
    b = build(torch, mxk, g, [q_len], [l], 4, 2, dim, 16, bits, "float16")
    want = attend(torch, mxk, b, window=window)
    check(torch, b, *want, window=window)
    first = l - q_len + 1 - window
    for byte in (0xff, 0xfe):
        poison(b, 0, np.arange(first), byte)
        got = attend(torch, mxk, b, window=window)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_what_lies_before_the_windows_of_several_sequences(torch_cuda, mxk):
    """The same for sequences of all sizes in one call."""
    torch, g = torch_cuda, np.random.default_rng(22)
    q_lens, kv_lens, window = [1, 7, 60, 400, 3, 150], [700, 90, 500, 900, 3, 1000], 70
    b = build(torch, mxk, g, q_lens, kv_lens, 4, 2, 128, 32, 8, "bfloat16")
    want = attend(torch, mxk, b, window=window)
    for i, (n, l) in enumerate(zip(q_lens, kv_lens)):
        poison(b, i, np.arange(max(0, l - n + 1 - window)))
    got = attend(torch, mxk, b, window=window)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
