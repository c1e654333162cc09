"""Attention over the paged MX cache: what a row does not see does not change it,
whatever magnitudes and bytes lie there; what it sees counts with its own magnitude.

Tolerance, per output element, against the definition in float64 over what the row
sees: the output's rounding (half a unit), exp(s) rounded to f16 (2^-11 of
sum w |v|), an error of the score of token t of at most ds_t = 2^-19 * scale *
sum_d |q_d k_td| (float32 sums, elements of q and k below 2^-24 of their row's
largest), which changes its weight by a factor within exp(+-ds_t) and the sum of
the weights accordingly, values below 2^-26 of the largest that the row sees, and the
subnormal step of the output type.
"""
import math

import numpy as np
import pytest
from test_cache_attention_gpu import attend, build, cached_rows, check

pytestmark = pytest.mark.gpu


def check_rows(torch, b, out, lse, rows=None, causal=True, window=0, scale=None, seq=0):
    """Query tokens `rows` of a sequence (None: all) against the definition."""
    c = b["cache"]
    n, l, heads = b["q_lens"][seq], b["kv_lens"][seq], b["q"].shape[1]
    first = sum(b["q_lens"][:seq])
    out, lse, queries = out[first:first + n], lse[first:first + n], b["q"][first:first + n]
    scale = c.head_dim ** -0.5 if scale is None else scale
    u, tiny = (2.0 ** -8, 0.0) if out.dtype == torch.bfloat16 else (2.0 ** -11, 2.0 ** -25)
    k, v = cached_rows(torch, b, seq)
    rows = torch.arange(n, device="cuda") if rows is None else rows
    p, t = l - n + rows, torch.arange(l, device="cuda")
    see = t[None] <= p[:, None] if causal else torch.ones(len(rows), l, dtype=torch.bool, device="cuda")
    if window:
        see &= t[None] > p[:, None] - window
    for h in range(heads):
        q = queries[rows, h].double()
        kh, vh = k[:, h * c.kv_heads // heads], v[:, h * c.kv_heads // heads]
        # nothing that is not seen enters the sums, infinite or not
        s = torch.where(see, scale * (q @ torch.where(see.any(0)[:, None], kh, 0.0).T), -math.inf)
        z = torch.logsumexp(s, -1)
        w = torch.where(see, torch.exp(s - z[:, None]), 0.0)
        ds = torch.where(w > 0, 2.0 ** -19 * abs(scale) * (q.abs() @ kh.abs().T), 0.0)
        off = w * torch.expm1(ds)
        vs = torch.where(see.any(0)[:, None], vh, 0.0)
        want, size = w @ vs, w @ vs.abs()
        most = torch.stack([vs[see[i]].abs().max() for i in range(len(rows))])[:, None]
        tol = u * want.abs() + (2.0 ** -11 + 2.0 ** -20) * size * (1 + u) + \
            2 * (off @ vs.abs() + off.sum(-1, keepdim=True) * size) + 2.0 ** -26 * most + tiny
        assert bool(torch.isfinite(tol).all())
        got = out[rows, h].double()
        bad = ~((got - want).abs() <= tol)
        assert not bad.any(), f"head {h}: {int(bad.sum())} values off, rows {bad.any(-1).nonzero()[:8, 0].tolist()}"
        dz = 2 * off.sum(-1) + 2.0 ** -20 * (1 + z.abs())
        assert bool(((lse[rows, h].double() - z).abs() <= dz).all()), f"head {h}: lse"


def filled(torch, mxk, g, n, l, dim, bits, change, dtype="bfloat16", page=32, heads=4):
    """One sequence of n new tokens in l, its keys and values changed by change(k, v)."""
    k, v = (g.standard_normal((l, 2, dim)).astype(np.float32) for _ in range(2))
    k[:, :, :3] *= 6
    change(k, v)
    return build(torch, mxk, g, [n], [l], heads, 2, dim, page, bits, dtype, cached=[(k, v)])


SIZES = [(6, 200), (6, 333), (40, 300), (40, 450), (300, 700)]  # every kernel, cuts inside and at tiles
FORMS = [(8, 128), (8, 64), (6, 128), (4, 64)]


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


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("n,l", SIZES)
@pytest.mark.parametrize("size", [2.0 ** 30, 2.0 ** 60, math.inf])
def test_a_later_key_of_any_size(torch_cuda, mxk, bits, dim, n, l, size):
    """The key of a token in the middle of the chunk is huge or has overflowed: the rows
    before it get their own scores."""
    torch, g = torch_cuda, np.random.default_rng(23)
    at = l - n + n // 2

    def change(k, v):
        k[at, :, 7] = size
    b = filled(torch, mxk, g, n, l, dim, bits, change)
    out, lse = attend(torch, mxk, b)
    check_rows(torch, b, out, lse, torch.arange(n // 2, device="cuda"))


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("n,l", SIZES)
def test_an_earlier_key_outside_the_window(torch_cuda, mxk, bits, dim, n, l):
    """A huge key that only the first rows' windows hold."""
    torch, g = torch_cuda, np.random.default_rng(24)
    window = 90

    def change(k, v):
        k[l - n - window + n // 2, :, 7] = 2.0 ** 40
    b = filled(torch, mxk, g, n, l, dim, bits, change)
    out, lse = attend(torch, mxk, b, window=window)
    check_rows(torch, b, out, lse, torch.arange(n // 2 + 1, n, device="cuda"), window=window)


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("n,l", SIZES)
def test_scores_far_below_the_others(torch_cuda, mxk, bits, dim, n, l):
    """Keys that point away from every query with a magnitude of 2^40: they weigh nothing,
    and the others keep their scores."""
    torch, g = torch_cuda, np.random.default_rng(25)

    def change(k, v):
        k[:, :, 5] = 0.25  # all queries are positive there
        k[[3, l // 2, l - n // 2 - 1]] = 0
        k[[3, l // 2, l - n // 2 - 1], :, 5] = -2.0 ** 40
    b = filled(torch, mxk, g, n, l, dim, bits, change)
    b["q"][..., 5] = 1.0
    out, lse = attend(torch, mxk, b)
    check_rows(torch, b, out, lse)


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("n,l", SIZES)
def test_blocks_of_zeros_beside_small_keys(torch_cuda, mxk, bits, dim, n, l):
    """Keys of about 2^-40 under a scale of 2^38, with blocks of zeros (whose scale byte
    stands for 1) and whole rows of them."""
    torch, g = torch_cuda, np.random.default_rng(26)

    def change(k, v):
        k *= 2.0 ** -40
        k[:, :, 32:64] = 0
        k[::7] = 0
    b = filled(torch, mxk, g, n, l, dim, bits, change)
    out, lse = attend(torch, mxk, b, scale=2.0 ** 38)
    check_rows(torch, b, out, lse, scale=2.0 ** 38)


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("n,l", SIZES + [(6, 6), (100, 100), (300, 300)])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 30, 2.0 ** 60, math.inf])
def test_a_later_value_of_any_size(torch_cuda, mxk, bits, dim, n, l, size):
    """The value of a token in the middle of the chunk is huge or has overflowed: the rows
    before it get their own values, those after it its part of it."""
    torch, g = torch_cuda, np.random.default_rng(27)
    at = l - n + n // 2

    def change(k, v):
        v[at, :, 7] = size
    b = filled(torch, mxk, g, n, l, dim, bits, change)
    out, lse = attend(torch, mxk, b)
    check_rows(torch, b, out, lse, torch.arange(n // 2 if size == math.inf else n, device="cuda"))


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("n,l", SIZES)
@pytest.mark.parametrize("size", [2.0 ** 9, 2.0 ** 20, 2.0 ** 70])
def test_earlier_values_outside_the_window(torch_cuda, mxk, bits, dim, n, l, size):
    """Huge values of several sizes that only the first rows' windows hold, one by one and
    a stretch of them."""
    torch, g = torch_cuda, np.random.default_rng(28)
    window = 140

    def change(k, v):
        start = l - n - window + 1
        v[start:start + n // 2] *= size
        v[start + n // 3] *= 2.0 ** 9
    b = filled(torch, mxk, g, n, l, dim, bits, change)
    out, lse = attend(torch, mxk, b, window=window)
    check_rows(torch, b, out, lse, window=window)


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("n,l", SIZES)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 180), (False, 0)])
def test_blocks_of_zeros_beside_small_values(torch_cuda, mxk, bits, dim, n, l, causal, window):
    """Values of about 2^-40 with blocks of zeros (whose scale byte stands for 1), whole
    rows and a stretch of them."""
    torch, g = torch_cuda, np.random.default_rng(29)

    def change(k, v):
        v *= 2.0 ** -40
        v[:, :, 32:64] = 0
        v[::7] = 0
        v[l // 2 - 64:l // 2 + 100] = 0
    b = filled(torch, mxk, g, n, l, dim, bits, change)
    out, lse = attend(torch, mxk, b, causal=causal, window=window)
    check_rows(torch, b, out, lse, causal=causal, window=window)


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("n,l", SIZES + [(300, 300)])
@pytest.mark.parametrize("window", [0, 100])
def test_magnitudes_all_over(torch_cuda, mxk, bits, dim, n, l, window):
    """Keys and values whose scales go up and down by 2^60 from token to token."""
    torch, g = torch_cuda, np.random.default_rng(30)

    def change(k, v):
        k *= np.ldexp(1.0, g.integers(-60, 1, (l, 2, 1))).astype(np.float32)
        v *= np.ldexp(1.0, g.integers(-30, 31, (l, 2, 1))).astype(np.float32)
    b = filled(torch, mxk, g, n, l, dim, bits, change)
    out, lse = attend(torch, mxk, b, window=window)
    check_rows(torch, b, out, lse, window=window)


@pytest.mark.parametrize("n", [5, 60, 300])
def test_nan_beside_huge_values(torch_cuda, mxk, n):
    """A NaN among the elements of a token, in a tile that is worked through by hand: it
    reaches the rows that see it, in its feature."""
    torch, g = torch_cuda, np.random.default_rng(31)
    l, at = 400, 400 - n + n // 2

    def change(k, v):
        v[at, :, 9] = 2.0 ** 50
    b = filled(torch, mxk, g, n, l, 128, 8, change)
    clean, lse = attend(torch, mxk, b)
    slot = int(b["slots"][0][at])
    b["cache"].v_values[slot // 32, 1, slot % 32, 37] = 0x7f
    out, lse2 = attend(torch, mxk, b)
    assert torch.equal(lse, lse2) and torch.equal(out[:, :2], clean[:, :2])
    assert torch.equal(out[:n // 2], clean[:n // 2])
    assert torch.isnan(out[n // 2:, 2:, 37]).all()
    rest = torch.arange(128, device="cuda") != 37
    assert torch.equal(out[:, 2:, rest], clean[:, 2:, rest])


@pytest.mark.parametrize("bits,dim", FORMS)
@pytest.mark.parametrize("sizes", [[(90, 90), (40, 333), (33, 33), (200, 460)] * 5, [(300, 300), (260, 700)] * 3],
                         ids=["packed", "ready"])
def test_units_one_after_the_other(torch_cuda, mxk, bits, dim, sizes):
    """Blocks that work through several units, by hand and not, first tiles and later ones."""
    torch, g = torch_cuda, np.random.default_rng(32)
    cached = []
    for i, (n, l) in enumerate(sizes):
        k, v = (g.standard_normal((l, 2, dim)).astype(np.float32) for _ in range(2))
        if i % 3 < 2:
            v[l - n + n // 3, :, 3] = 2.0 ** 40
            k[l - n + n // 4, :, 5] = 2.0 ** 30
        cached.append((k, v))
    q_lens, kv_lens = [n for n, _ in sizes], [l for _, l in sizes]
    b = build(torch, mxk, g, q_lens, kv_lens, 8, 2, dim, 32, bits, "bfloat16", cached=cached)
    out, lse = attend(torch, mxk, b)
    for i, (n, l) in enumerate(sizes):
        check_rows(torch, b, out, lse, torch.arange(n // 4, device="cuda") if i % 3 < 2 else None, seq=i)
    again, lse2 = attend(torch, mxk, b)
    same = (out == again) | (torch.isnan(out) & torch.isnan(again))
    assert bool(same.all()), "the same call twice differs"
