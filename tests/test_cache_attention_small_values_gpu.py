"""Attention over cached values whose scale bytes lie at the bottom of UE8M0: 2^-127 and a
little above, alone and before tokens of ordinary magnitude, by every kernel.

Tolerance: that of test_cache_attention_gpu.check, and for rows that are small altogether the
same with two absolute terms: half of bfloat16's subnormal step, 2^-134, and the roundings to
float32's, of which a merged row takes fewer than 2^6 of 2^-150 each."""
import numpy as np
import pytest
from test_cache_attention_gpu import cached_rows, check
from test_cache_attention_shared_gpu import attend, build

pytestmark = pytest.mark.gpu

# Standard deviations of values whose blocks get scale bytes of 1 to 6, or only the lowest, 0.
SMALL = {8: 2.0 ** -116, 6: 2.0 ** -121, 4: 2.0 ** -121}
LEAST = {8: 2.0 ** -122, 6: 2.0 ** -127, 4: 2.0 ** -127}


def calls(torch, mxk, b):
    """The call of the groups, and the ordinary one."""
    out = torch.full_like(b["q"], 77.0)
    mxk.cache_attention(b["cache"], b["q"], b["cu"], b["table"], b["kv"], out, max_q=max(b["q_lens"]), max_kv=max(b["kv_lens"]))
    return [attend(torch, mxk, b)[0], out]


def check_small(torch, b, out):
    c, group, row = b["cache"], b["q"].shape[1] // b["cache"].kv_heads, 0
    for i, (n, l) in enumerate(zip(b["q_lens"], b["kv_lens"])):
        k, v = (x.repeat_interleave(group, 1) for x in cached_rows(torch, b, i))
        q = b["q"][row:row + n].double()
        s = torch.einsum("nhd,thd->hnt", q, k) * c.head_dim ** -0.5
        see = torch.arange(l, device="cuda")[None] <= l - n + torch.arange(n, device="cuda")[:, None]
        w = torch.softmax(s.masked_fill(~see, -float("inf")), -1)
        want, size = torch.einsum("hnt,thd->nhd", w, v), torch.einsum("hnt,thd->nhd", w, v.abs())
        ds = 2.0 ** -19 * c.head_dim ** -0.5 * torch.einsum("nhd,thd->hnt", q.abs(), k.abs()).amax(-1).T[..., None]
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -20 + torch.expm1(2 * ds)) * size * (1 + 2.0 ** -8) + \
            2.0 ** -26 * v.abs().max() + 2.0 ** -134 + 2.0 ** -144
        bad = ~((out[row:row + n].double() - want).abs() <= tol)
        assert want.abs().max() > 8 * tol.max(), "the test would pass zeros"
        assert not bad.any(), f"sequence {i}: {int(bad.sum())} of {bad.numel()} values off"
        row += n


# (new tokens, own tokens): many single tokens, each a warp's; few of them; chunks in packed and
# in converted tiles
MANY = [(1, 33 + i) for i in range(70)]
SHAPES = {"many": MANY, "few": [(1, 40), (1, 200)], "chunks": [(1, 50), (20, 150), (70, 300)], "long": [(300, 700), (2, 50)]}


def groups(shape):
    return [(0, None, SHAPES[shape]), (128, 128, [(1, 1), (1, 2)])]


@pytest.mark.parametrize("bits", [8, 6, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("blocks", ["one", "all"])
def test_small_values_before_ordinary_ones(torch_cuda, mxk, bits, dim, shape, blocks):
    """The first 16 tokens of every sequence hold the smallest values, in one block or altogether."""
    torch, g = torch_cuda, np.random.default_rng(1)
    b = build(torch, mxk, g, groups(shape), 4, 2, dim, 16, bits, "bfloat16")
    for slots in b["slots"][:len(SHAPES[shape])]:
        slots = torch.from_numpy(slots[:16]).cuda()
        v = torch.from_numpy(g.standard_normal((16, 2, dim)).astype(np.float32))
        v[:, :, slice(32, 64) if blocks == "one" else slice(None)] *= SMALL[bits]
        k = torch.from_numpy(g.standard_normal((16, 2, dim)).astype(np.float32))
        mxk.cache_write(b["cache"], k.cuda(), v.cuda(), slots)
    for out in calls(torch, mxk, b):
        check(torch, b, out, None)


@pytest.mark.parametrize("bits", [8, 6, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", ["small", "least"])
def test_small_values_alone(torch_cuda, mxk, bits, dim, shape, size):
    torch, g = torch_cuda, np.random.default_rng(2)
    b = build(torch, mxk, g, groups(shape), 4, 2, dim, 16, bits, "bfloat16", scale_v=(SMALL if size == "small" else LEAST)[bits])
    for out in calls(torch, mxk, b):
        check_small(torch, b, out)
