"""E4M3 products whose two scales together come near the end of float32 and beyond it."""
import pytest
from test_gemm_fp8_gpu import expected, product_limit, scaled

pytestmark = pytest.mark.gpu

# the clusters with few and many rows, the pairs, the clusters beside the pairs
SIZES = [(3, 130, 512), (64, 300, 640), (129, 400, 512), (200, 7168, 512), (2560, 2048, 4096)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_large_scales(torch_cuda, mxk, dtype, m, n, k):
    """Block 0 has sums of 0 and block 1 the smallest there are, under scales of 2^67 and 2^60, whose
    product is the largest power of two, for every third row and every other 128 columns.  One
    step more, and these outputs are infinite or no numbers; the others stay."""
    torch = torch_cuda
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(m + n)
    a, a_scales = expected(torch, torch.randn(m, k, generator=g, device="cuda"), 1)
    b, b_scales = expected(torch, torch.randn(n, k, generator=g, device="cuda") * k ** -0.5, 128)
    a, b = a.to(torch.uint8), b.to(torch.uint8)
    b[:, :256] = 0
    a[:, 128:256] = 0
    a[:, 130], b[:, 130] = 1, 1  # 2^-9 each
    a_scales[::3, :2], b_scales[::2, :2] = 2.0 ** 67, 2.0 ** 60
    x, w = scaled(torch, a, a_scales, 1), scaled(torch, b, b_scales, 128)
    want = x @ w.T
    out = torch.full((m, n), 9.0, dtype=dtype, device="cuda")
    mxk.gemm_fp8(a, a_scales, b, b_scales, out)
    assert ((out.double() - want).abs() <= product_limit(torch, x, w, -(-k // 128), dtype, want)).all()
    a_scales[::3, :2] *= 2
    again = torch.empty_like(out)
    mxk.gemm_fp8(a, a_scales, b, b_scales, again)
    over = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    over[::3] = torch.arange(n, device="cuda") // 128 % 2 == 0
    assert not again[over].isfinite().any()
    over[::3] = True  # (the other columns' scales doubled as well)
    assert torch.equal(again[~over], out[~over])


def test_scales_that_are_infinite(torch_cuda, mxk):
    """Zero times infinity is no number, as the definition has it, in that row alone."""
    torch = torch_cuda
    a, a_scales = expected(torch, torch.randn(5, 256, device="cuda"), 1)
    b, b_scales = expected(torch, torch.randn(200, 256, device="cuda"), 128)
    a, b = a.to(torch.uint8), b.to(torch.uint8)
    a[2, :128], a_scales[2, 0] = 0, float("inf")
    out = torch.empty(5, 200, device="cuda")
    mxk.gemm_fp8(a, a_scales, b, b_scales, out)
    assert out[2].isnan().all() and out[[0, 1, 3, 4]].isfinite().all()
