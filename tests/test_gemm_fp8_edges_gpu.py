"""Large E4M3 products into slices of a wider matrix whose rows are aligned to 16 bytes and whose
columns fill no whole 16 bytes: what lies beside and behind the slice stays."""
import pytest
from test_gemm_fp8_gpu import expected, product_limit, scaled

pytestmark = pytest.mark.gpu


# the last two: columns beside the pairs for the other kernel; fewer columns than 16 bytes hold
@pytest.mark.parametrize("m,k", [(2729, 48), (300, 256), (2560, 4096), (7400, 144)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("odd", [1, 2, 3, 4, 5, 7])
def test_columns_that_fill_no_piece(torch_cuda, mxk, dtype, m, k, odd):
    torch = torch_cuda
    dtype = getattr(torch, dtype)
    n = {2729: 1640, 300: 8000, 2560: 2040, 7400: 0}[m] + odd
    g = torch.Generator(device="cuda").manual_seed(m + odd)
    a, a_scales = expected(torch, torch.randn(m, k, generator=g, device="cuda"), 1)
    b, b_scales = expected(torch, torch.randn(n, k, generator=g, device="cuda") * k ** -0.5, 128)
    a, b = a.to(torch.uint8), b.to(torch.uint8)
    x, w = scaled(torch, a, a_scales, 1), scaled(torch, b, b_scales, 128)
    want = x @ w.T
    limit = product_limit(torch, x, w, -(-k // 128), dtype, want)
    for left, right in ((8, 24 - n % 8), (0, 8 - n % 8), (64, 136 - n % 8)):
        wide = torch.full((m + 2, left + n + right), 9.0, dtype=dtype, device="cuda")
        out = wide[1:m + 1, left:left + n]
        assert out.data_ptr() % 16 == 0 and out.stride(0) * out.element_size() % 16 == 0
        mxk.gemm_fp8(a, a_scales, b, b_scales, out)
        assert ((out.double() - want).abs() <= limit).all()
        out.fill_(9.0)
        assert (wide == 9.0).all(), "an element beside the output changed"
