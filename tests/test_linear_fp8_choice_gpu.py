"""Which layers quantise their rows in the product's kernel, and that both ways give the same."""
import pytest
from test_gemm_fp8_gpu import expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k,own", [(1, 4096, 4096, True), (8, 6144, 4096, True), (8, 6272, 4096, False), (1, 8192, 4096, False),
                                       (9, 1024, 4096, True), (9, 1152, 4096, False), (16, 4096, 4096, False), (17, 256, 512, False)])
def test_layers_of_few_rows(torch_cuda, mxk, m, n, k, own):
    torch = torch_cuda
    x = torch.randn(m, k, device="cuda").to(torch.bfloat16)
    b, b_scales = expected(torch, torch.randn(n, k, device="cuda") * k ** -0.5, 128)
    b = b.to(torch.uint8)
    out, want = (torch.empty(m, n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    mxk.profile_enable()
    mxk.linear_fp8(x, b, b_scales, out)
    names = mxk.profile_read()
    mxk.profile_enable(False)
    assert ("linear_fp8" in names) == own and ("quantize_fp8" in names) != own
    a, a_scales = torch.empty(m, k, dtype=torch.uint8, device="cuda"), torch.empty(m, -(-k // 128), device="cuda")
    mxk.quantize_fp8(x, a, a_scales)
    mxk.gemm_fp8(a, a_scales, b, b_scales, want)
    assert torch.equal(out, want)
