"""Attention over the paged MX cache with values near the ends of float32's range: a mean
of values is no larger than they are, whatever sums it takes."""
import numpy as np
import pytest
from test_cache_attention_gpu import attend, build, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [2.0 ** 118, 2.0 ** 121, 2.0 ** -105])
@pytest.mark.parametrize("bits,dim", [(8, 128), (6, 64), (4, 128)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [20, 400]), ([1], [30000]), ([50, 3], [9000, 90]),
                                            ([300, 300], [301, 5000]), ([600], [20000])])
def test_values_near_the_ends_of_the_range(torch_cuda, mxk, scale, bits, dim, q_lens, kv_lens):
    """Units of one block and units in a few and in many parts."""
    torch, g = torch_cuda, np.random.default_rng(61)
    b = build(torch, mxk, g, q_lens, kv_lens, 4, 2, dim, 128, bits, "bfloat16", scale_v=scale)
    check(torch, b, *attend(torch, mxk, b))
