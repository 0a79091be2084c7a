"""The 8-bit rows of the gated product are the rows of its f32 results."""
import pytest
import torch

from test_gpu_fp8 import operands, randn
from witchcraft_b200 import fp8

pytestmark = pytest.mark.gpu


# one product of many rows, and few rows many times: ten million codes each,
# where a product with the rounded reciprocal puts several beside the right one
# (columns in fours: f32 rows that start on 16 bytes, and so the same kernel)
@pytest.mark.parametrize("m,k,n,times", [(8192, 768, 2048, 1), (32, 256, 8192, 40), (100, 700, 520, 5), (700, 130, 332, 5)])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_codes_are_those_of_the_rounded_quotient(m, k, n, times, act):
    _, _, (gate, up) = operands(1, k, n, seed=n, mats=2)
    for i in range(times):
        a, sa = fp8.quantize(randn(m, k, seed=i, scale=1.5))
        codes, scales = fp8.gated_matmul(a, sa, *gate, *up, act=act)
        h = fp8.gated_matmul(a, sa, *gate, *up, out_dtype=torch.float32, act=act)
        want, want_scales = fp8.quantize(h)
        assert torch.equal(scales, want_scales)
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
        quotient = h / scales.repeat_interleave(128, 1)[:, :n]
        assert torch.equal(codes.float(), quotient.to(torch.float8_e4m3fn).float())
