"""The 8-bit operators have no gradient: tensors that require grad are refused
while grad mode is on (before any CUDA call), and taken when it is off."""
import pytest
import torch

from witchcraft_b200 import fp8


def calls():
    x = torch.zeros(4, 256, requires_grad=True)
    plain, norm = torch.zeros(4, 256), torch.ones(256)
    a, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.ones(4, 2, requires_grad=True)
    w, sw = torch.zeros(8, 256).to(torch.float8_e4m3fn), torch.ones(1, 2)
    return {
        "quantize": lambda: fp8.quantize(x),
        "quantize_weight": lambda: fp8.quantize_weight(x),
        "rmsnorm": lambda: fp8.rmsnorm(x, norm),
        "matmul": lambda: fp8.matmul(a.requires_grad_(), s, w, sw),
        "gated_matmul": lambda: fp8.gated_matmul(a.requires_grad_(), s, w, sw, w, sw),
    }


@pytest.mark.parametrize("name", calls())
def test_requires_grad_is_refused(name):
    with pytest.raises(ValueError, match="requires grad"):
        calls()[name]()
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # the next check: these are host tensors
        calls()[name]()
