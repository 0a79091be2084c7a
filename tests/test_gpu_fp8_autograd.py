"""8-bit operators next to autograd: every float input is checked, and `out`
counts as written."""
import pytest
import torch

from test_gpu_fp8 import operands, randn
from witchcraft_b200 import fp8

pytestmark = pytest.mark.gpu


def test_each_input_that_requires_grad_is_refused():
    x, d, w = randn(4, 256), randn(4, 256, seed=1), torch.ones(256, device="cuda")
    a, sa, [(q, sq)] = operands(4, 256, 256)
    grad = lambda t: t.clone().requires_grad_()
    for call in (lambda: fp8.rmsnorm(x, grad(w)), lambda: fp8.rmsnorm(x, w, delta=grad(d)),
                 lambda: fp8.rmsnorm(x, w, delta=d, out=x.clone().requires_grad_()),
                 lambda: fp8.matmul(a, grad(sa), q, sq), lambda: fp8.matmul(a, sa, q, grad(sq)),
                 lambda: fp8.matmul(a, sa, q, sq, residual=grad(x)),
                 lambda: fp8.matmul(a, sa, q, sq, torch.float32, out=grad(x)),
                 lambda: fp8.gated_matmul(a, sa, q, sq, q, grad(sq))):
        with pytest.raises(ValueError, match="requires grad"):
            call()
        with torch.no_grad():
            call()


def test_out_counts_as_written():
    x, d, w = randn(4, 256), randn(4, 256, seed=1), torch.ones(256, device="cuda")
    a, sa, [(q, sq)] = operands(4, 256, 256)
    leaf = torch.ones(4, 256, device="cuda", requires_grad=True)
    for call in (lambda: fp8.rmsnorm(x, w, delta=d, out=x), lambda: fp8.matmul(a, sa, q, sq, residual=x, out=x),
                 lambda: fp8.matmul(a, sa, q, sq, torch.float32, out=x)):
        y = leaf * x               # saves x for the gradient
        before = x._version
        call()
        assert x._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_inference_tensors():
    with torch.inference_mode():
        x, d, w = randn(4, 256), randn(4, 256, seed=1), torch.ones(256, device="cuda")
        a, sa, [(q, sq)] = operands(4, 256, 256)
        fp8.matmul(a, sa, q, sq, residual=x, out=x)
    fp8.rmsnorm(x, w, delta=d, out=x)   # outside too
