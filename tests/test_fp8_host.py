"""Argument checks of the 8-bit operators: they come before any CUDA call, so
a process without a GPU gets the same refusals."""
import ctypes

import pytest
import torch

from witchcraft_b200 import fp8

F32, F16, BF16, E4M3 = 0, 1, 2, 3
OK, INVALID = 0, -1
P = 1 << 20       # a non-null, well-aligned address that no refused call reads


def rows(lib, x=P, t=F32, m=4, k=256, ldx=256, codes=P, ldc=256, scales=P, lds=2, weight=False):
    f = lib.wc_fp8_quantize_weight if weight else lib.wc_fp8_quantize_rows
    return f(x, t, m, k, ldx, codes, ldc, scales, lds, None)


def norm(lib, x=P, t=F32, ldx=256, delta=P, dt=F16, ldd=256, total=P, lds_=256, w=P, m=4, k=256, eps=1e-6, codes=P,
         ldc=256, scales=P, lds=2):
    return lib.wc_fp8_rmsnorm(x, t, ldx, delta, dt, ldd, total, lds_, w, m, k, eps, codes, ldc, scales, lds, None)


def mm(lib, a=P, lda=256, sa=P, ldsa=2, m=4, k=256, w=P, ldw=256, sw=P, ldsw=2, n=8, res=None, ldr=0, out=P, t=F16,
       ldo=8):
    return lib.wc_fp8_matmul(a, lda, sa, ldsa, m, k, w, ldw, sw, ldsw, n, res, ldr, out, t, ldo, None)


def gated(lib, a=P, lda=256, sa=P, ldsa=2, m=4, k=256, w=P, ldw=256, sw=P, ldsw=2, up=P, ldup=256, sup=P, ldsup=2,
          n=8, act=0, out=P, t=E4M3, ldo=16, os=P, ldos=1):
    return lib.wc_fp8_gated_matmul(a, lda, sa, ldsa, m, k, w, ldw, sw, ldsw, up, ldup, sup, ldsup, n, act, out, t, ldo,
                                   os, ldos, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(x=P + 2), dict(t=E4M3), dict(t=9), dict(m=-1), dict(k=0),
                                 dict(k=1 << 40), dict(ldx=255), dict(codes=None), dict(codes=P + 8), dict(ldc=250),
                                 dict(ldc=264), dict(scales=None), dict(scales=P + 2), dict(lds=1)])
@pytest.mark.parametrize("weight", [False, True])
def test_quantisation_refuses(cuda_lib, bad, weight):
    assert rows(cuda_lib, weight=weight, **bad) == INVALID
    assert cuda_lib.wc_fp8_last_error()


@pytest.mark.parametrize("bad", [dict(x=None), dict(t=E4M3), dict(ldx=100), dict(dt=E4M3), dict(delta=P + 1),
                                 dict(ldd=255), dict(total=None), dict(total=P + 2), dict(lds_=255), dict(w=None),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(m=-5), dict(k=0), dict(codes=P + 4),
                                 dict(ldc=272 - 8), dict(lds=1)])
def test_rmsnorm_refuses(cuda_lib, bad):
    assert norm(cuda_lib, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(a=None), dict(a=P + 1), dict(lda=264), dict(lda=240), dict(sa=None), dict(ldsa=1),
                                 dict(m=-1), dict(k=0), dict(n=0), dict(n=1 << 33), dict(w=None), dict(ldw=8),
                                 dict(sw=None), dict(ldsw=0), dict(res=P + 1, ldr=8), dict(res=P, ldr=7), dict(out=None),
                                 dict(out=P + 1), dict(t=E4M3), dict(t=-1), dict(ldo=7)])
def test_matmul_refuses(cuda_lib, bad):
    assert mm(cuda_lib, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(a=None), dict(up=None), dict(ldup=250), dict(sup=None), dict(ldsup=1),
                                 dict(act=2), dict(out=None), dict(out=P + 4), dict(ldo=8), dict(os=None),
                                 dict(ldos=0), dict(t=4), dict(t=F16, out=P + 1), dict(t=F16, ldo=7), dict(k=0)])
def test_gated_refuses(cuda_lib, bad):
    assert gated(cuda_lib, **bad) == INVALID


def test_no_rows_is_no_work(cuda_lib):
    assert rows(cuda_lib, m=0, x=None, codes=None, scales=None) == OK
    assert rows(cuda_lib, m=0, weight=True) == OK
    assert norm(cuda_lib, m=0) == OK
    assert mm(cuda_lib, m=0) == OK
    assert gated(cuda_lib, m=0) == OK


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 256)
    a, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.ones(4, 2)
    w, sw = torch.zeros(8, 256).to(torch.float8_e4m3fn), torch.ones(1, 2)
    for call in (lambda: fp8.quantize(x), lambda: fp8.quantize_weight(x),
                 lambda: fp8.rmsnorm(x, torch.ones(256)), lambda: fp8.matmul(a, s, w, sw),
                 lambda: fp8.gated_matmul(a, s, w, sw, w, sw)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_codes_start_on_16_bytes():
    t = fp8.empty_codes(3, 17, "cpu")
    assert t.shape == (3, 17) and t.stride() == (32, 1) and t.dtype == torch.float8_e4m3fn
    assert fp8.empty_codes(3, 32, "cpu").is_contiguous()
