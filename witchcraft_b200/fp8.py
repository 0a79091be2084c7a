"""8-bit layers over the CUDA kernels of include/wc_fp8.h: rows and weights in
`torch.float8_e4m3fn` with f32 scales, the RMSNorm that writes such rows, and
the products that read them.

A value is code * scale.  Rows [m, k] have scales [m, ceil(k / 128)], one per
row and 128 columns; weights [n, k] have scales [ceil(n / 128), ceil(k / 128)],
one per 128 x 128 block.  A feed-forward block reads

    x, codes, scales = fp8.rmsnorm(x, norm_weight, delta=attention_output)
    codes, scales = fp8.gated_matmul(codes, scales, *wi_0, *wi_1)
    x = fp8.matmul(codes, scales, *wo, residual=x)

with each weight once through `quantize_weight`.  Everything runs on the
current stream of the tensors' device; results are new tensors unless `out` is
given.  For inference: the operators have no gradient and refuse tensors that
require grad where grad mode is on.  (No counterpart in the reference, whose layers run in f32.)
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os

import torch

from ._lib import HERE, WcError, lib  # noqa: F401  (WcError: what the calls raise)

BLOCK = 128


def _load():
    path = os.path.join(HERE, "_fp8_torch.so")
    if not os.path.exists(path):
        raise ImportError(f"{path} is not built; run `python -m witchcraft_b200.build`")
    loader = importlib.machinery.ExtensionFileLoader("_fp8_torch", path)
    spec = importlib.util.spec_from_file_location("_fp8_torch", path, loader=loader)
    module = importlib.util.module_from_spec(spec)
    loader.exec_module(module)
    names = ("quantize_rows", "quantize_weight", "rmsnorm", "matmul", "gated_matmul", "last_error")
    module.bind(*(ctypes.cast(getattr(lib(), "wc_fp8_" + n), ctypes.c_void_p).value for n in names))
    return module


_native = _load()


def empty_codes(rows: int, cols: int, device) -> torch.Tensor:
    """Uninitialised codes [rows, cols] whose rows start at multiples of 16
    bytes, as the kernels need them."""
    wide = -(-cols // 16) * 16
    t = torch.empty((rows, wide), dtype=torch.float8_e4m3fn, device=device)
    return t if wide == cols else t[:, :cols]


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [m, k] (f32, f16, bf16) -> codes [m, k], scales [m, ceil(k / 128)]."""
    return _native.quantize(x)


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights [n, k] -> codes [n, k], scales [ceil(n / 128), ceil(k / 128)]."""
    return _native.quantize_weight(w)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, delta: torch.Tensor | None = None,
            out: torch.Tensor | None = None):
    """t = x (+ delta); codes, scales of t / sqrt(mean(t^2) + eps) * weight.

    Returns (codes, scales), or with delta (sum, codes, scales), sum = t in
    x's type; `out` takes the sum (`out=x`: in place)."""
    return _native.rmsnorm(x, weight, eps, delta, out)


def matmul(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
           out_dtype: torch.dtype = torch.float16, residual: torch.Tensor | None = None,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """rows a [m, k] . weights w [n, k]^T (+ residual) -> [m, n] of out_dtype
    (f32, f16, bf16), f32 sums rounded once.

    A residual has the result's type and fixes out_dtype; `out=residual` adds
    in place."""
    return _native.matmul(a, a_scales, w, w_scales, out_dtype, residual, out)


def gated_matmul(a: torch.Tensor, a_scales: torch.Tensor, gate: torch.Tensor, gate_scales: torch.Tensor,
                 up: torch.Tensor, up_scales: torch.Tensor, out_dtype: torch.dtype | None = None, act: str = "gelu"):
    """h = act(a . gate^T) * (a . up^T), gate and up [n, k]; act "gelu" (tanh
    form) or "silu".

    out_dtype None: (codes, scales) of h, the rows of the product that
    follows; f32, f16 or bf16: h itself."""
    return _native.gated_matmul(a, a_scales, gate, gate_scales, up, up_scales, out_dtype, act)


def synchronize(device=None) -> None:
    """Waits for the current stream of `device`; raises if a product's
    in-kernel wait ran out on the device, on any stream, since the last call.

    No other call reports that: call this before results are used, once every
    stream with products has been waited for."""
    with torch.cuda.device(device):
        rc = lib().wc_fp8_sync(torch.cuda.current_stream().cuda_stream)
        if rc != 0:
            msg = lib().wc_fp8_last_error()
            raise WcError(rc, msg.decode() if msg else "")
