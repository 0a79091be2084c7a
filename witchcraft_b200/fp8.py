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
given.  (No counterpart in the reference, whose layers run in f32.)
"""
from __future__ import annotations

import torch

from ._lib import WcError, lib

BLOCK = 128
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_E4M3 = 3
_ACTS = {"gelu": 0, "silu": 1}
_CODES = torch.float8_e4m3fn


def _check(rc: int) -> None:
    if rc != 0:
        msg = lib().wc_fp8_last_error()
        raise WcError(rc, msg.decode() if msg else "")


class _On:
    """Makes a tensor's device the current one for a launch where it is not."""

    def __init__(self, t: torch.Tensor):
        self.device = t.device

    def __enter__(self):
        index = self.device.index
        self.before = torch.cuda.current_device()
        if index != self.before:
            torch.cuda.set_device(index)
        return torch.cuda.current_stream(index).cuda_stream

    def __exit__(self, *exc):
        if self.device.index != self.before:
            torch.cuda.set_device(self.before)


def _matrix(t: torch.Tensor, name: str, like: torch.Tensor | None = None, shape=None) -> None:
    if t.dim() != 2 or not t.is_cuda or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be a CUDA matrix with contiguous rows")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")


def _ld(t: torch.Tensor) -> int:
    """Leading dimension; a single row may have any stride."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _codes_ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else -(-max(t.stride(0), t.shape[1]) // 16) * 16


def _operand(codes: torch.Tensor, scales: torch.Tensor, name: str, like: torch.Tensor, rows_per_scale: int) -> None:
    _matrix(codes, name, like)
    if codes.dtype != _CODES:
        raise ValueError(f"{name} must be float8_e4m3fn codes, not {codes.dtype}")
    r, k = codes.shape
    if k < 1:
        raise ValueError(f"{name} has no columns")
    _matrix(scales, f"scales of {name}", like, (-(-r // rows_per_scale), -(-k // BLOCK)))
    if scales.dtype != torch.float32:
        raise ValueError(f"scales of {name} must be float32, not {scales.dtype}")


def _values(t: torch.Tensor, name: str, like: torch.Tensor | None = None, shape=None) -> int:
    _matrix(t, name, like, shape)
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def empty_codes(rows: int, cols: int, device) -> torch.Tensor:
    """Uninitialised codes [rows, cols] whose rows start at multiples of 16
    bytes, as the kernels need them."""
    wide = -(-cols // 16) * 16
    t = torch.empty((rows, wide), dtype=_CODES, device=device)
    return t if wide == cols else t[:, :cols]


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [m, k] (f32, f16, bf16) -> codes [m, k], scales [m, ceil(k / 128)]."""
    code = _values(x, "x")
    m, k = x.shape
    if k < 1:
        raise ValueError("x has no columns")
    codes = empty_codes(m, k, x.device)
    kb = -(-k // BLOCK)
    scales = torch.empty((m, kb), dtype=torch.float32, device=x.device)
    if m:
        with _On(x) as st:
            _check(lib().wc_fp8_quantize_rows(x.data_ptr(), code, m, k, _ld(x), codes.data_ptr(), _codes_ld(codes),
                                              scales.data_ptr(), kb, st))
    return codes, scales


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights [n, k] -> codes [n, k], scales [ceil(n / 128), ceil(k / 128)]."""
    code = _values(w, "w")
    n, k = w.shape
    if n < 1 or k < 1:
        raise ValueError("w is empty")
    codes = empty_codes(n, k, w.device)
    kb = -(-k // BLOCK)
    scales = torch.empty((-(-n // BLOCK), kb), dtype=torch.float32, device=w.device)
    with _On(w) as st:
        _check(lib().wc_fp8_quantize_weight(w.data_ptr(), code, n, k, _ld(w), codes.data_ptr(), _codes_ld(codes),
                                            scales.data_ptr(), kb, st))
    return codes, scales


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, delta: torch.Tensor | None = None,
            out: torch.Tensor | None = None):
    """t = x (+ delta); codes, scales of t / sqrt(mean(t^2) + eps) * weight.

    Returns (codes, scales), or with delta (sum, codes, scales), sum = t in
    x's type; `out` takes the sum (`out=x`: in place)."""
    code = _values(x, "x")
    m, k = x.shape
    if weight.dtype != torch.float32 or weight.shape != (k,) or weight.device != x.device or not weight.is_contiguous():
        raise ValueError(f"weight must be {k} contiguous float32 values on {x.device}")
    if k < 1:
        raise ValueError("x has no columns")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    dcode = 0
    if delta is not None:
        dcode = _values(delta, "delta", x, (m, k))
        if out is None:
            out = torch.empty((m, k), dtype=x.dtype, device=x.device)
        elif _values(out, "out", x, (m, k)) != code:
            raise ValueError(f"out must have x's type {x.dtype}")
    elif out is not None:
        raise ValueError("out is the sum with delta; there is no delta")
    codes = empty_codes(m, k, x.device)
    kb = -(-k // BLOCK)
    scales = torch.empty((m, kb), dtype=torch.float32, device=x.device)
    if m:
        with _On(x) as st:
            if delta is None:
                _check(lib().wc_fp8_rmsnorm(x.data_ptr(), code, _ld(x), None, 0, 0, None, 0, weight.data_ptr(), m, k,
                                            eps, codes.data_ptr(), _codes_ld(codes), scales.data_ptr(), kb, st))
            else:
                _check(lib().wc_fp8_rmsnorm(x.data_ptr(), code, _ld(x), delta.data_ptr(), dcode, _ld(delta),
                                            out.data_ptr(), _ld(out), weight.data_ptr(), m, k, eps, codes.data_ptr(),
                                            _codes_ld(codes), scales.data_ptr(), kb, st))
    return (codes, scales) if delta is None else (out, codes, scales)


def matmul(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
           out_dtype: torch.dtype = torch.float16, residual: torch.Tensor | None = None,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """rows a [m, k] . weights w [n, k]^T (+ residual) -> [m, n] of out_dtype
    (f32, f16, bf16), f32 sums rounded once.

    A residual has the result's type and fixes out_dtype; `out=residual` adds
    in place."""
    _operand(a, a_scales, "a", a, 1)
    _operand(w, w_scales, "w", a, BLOCK)
    (m, k), n = a.shape, w.shape[0]
    if w.shape[1] != k or n < 1:
        raise ValueError(f"w has shape {tuple(w.shape)}, expected [n >= 1, {k}]")
    if residual is not None:
        _values(residual, "residual", a, (m, n))
        out_dtype = residual.dtype
    code = _TYPES.get(out_dtype)
    if code is None:
        raise ValueError(f"out_dtype must be float32, float16 or bfloat16, not {out_dtype}")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    elif _values(out, "out", a, (m, n)) != code:
        raise ValueError(f"out is {out.dtype}, expected {out_dtype}")
    if m:
        with _On(a) as st:
            _check(lib().wc_fp8_matmul(a.data_ptr(), _codes_ld(a), a_scales.data_ptr(), _ld(a_scales), m, k,
                                       w.data_ptr(), _codes_ld(w), w_scales.data_ptr(), _ld(w_scales), n,
                                       None if residual is None else residual.data_ptr(),
                                       0 if residual is None else _ld(residual), out.data_ptr(), code, _ld(out), st))
    return out


def gated_matmul(a: torch.Tensor, a_scales: torch.Tensor, gate: torch.Tensor, gate_scales: torch.Tensor,
                 up: torch.Tensor, up_scales: torch.Tensor, out_dtype: torch.dtype | None = None, act: str = "gelu"):
    """h = act(a . gate^T) * (a . up^T), gate and up [n, k]; act "gelu" (tanh
    form) or "silu".

    out_dtype None: (codes, scales) of h, the rows of the product that
    follows; f32, f16 or bf16: h itself."""
    _operand(a, a_scales, "a", a, 1)
    _operand(gate, gate_scales, "gate", a, BLOCK)
    _operand(up, up_scales, "up", a, BLOCK)
    (m, k), n = a.shape, gate.shape[0]
    if gate.shape[1] != k or n < 1 or up.shape != gate.shape:
        raise ValueError(f"gate {tuple(gate.shape)} and up {tuple(up.shape)} must both be [n >= 1, {k}]")
    if act not in _ACTS:
        raise ValueError(f"act must be one of {sorted(_ACTS)}, not {act!r}")
    scales = None
    if out_dtype is None:
        code, out = _E4M3, empty_codes(m, n, a.device)
        scales = torch.empty((m, -(-n // BLOCK)), dtype=torch.float32, device=a.device)
        ldo = _codes_ld(out)
    else:
        code = _TYPES.get(out_dtype)
        if code is None:
            raise ValueError(f"out_dtype must be None, float32, float16 or bfloat16, not {out_dtype}")
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
        ldo = n
    if m:
        with _On(a) as st:
            _check(lib().wc_fp8_gated_matmul(a.data_ptr(), _codes_ld(a), a_scales.data_ptr(), _ld(a_scales), m, k,
                                             gate.data_ptr(), _codes_ld(gate), gate_scales.data_ptr(),
                                             _ld(gate_scales), up.data_ptr(), _codes_ld(up), up_scales.data_ptr(),
                                             _ld(up_scales), n, _ACTS[act], out.data_ptr(), code, ldo,
                                             None if scales is None else scales.data_ptr(),
                                             0 if scales is None else scales.shape[1], st))
    return out if scales is None else (out, scales)


def synchronize(device=None) -> None:
    """Waits for the current stream of `device`; raises if a product's
    in-kernel wait ran out since the last call."""
    with torch.cuda.device(device):
        _check(lib().wc_fp8_sync(torch.cuda.current_stream().cuda_stream))
