"""The second half of a T5 encoder block in 8 bits (witchcraft_b200.fp8):

    x, codes, scales = rmsnorm(x + attention output)          8-bit rows
    codes, scales    = gelu(rows . wi_0^T) * (rows . wi_1^T)  8-bit rows
    x                = x + rows . wo^T

in three kernels, with the block's Q4_K weights brought to 8 bits once.  Run as

    python examples/fp8_feed_forward.py [--tokens 16384] [--layer 0]

it prints how far the result is from the same block in f32 and how long both
this and the f16 products that the encoder runs (`wc_gemm_f16`) take.
"""
from __future__ import annotations

import argparse
import ctypes
import os
import sys
from dataclasses import dataclass

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from witchcraft_b200 import fp8  # noqa: E402
from witchcraft_b200._lib import check, lib  # noqa: E402
from witchcraft_b200.synth import SyntheticModel, T5Config, make_synthetic_model  # noqa: E402

Codes = tuple[torch.Tensor, torch.Tensor]


def _p(t: torch.Tensor):
    return ctypes.c_void_p(t.data_ptr())


def dequantise(blocks: np.ndarray) -> torch.Tensor:
    """Q4_K rows [n, k / 256, 144] -> f32 [n, k] on the GPU."""
    raw = torch.from_numpy(np.ascontiguousarray(blocks).reshape(-1)).cuda()
    out = torch.empty(blocks.shape[0], raw.numel() // 144 * 256 // blocks.shape[0], device="cuda")
    check(lib().wc_q4k_dequant(_p(raw), raw.numel() // 144, _p(out),
                               ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    return out


@dataclass
class FeedForward:
    """One block's norm weights and its three matrices in 8 bits."""
    norm: torch.Tensor
    wi_0: Codes
    wi_1: Codes
    wo: Codes
    eps: float = 1e-6

    @staticmethod
    def load(model: SyntheticModel, layer: int) -> "FeedForward":
        p = f"encoder.block.{layer}.layer.1."
        w = [fp8.quantize_weight(dequantise(model.q4k[p + f"DenseReluDense.{n}.weight"])) for n in ("wi_0", "wi_1", "wo")]
        norm = torch.from_numpy(np.asarray(model.f32[p + "layer_norm.weight"], np.float32).reshape(-1)).cuda()
        return FeedForward(norm, *w, eps=model.config.layer_norm_epsilon)

    def __call__(self, x: torch.Tensor, attention: torch.Tensor) -> torch.Tensor:
        """Residual stream x [tokens, d_model] (f32) and the attention
        sub-layer's output -> the stream after the block; x is not changed."""
        x, codes, scales = fp8.rmsnorm(x, self.norm, self.eps, attention)
        codes, scales = fp8.gated_matmul(codes, scales, *self.wi_0, *self.wi_1)
        return fp8.matmul(codes, scales, *self.wo, residual=x, out=x)


def reference(model: SyntheticModel, layer: int, x: torch.Tensor, attention: torch.Tensor) -> torch.Tensor:
    """The same in f32 from the dequantised weights."""
    p = f"encoder.block.{layer}.layer.1."
    wi_0, wi_1, wo = (dequantise(model.q4k[p + f"DenseReluDense.{n}.weight"]) for n in ("wi_0", "wi_1", "wo"))
    norm = torch.from_numpy(np.asarray(model.f32[p + "layer_norm.weight"], np.float32).reshape(-1)).cuda()
    x = x + attention.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + model.config.layer_norm_epsilon) * norm
    return x + (torch.nn.functional.gelu(y @ wi_0.T, approximate="tanh") * (y @ wi_1.T)) @ wo.T


def microseconds(f, calls: int = 50) -> float:
    """Time of one call among others."""
    for _ in range(5):
        f()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(calls):
        f()
    end.record()
    end.synchronize()
    return begin.elapsed_time(end) * 1e3 / calls


def f16_products(model: SyntheticModel, layer: int, tokens: int):
    """The block's two products as the encoder runs them for many tokens."""
    p = f"encoder.block.{layer}.layer.1.DenseReluDense."
    wi_0, wi_1, wo = (dequantise(model.q4k[p + n + ".weight"]).half() for n in ("wi_0", "wi_1", "wo"))
    d, f = wo.shape
    xn, h, x = (torch.zeros(tokens, n, dtype=t, device="cuda") for n, t in
                ((d, torch.float16), (f, torch.float16), (d, torch.float32)))

    def run():
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        check(lib().wc_gemm_f16(_p(xn), tokens, d, _p(wi_0), _p(wi_1), f, 1, _p(h), st))
        check(lib().wc_gemm_f16(_p(h), tokens, f, _p(wo), None, d, 2, _p(x), st))
    return run


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=16384)
    ap.add_argument("--layer", type=int, default=0)
    a = ap.parse_args()
    model = make_synthetic_model(T5Config(num_layers=a.layer + 1, vocab_size=512), seed=0)
    block = FeedForward.load(model, a.layer)
    g = torch.Generator(device="cuda").manual_seed(1)
    d = model.config.d_model
    x = torch.randn(a.tokens, d, generator=g, device="cuda")
    attention = torch.randn(a.tokens, d, generator=g, device="cuda").half()
    y, want = block(x, attention), reference(model, a.layer, x, attention)
    fp8.synchronize()
    added = want - x - attention.float()
    print(f"error of what the block adds: {float((y - want).norm() / added.norm()):.4f} (2-norm, relative to f32)")
    codes, scales = fp8.rmsnorm(x, block.norm)
    gated = fp8.gated_matmul(codes, scales, *block.wi_0, *block.wi_1)
    stream = x.clone()
    print(f"whole block, 8 bits:        {microseconds(lambda: block(x, attention)):8.1f} us")
    print(f"its two products, 8 bits:   "
          f"{microseconds(lambda: (fp8.gated_matmul(codes, scales, *block.wi_0, *block.wi_1), fp8.matmul(*gated, *block.wo, residual=stream, out=stream))):8.1f} us")
    if a.tokens >= 512:
        print(f"its two products, f16:      {microseconds(f16_products(model, a.layer, a.tokens)):8.1f} us")


if __name__ == "__main__":
    main()
