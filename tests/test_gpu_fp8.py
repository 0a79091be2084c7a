"""8-bit operators (witchcraft_b200.fp8) against plain implementations in 64
bits.  Tolerances follow from the arithmetic and are stated where they are
used; e4m3 codes may differ from the 64-bit value by half a step of e4m3 plus
the f32 error of what was rounded."""
import math

import pytest
import torch

from witchcraft_b200 import fp8
from witchcraft_b200._lib import lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # unit roundoff of f32
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def blocks64(v, rows):
    """Largest magnitude of each block of `rows` x 128, f64, and its spread over the elements."""
    r, c = v.shape
    rb, cb = -(-r // rows), -(-c // 128)
    p = torch.zeros(rb * rows, cb * 128, dtype=torch.float64, device=v.device)
    p[:r, :c] = v.abs()
    top = p.view(rb, rows, cb, 128).amax((1, 3))
    return top, lambda t: t.repeat_interleave(rows, 0)[:r].repeat_interleave(128, 1)[:, :c]


def half_step(q):
    """Half the distance between e4m3 values at |q| (2^-10 in the subnormal range)."""
    q = q.abs().clamp_min(2.0 ** -6) * (1 + 2.0 ** -18)  # a value just under a power of two may round across it
    return torch.exp2(torch.floor(torch.log2(q)) - 4)


def check_codes(codes, scales, v64, rows=1, err=None, rel=0.0):
    """codes * scales stand for v64, known to `err` (absolute, per element) and
    `rel` (relative, per element) in f32.  The scale carries the error of the
    block's largest value and two f32 roundings; the factor 1 / scale is good
    to 2 ulp and its product rounded once: 2^-20 of the quotient in all."""
    err = torch.zeros_like(v64) if err is None else err
    top, spread = blocks64(v64, rows)
    top_err, _ = blocks64(err, rows)
    want = (top / 448).clamp_min(2.0 ** -126)
    assert scales.dtype == torch.float32 and scales.shape == want.shape
    assert ((scales.double() - want).abs() <= (top_err + rel * top) / 448 + 4 * U * want).all()
    s = spread(scales.double())
    q = v64 / s
    off = (codes.double() - q).abs()
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == v64.shape
    assert (off <= half_step(q) + (2.0 ** -20 + 2 * rel) * q.abs() + err / s).all()


# ---------------------------------------------------------------- rows and weights

SHAPES = [(1, 1), (1, 128), (3, 129), (2, 127), (7, 1000), (129, 768), (64, 1024), (5, 1030), (33, 4100), (2, 20001)]


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_rows(m, k, dtype):
    x = randn(m, k, seed=m + k, dtype=dtype, scale=3.0)
    codes, scales = fp8.quantize(x)
    check_codes(codes, scales, x.double())


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (127, 130), (129, 127), (300, 1000), (768, 2048), (1, 4099)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_weight(n, k, dtype):
    w = randn(n, k, seed=n + k, dtype=dtype, scale=0.02)
    codes, scales = fp8.quantize_weight(w)
    check_codes(codes, scales, w.double(), rows=128)


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_codes_are_those_of_the_rounded_quotient(dtype):
    """x / scale in f32, rounded, then to e4m3: ties between two codes, which
    16-bit values meet often, included."""
    x = randn(2000, 700, seed=3, dtype=dtype)
    x[:, ::128] = 448.0 * 2.0 ** torch.randint(-8, 8, (2000, 6), generator=gen(4), device="cuda")  # scales that are powers of two
    for codes, scales, rows in ((*fp8.quantize(x), 1), (*fp8.quantize_weight(x), 128)):
        s = scales.repeat_interleave(rows, 0)[:2000].repeat_interleave(128, 1)[:, :700]
        assert torch.equal(codes.float(), (x.float() / s).to(torch.float8_e4m3fn).float())


def test_rows_special_values():
    x = torch.zeros(9, 256, device="cuda")
    x[1] = 1e-40                    # denormal
    x[2] = 3e38                     # largest magnitudes
    x[3, :128] = float("nan")
    x[4, 5] = float("inf")
    x[5, 200] = -float("inf")
    x[6, 0] = float("nan")
    x[7] = torch.finfo(torch.float32).min
    x[8, 130] = 1.0
    codes, scales = fp8.quantize(x)
    values = codes.float() * scales.repeat_interleave(128, 1)
    assert (codes[0].float() == 0).all() and torch.isfinite(scales[0]).all()
    for r in (1, 2, 7, 8):
        check_codes(codes[r:r + 1], scales[r:r + 1], x[r:r + 1].double())
    # a block that holds a NaN or an infinity stands for NaN; its neighbour is untouched
    for r, b in ((3, 0), (4, 0), (5, 1), (6, 0)):
        assert torch.isnan(values[r, 128 * b:128 * b + 128]).all()
        assert (values[r, 128 * (1 - b):128 * (1 - b) + 128] == 0).all()


def test_weight_special_values():
    w = randn(256, 256, seed=1)
    w[3, 7] = float("nan")
    w[200, 7] = float("inf")
    codes, scales = fp8.quantize_weight(w)
    values = codes.float() * scales.repeat_interleave(128, 0).repeat_interleave(128, 1)
    assert torch.isnan(values[:, :128]).all()
    check_codes(codes[:, 128:], scales[:, 1:], w[:, 128:].double(), rows=128)


def test_no_rows():
    x = torch.empty(0, 300, device="cuda")
    codes, scales = fp8.quantize(x)
    assert codes.shape == (0, 300) and scales.shape == (0, 3)
    codes, scales = fp8.rmsnorm(x, torch.ones(300, device="cuda"))
    assert codes.shape == (0, 300) and scales.shape == (0, 3)
    w, sw = fp8.quantize_weight(randn(40, 300))
    assert fp8.matmul(codes, scales, w, sw).shape == (0, 40)
    c, s = fp8.gated_matmul(codes, scales, w, sw, w, sw)
    assert c.shape == (0, 40) and s.shape == (0, 1)


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_rows_of_a_wider_matrix(offset):
    wide = randn(37, 1003, seed=5, dtype=torch.float16)
    x = wide[:, offset:offset + 700]
    codes, scales = fp8.quantize(x)
    check_codes(codes, scales, x.double())


def test_rows_offsets_past_32_bits():
    ld, m = 1 << 26, 40                       # last row starts at 2.6e9 elements
    x = torch.empty(m, ld, dtype=torch.float16, device="cuda")[:, :300]
    x.copy_(randn(m, 300, seed=6))
    codes, scales = fp8.quantize(x)
    check_codes(codes, scales, x.double())
    w = torch.ones(300, device="cuda")
    total, c2, s2 = fp8.rmsnorm(x, w, delta=x, out=x)
    d1, e1 = fp8.rmsnorm(total.contiguous(), w)
    assert torch.equal(c2.float(), d1.float()) and torch.equal(s2, e1)


# ---------------------------------------------------------------- RMSNorm

def norm_rel(k):
    """Relative f32 error of y: the sum of squares (at most k / 32 additions in
    a lane, 5 across lanes, 8 across warps, half of it after the root), the
    quotient, root, reciprocal and two products."""
    return ((k / 32 + 16) / 2 + 6) * U


@pytest.mark.parametrize("m,k", [(1, 1), (1, 768), (32, 768), (129, 768), (9, 1000), (5, 1025), (3, 2048), (7, 4099),
                                 (2, 8192), (3, 8200), (2, 20001)])
@pytest.mark.parametrize("dtype,delta", [("f32", None), ("f32", "f32"), ("f32", "f16"), ("f16", "f16"),
                                         ("bf16", "bf16"), ("bf16", "f32"), ("f16", None)])
def test_rmsnorm(m, k, dtype, delta):
    x = randn(m, k, seed=m, dtype=TYPES[dtype], scale=2.0)
    w = 1 + randn(k, seed=k, scale=0.2)
    eps = 1e-6
    if delta is None:
        codes, scales = fp8.rmsnorm(x, w, eps)
        t = x.double()
    else:
        d = randn(m, k, seed=m + 1, dtype=TYPES[delta])
        total, codes, scales = fp8.rmsnorm(x, w, eps, d)
        t32 = x.float() + d.float()  # one f32 rounding
        assert torch.equal(total, t32.to(x.dtype))
        t = t32.double()
    y = t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * w.double()
    check_codes(codes, scales, y, rel=norm_rel(k))


def test_rmsnorm_in_place_and_strided():
    wide = randn(50, 1541, seed=3)
    x, d = wide[:, 1:769], randn(50, 768, seed=4)
    w = torch.ones(768, device="cuda")
    keep, edge = x.clone(), wide[:, 769:].clone()
    total, codes, scales = fp8.rmsnorm(x, w, delta=d, out=x)
    assert total.data_ptr() == x.data_ptr() and torch.equal(x, keep + d) and torch.equal(wide[:, 769:], edge)
    c2, s2 = fp8.rmsnorm(x.contiguous(), w)
    assert torch.equal(codes.float(), c2.float()) and torch.equal(scales, s2)


def test_rmsnorm_zero_nan_rows():
    x = torch.zeros(4, 256, device="cuda")
    x[1, 9] = float("nan")
    x[2] = 1.0
    x[3, 9] = float("inf")
    codes, scales = fp8.rmsnorm(x, torch.ones(256, device="cuda"))
    v = codes.float() * scales.repeat_interleave(128, 1)
    assert (v[0] == 0).all() and torch.isnan(v[1]).all() and torch.isnan(v[3, :128]).all() and (v[3, 128:] == 0).all()
    assert (v[2] - 1).abs().max() < 1e-3


# ---------------------------------------------------------------- products

def operands(m, k, n, seed=0, mats=1):
    a, sa = fp8.quantize(randn(m, k, seed=seed, scale=1.5))
    ws = [fp8.quantize_weight(randn(n, k, seed=seed + 1 + i, scale=k ** -0.5)) for i in range(mats)]
    return a, sa, ws


def values64(codes, scales, rows):
    r, c = codes.shape
    return codes.double() * scales.double().repeat_interleave(rows, 0)[:r].repeat_interleave(128, 1)[:, :c]


def product64(a, sa, w, sw):
    """The product in 64 bits and a bound of the f32 error: every term passes
    at most 128 additions in its block (each good to 2^-23 however the tensor
    core rounds), one per block after that, and three roundings of the scale."""
    A, W = values64(a, sa, 1), values64(w, sw, 128)
    kb = sa.shape[1]
    return A @ W.T, (128 + kb + 8) * 2 * U * (A.abs() @ W.abs().T)


SIZES = [(1, 128, 128), (1, 768, 2304), (2, 100, 7), (5, 1, 1), (7, 129, 65), (8, 2048, 768), (16, 768, 768),
         (31, 1000, 300), (32, 768, 2304), (33, 768, 129), (64, 256, 512), (100, 640, 1000), (127, 127, 127),
         (128, 128, 256), (129, 384, 257), (200, 4096, 260), (300, 2048, 768), (511, 768, 768), (513, 1000, 1100),
         (1000, 130, 520), (2048, 768, 768), (1, 8192, 64), (32, 8192, 192), (4100, 256, 260)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_matmul(m, k, n, dtype):
    a, sa, [(w, sw)] = operands(m, k, n, seed=m + k + n)
    y = fp8.matmul(a, sa, w, sw, dtype)
    want, err = product64(a, sa, w, sw)
    assert y.dtype == dtype and y.shape == (m, n)
    assert ((y.double() - want).abs() <= err + ROUND[dtype] * (want.abs() + err) + 2.0 ** -25).all()


@pytest.mark.parametrize("m,k,n", [(1, 768, 768), (17, 300, 101), (32, 2048, 768), (129, 1000, 301), (700, 2048, 768),
                                   (2100, 256, 516)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_matmul_residual(m, k, n, dtype):
    a, sa, [(w, sw)] = operands(m, k, n, seed=m)
    r = randn(m, n, seed=9, dtype=dtype, scale=4.0)
    y = fp8.matmul(a, sa, w, sw, residual=r)
    want, err = product64(a, sa, w, sw)
    want = want + r.double()
    assert ((y.double() - want).abs() <= err + (U + ROUND[dtype]) * (want.abs() + err) + 2.0 ** -25).all()
    fp8.matmul(a, sa, w, sw, residual=r, out=r)   # in place: the same bits
    assert torch.equal(r, y)


def act64(g, act):
    if act == "silu":
        return g * torch.sigmoid(g)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def gated64(a, sa, gate, up, act):
    """h and its f32 error: both activations have slopes below 1.13; exp and
    the quotient are good to a few ulp of a number below |z| 2^-23 + 2^-21."""
    g, eg = product64(a, sa, *gate)
    u, eu = product64(a, sa, *up)
    h = act64(g, act) * u
    z = (g if act == "silu" else 1.6 * (g + 0.045 * g ** 3)).abs()
    return h, 1.13 * eg * (u.abs() + eu) + (act64(g, act).abs() + 1.13 * eg) * eu + (z.clamp_max(100) + 8) * 4 * U * h.abs() + 1e-30


@pytest.mark.parametrize("m,k,n", [(1, 768, 2048), (3, 100, 1), (8, 300, 130), (32, 768, 2048), (33, 256, 64),
                                   (130, 1000, 200), (257, 768, 2048), (600, 130, 385), (2100, 256, 640)])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "fp8"])
def test_gated(m, k, n, act, out):
    a, sa, (gate, up) = operands(m, k, n, seed=m + n, mats=2)
    h, err = gated64(a, sa, gate, up, act)
    if out == "fp8":
        codes, scales = fp8.gated_matmul(a, sa, *gate, *up, act=act)
        check_codes(codes, scales, h, err=err)
        return
    y = fp8.gated_matmul(a, sa, *gate, *up, out_dtype=TYPES[out], act=act)
    assert ((y.double() - h).abs() <= err + ROUND[TYPES[out]] * (h.abs() + err) + 2.0 ** -25).all()


@pytest.mark.parametrize("m", [3, 40, 700])
def test_products_keep_nan_and_inf_in_their_rows_and_columns(m):
    a, sa, [(w, sw), up] = operands(m, 300, 400, seed=m, mats=2)
    clean = fp8.matmul(a, sa, w, sw, torch.float32)
    sa2, sw2 = sa.clone(), sw.clone()
    sa2[1, 1] = float("nan")
    sw2[2, 0] = float("inf")
    y = fp8.matmul(a, sa2, w, sw2, torch.float32)
    good = torch.ones_like(y, dtype=torch.bool)
    good[1] = False
    good[:, 256:384] = False
    assert torch.equal(y[good], clean[good]) and not torch.isfinite(y[~good]).any()
    codes, scales = fp8.gated_matmul(a, sa2, w, sw, *up)
    c0, s0 = fp8.gated_matmul(a, sa, w, sw, *up)
    rows = torch.arange(m, device="cuda") != 1
    assert torch.equal(codes[rows].float(), c0[rows].float()) and torch.equal(scales[rows], s0[rows])
    assert torch.isnan(scales[1]).all()


def test_gate_far_from_zero():
    """Gates of -1e8..1e8: exp leaves the f32 range, the result does not."""
    g = torch.tensor([-1e8, -200.0, -20.0, 0.0, 20.0, 200.0, 1e8], device="cuda")
    x = torch.zeros(7, 128, device="cuda")
    x[:, 0] = 1.0
    a, sa = fp8.quantize(x)
    sa = sa * g.abs().clamp_min(1e-3)[:, None]
    a = torch.where((g < 0)[:, None], -a.float(), a.float()).to(torch.float8_e4m3fn)
    w = torch.zeros(64, 128, device="cuda")
    w[:, 0] = 1.0
    gate = fp8.quantize_weight(w)
    for act in ("gelu", "silu"):
        y = fp8.gated_matmul(a, sa, *gate, *gate, out_dtype=torch.float32, act=act).double()
        want, _ = gated64(a, sa, gate, gate, act)
        assert ((y - want).abs() <= 1e-4 * want.abs() + 1e-30).all()


@pytest.mark.parametrize("m", [2, 33, 300, 1300])
def test_strided_and_unaligned_operands(m):
    k, n = 270, 203
    wide_a, wide_w = fp8.empty_codes(m, 512, "cuda"), fp8.empty_codes(n, 640, "cuda")
    wide_a.view(torch.uint8).fill_(0x7F)     # NaN codes around the operands
    wide_w.view(torch.uint8).fill_(0x7F)
    a0, sa0, [(w0, sw0), _] = operands(m, k, n, seed=m, mats=2)
    a, w = wide_a[:, 16:16 + k], wide_w[:, 128:128 + k]
    a.copy_(a0)
    w.copy_(w0)
    sa = torch.full((m, 9), float("nan"), device="cuda")[:, 2:5]
    sa.copy_(sa0)
    sw = torch.full((sw0.shape[0], 7), float("nan"), device="cuda")[:, 1:4]
    sw.copy_(sw0)
    for dtype in TYPES.values():
        want = fp8.matmul(a0, sa0, w0, sw0, dtype)
        frame = torch.full((m + 2, n + 9), 7.0, dtype=dtype, device="cuda")
        out = frame[1:m + 1, 3:n + 3]
        fp8.matmul(a, sa, w, sw, dtype, out=out)
        assert torch.equal(out, want)
        frame[1:m + 1, 3:n + 3] = 7.0
        assert (frame == 7.0).all()
    c, s = fp8.gated_matmul(a, sa, w, sw, w, sw)
    c0, s0 = fp8.gated_matmul(a0, sa0, w0, sw0, w0, sw0)
    assert torch.equal(c.float(), c0.float()) and torch.equal(s, s0)


@pytest.mark.parametrize("n,start,res_start", [(701, 1, 6), (512, 3, 0), (513, 0, 5), (130, 7, 2), (6, 2, 3), (1, 5, 7)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_many_rows_off_the_boundary(n, start, res_start, dtype):
    """Rows of results and of the residual that start anywhere in a 16-byte
    block, each at its own place; what surrounds them stays as it is."""
    m, k = 8003, 140
    a, sa, (gate, up) = operands(m, k, n, seed=n, mats=2)
    frame = torch.full((m + 1, n + 11), 7.0, dtype=dtype, device="cuda")
    out = frame[1:, start:start + n]
    res = randn(m, n + 9, seed=start, dtype=dtype)[:, res_start:res_start + n]

    def near(y, want, err):
        return ((y.double() - want).abs() <= err + ROUND[dtype] * (want.abs() + err) + 2.0 ** -25).all()

    def check(want, err):
        assert near(out, want, err)
        out.fill_(7.0)
        assert (frame == 7.0).all()

    y, err = product64(a, sa, *gate)
    fp8.matmul(a, sa, *gate, dtype, out=out)
    check(y, err)
    fp8.matmul(a, sa, *gate, dtype, residual=res, out=out)
    y = y + res.double()
    check(y, err + U * y.abs())
    out.copy_(res)
    fp8.matmul(a, sa, *gate, dtype, residual=out, out=out)
    check(y, err + U * y.abs())
    assert near(fp8.gated_matmul(a, sa, *gate, *up, out_dtype=dtype), *gated64(a, sa, gate, up, "gelu"))


@pytest.mark.parametrize("m", [3, 130, 5000])
@pytest.mark.parametrize("n", [64, 100, 129, 250, 328])
def test_codes_end_where_the_row_ends(m, n):
    """8-bit rows into wider ones: the bytes behind them stay as they are."""
    k, ld = 300, 384
    a, sa, (gate, up) = operands(m, k, n, seed=n, mats=2)
    x, w = randn(m, n, seed=1), torch.ones(n, device="cuda")
    frame = torch.empty(m, ld, dtype=torch.uint8, device="cuda")
    scales = torch.empty(m, 5, device="cuda")
    blocks = -(-n // 128)

    def check(call, codes, s):
        frame.fill_(0x55)
        scales.fill_(7.0)
        assert call(frame.data_ptr(), ld, scales.data_ptr(), 5) == 0
        torch.cuda.synchronize()
        assert torch.equal(frame[:, :n], codes.view(torch.uint8)) and (frame[:, n:] == 0x55).all()
        assert torch.equal(scales[:, :blocks], s) and (scales[:, blocks:] == 7.0).all()

    f32, e4m3, stream = 0, 3, torch.cuda.current_stream().cuda_stream
    mat = lambda t: (t.data_ptr(), t.stride(0))
    check(lambda c, ldc, s, lds: lib().wc_fp8_quantize_rows(x.data_ptr(), f32, m, n, n, c, ldc, s, lds, stream),
          *fp8.quantize(x))
    check(lambda c, ldc, s, lds: lib().wc_fp8_rmsnorm(x.data_ptr(), f32, n, None, f32, 0, None, 0, w.data_ptr(), m, n, 1e-6,
                                                      c, ldc, s, lds, stream), *fp8.rmsnorm(x, w))
    check(lambda c, ldc, s, lds: lib().wc_fp8_gated_matmul(
        *mat(a), *mat(sa), m, k, *mat(gate[0]), *mat(gate[1]), *mat(up[0]), *mat(up[1]), n, 0, c, e4m3, ldc, s, lds, stream),
        *fp8.gated_matmul(a, sa, *gate, *up))


def test_product_offsets_past_32_bits():
    m = n = 40
    k, ld = 300, 1 << 26
    a0, sa, [(w0, sw)] = operands(m, k, n)
    a, w = fp8.empty_codes(m, ld, "cuda")[:, :k], fp8.empty_codes(n, ld, "cuda")[:, :k]
    a.copy_(a0)
    w.copy_(w0)
    out = torch.empty(m, ld, dtype=torch.float16, device="cuda")[:, :n]
    fp8.matmul(a, sa, w, sw, out=out)
    assert torch.equal(out, fp8.matmul(a0, sa, w0, sw))


@pytest.mark.parametrize("m,k,n", [(1, 2048, 768), (32, 768, 2304), (300, 2048, 768), (1500, 768, 2304)])
def test_same_bits_every_time(m, k, n):
    a, sa, (gate, up) = operands(m, k, n, mats=2)
    y = fp8.matmul(a, sa, *gate, torch.float32)
    c, s = fp8.gated_matmul(a, sa, *gate, *up)
    for _ in range(5):
        assert torch.equal(fp8.matmul(a, sa, *gate, torch.float32), y)
        c2, s2 = fp8.gated_matmul(a, sa, *gate, *up)
        assert torch.equal(c2.float(), c.float()) and torch.equal(s2, s)


def test_order_on_another_stream():
    """A chain of calls behind slow work on a side stream sees its inputs."""
    m, k, f = 600, 768, 2048
    x0, w = randn(m, k, seed=1), torch.ones(k, device="cuda")
    gate, up = (fp8.quantize_weight(randn(f, k, seed=i, scale=0.03)) for i in (2, 3))
    wo32 = randn(k, f, seed=4, scale=0.02)

    def chain(x):
        wo = fp8.quantize_weight(wo32)           # produced by the call before it is read
        codes, scales = fp8.rmsnorm(x, w)
        codes, scales = fp8.gated_matmul(codes, scales, *gate, *up)
        return fp8.matmul(codes, scales, *wo, residual=x)

    want = chain(x0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.zeros_like(x0)
        big = randn(4096, 4096, seed=5)
        for _ in range(20):
            big = big @ big * 1e-3
        x.copy_(x0)
        got = [chain(x) for _ in range(3)]
    fp8.synchronize()
    side.synchronize()
    for y in got:
        assert torch.equal(y, want)


def test_refusals_on_the_gpu():
    x = randn(4, 256)
    a, sa = fp8.quantize(x)
    w, sw = fp8.quantize_weight(randn(8, 256))
    with pytest.raises(ValueError, match="float8"):
        fp8.matmul(x, sa, w, sw)
    with pytest.raises(ValueError, match="expected"):
        fp8.matmul(a, sa[:, :1], w, sw)
    with pytest.raises(ValueError, match="expected"):
        fp8.matmul(a[:, :128], sa[:, :1], w, sw)
    with pytest.raises(ValueError, match="scales of a"):
        fp8.matmul(a, sa.double(), w, sw)
    with pytest.raises(ValueError, match="out_dtype"):
        fp8.matmul(a, sa, w, sw, torch.float64)
    with pytest.raises(ValueError, match="out is"):
        fp8.matmul(a, sa, w, sw, torch.float16, out=torch.empty(4, 8, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        fp8.matmul(a, sa, w, sw, residual=torch.empty(4, 9, device="cuda"))
    with pytest.raises(ValueError, match="act"):
        fp8.gated_matmul(a, sa, w, sw, w, sw, act="relu")
    with pytest.raises(ValueError, match="up"):
        fp8.gated_matmul(a, sa, w, sw, w[:4], sw)
    with pytest.raises(ValueError, match="contiguous rows"):
        fp8.quantize(x.T)
    with pytest.raises(ValueError, match="weight"):
        fp8.rmsnorm(x, torch.ones(255, device="cuda"))
    with pytest.raises(ValueError, match="delta"):
        fp8.rmsnorm(x, torch.ones(256, device="cuda"), out=x)
    with pytest.raises(fp8.WcError, match="16 bytes"):    # rows of codes that start off the boundary
        fp8.matmul(torch.empty(4, 260, dtype=torch.float8_e4m3fn, device="cuda")[:, :256], sa, w, sw)
    with pytest.raises(fp8.WcError, match="16 bytes"):
        fp8.matmul(fp8.empty_codes(4, 512, "cuda")[:, 8:264], sa, w, sw)


# ---------------------------------------------------------------- the operators together

@pytest.mark.parametrize("tokens", [1, 32, 700])
def test_feed_forward_example(tiny_model, tokens):
    """The example's block (norm, gate, product) against the same block in f32.

    Every code is off by at most 2^-4 of its value (3 fraction bits), about
    evenly spread: 2^-4 / sqrt(3) = 0.036 in the mean square at worst.  The first product has two
    such factors (0.051); the gate multiplies two results of it (slope of GELU
    at most 1.13: 0.077), its rows are rounded again (0.085 with 0.036), and the
    last weights too (0.093).  Twice that bounds what the block adds."""
    import importlib.util
    import os
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("fp8_feed_forward",
                                                  os.path.join(ROOT, "examples", "fp8_feed_forward.py"))
    example = importlib.util.module_from_spec(spec)
    import sys
    sys.modules[spec.name] = example
    spec.loader.exec_module(example)
    block = example.FeedForward.load(tiny_model, 1)
    d = tiny_model.config.d_model
    x, attention = randn(tokens, d, seed=tokens), randn(tokens, d, seed=2, dtype=torch.float16)
    keep = x.clone()
    y, want = block(x, attention), example.reference(tiny_model, 1, x, attention)
    assert torch.equal(x, keep)
    added = want - x - attention.float()
    assert float((y - want).norm() / added.norm()) < 0.19
    fp8.synchronize()
