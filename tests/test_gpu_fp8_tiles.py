"""8-bit products with several tiles to a pair of SMs, so that what one tile
leaves behind (staging rooms, barriers' parities, block maxima) meets the next
one.  Against 64 bits, with the bounds of test_gpu_fp8.py."""
import pytest
import torch

from test_gpu_fp8 import ROUND, TYPES, U, check_codes, gated64, operands, product64, randn
from witchcraft_b200 import fp8
from witchcraft_b200._lib import lib

pytestmark = pytest.mark.gpu

# 74 pairs: 256 tiles of 256 x 256 columns (or of 128 gated features) are three
# or four to a pair; 150 are two or three, with ragged ends both ways.
PLAIN = [(16384, 64, 1024), (16384, 128, 1024), (16384, 256, 1024), (6300, 300, 1360)]
GATED = [(16384, 64, 512), (16384, 128, 512), (16384, 256, 512), (6300, 300, 688)]


CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}


def on_pairs(m, k, n, dtype, gated=False, residual=False, boxes=True):
    """Fails where the library would take the kernel for few rows."""
    assert lib().wc_selftest_fp8_split(gated, m, k, n, CODE[dtype], residual, boxes) == 0
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert -(-m // 256) * -(-n // (128 if gated else 256)) > pairs       # more than one tile to a pair


def near(y, want, err):
    return ((y.double() - want).abs() <= err + ROUND[y.dtype] * (want.abs() + err) + 2.0 ** -25).all()


@pytest.mark.parametrize("m,k,n", PLAIN)
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_boxes_of_results(m, k, n, dtype):
    """The rooms of the boxes start over with every tile: a tile's last boxes
    have to be read before the next one's are written."""
    on_pairs(m, k, n, dtype)
    a, sa, [(w, sw)] = operands(m, k, n, seed=k)
    want, err = product64(a, sa, w, sw)
    for _ in range(3):
        assert near(fp8.matmul(a, sa, w, sw, dtype), want, err)


@pytest.mark.parametrize("m,k,n", GATED)
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_boxes_of_gated_results(m, k, n, dtype):
    on_pairs(m, k, n, dtype, gated=True)
    a, sa, (gate, up) = operands(m, k, n, seed=k, mats=2)
    want, err = gated64(a, sa, gate, up, "gelu")
    for _ in range(3):
        assert near(fp8.gated_matmul(a, sa, *gate, *up, out_dtype=dtype), want, err)


@pytest.mark.parametrize("m,n", [(20001, 3), (20001, 1), (20001, 129), (20001, 257), (20001, 130)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("offset", [0, 2])
def test_residual_of_adjoining_rows(m, n, dtype, offset):
    """Rows without a gap, off the 16-byte boundary, some of them several to a
    block: the residual's own values and nothing of its neighbours."""
    on_pairs(m, 140, n, dtype, residual=True, boxes=False)
    a, sa, [(w, sw)] = operands(m, 140, n, seed=n)
    flat = torch.full((m * n + 16,), float("nan"), dtype=dtype, device="cuda")
    res = flat[4 + offset:4 + offset + m * n].view(m, n)
    res.copy_(randn(m, n, seed=1, dtype=dtype))
    want, err = product64(a, sa, w, sw)
    want = want + res.double()
    err = err + U * want.abs()
    assert near(fp8.matmul(a, sa, w, sw, residual=res), want, err)
    fp8.matmul(a, sa, w, sw, residual=res, out=res)
    assert near(res, want, err)
    assert torch.isnan(flat[:4 + offset]).all() and torch.isnan(flat[4 + offset + m * n:]).all()


@pytest.mark.parametrize("m,k,n", PLAIN)
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_boxes_of_the_residual(m, k, n, dtype):
    """Each box's barrier is used again by the next tile, with the other parity."""
    on_pairs(m, k, n, dtype, residual=True)
    a, sa, [(w, sw)] = operands(m, k, n, seed=k)
    r = randn(m, n, seed=2, dtype=dtype, scale=4.0)
    want, err = product64(a, sa, w, sw)
    want = want + r.double()
    err = err + U * want.abs()
    y = fp8.matmul(a, sa, w, sw, residual=r)
    assert near(y, want, err)
    for _ in range(3):
        assert torch.equal(fp8.matmul(a, sa, w, sw, residual=r), y)
    fp8.matmul(a, sa, w, sw, residual=r, out=r)
    assert torch.equal(r, y)


@pytest.mark.parametrize("m,k,n", GATED + [(16384, 256, 520), (9000, 200, 601)])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gated_codes(m, k, n, act):
    """Block maxima meet in shared memory that the tile before last has used;
    n off 128 and off 16."""
    on_pairs(m, k, n, torch.float8_e4m3fn, gated=True)
    a, sa, (gate, up) = operands(m, k, n, seed=n, mats=2)
    codes, scales = fp8.gated_matmul(a, sa, *gate, *up, act=act)
    h, err = gated64(a, sa, gate, up, act)
    check_codes(codes, scales, h, err=err)
    for _ in range(3):
        c, s = fp8.gated_matmul(a, sa, *gate, *up, act=act)
        assert torch.equal(c.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s, scales)


@pytest.mark.parametrize("boxes", [True, False])
def test_offsets_past_32_bits(boxes):
    """Operands, residual and results whose last rows lie past 2^31 elements."""
    m, k, n, ld = 20000, 140, 264, 1 << 17
    start = 0 if boxes else 3
    on_pairs(m, k, n, torch.float16, residual=True, boxes=boxes)
    a0, sa0, [(w, sw)] = operands(m, k, n)
    a = fp8.empty_codes(m, ld, "cuda")[:, :k]
    a.copy_(a0)
    sa = torch.empty(m, ld, device="cuda")[:, :2]
    sa.copy_(sa0)
    frame = torch.empty(m, ld, dtype=torch.float16, device="cuda")
    r, y = frame[:, start:start + n], frame[:, 8192 + start:8192 + start + n]
    r.copy_(randn(m, n, seed=3))
    fp8.matmul(a, sa, w, sw, residual=r, out=y)
    want, err = product64(a0, sa0, w, sw)
    want = want + r.double()
    assert near(y, want, err + U * want.abs())


def test_choice():
    """Few rows on single tiles, many on pairs, and refusals of the query."""
    split = lib().wc_selftest_fp8_split
    for gated in (0, 1):
        assert split(gated, 1, 768, 768, 1, 0, 1) in (1, 2, 4, 8)
        assert split(gated, 16384, 768, 2304, 1, 0, 1) == 0
    for bad in ((0, 0, 768, 768, 1, 0, 1), (0, 4, 0, 768, 1, 0, 1), (0, 4, 768, 768, 3, 0, 1), (1, 4, 768, 768, 4, 0, 1)):
        assert split(*bad) == -1
