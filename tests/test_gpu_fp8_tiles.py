"""8-bit products with several tiles to a pair of SMs, so that what one tile
leaves behind (staging rooms, barriers' parities, block maxima) meets the next
one.  Against 64 bits, with the bounds of test_gpu_fp8.py."""
import pytest
import torch

from test_gpu_fp8 import ROUND, TYPES, U, gated64, operands, product64, randn
from witchcraft_b200 import fp8

pytestmark = pytest.mark.gpu

# 74 pairs: 256 tiles of 256 x 256 columns (or of 128 gated features) are three
# or four to a pair; 150 are two or three, with ragged ends both ways.
PLAIN = [(16384, 64, 1024), (16384, 128, 1024), (16384, 256, 1024), (6300, 300, 1360)]
GATED = [(16384, 64, 512), (16384, 128, 512), (16384, 256, 512), (6300, 300, 688)]


def near(y, want, err):
    return ((y.double() - want).abs() <= err + ROUND[y.dtype] * (want.abs() + err) + 2.0 ** -25).all()


@pytest.mark.parametrize("m,k,n", PLAIN)
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_boxes_of_results(m, k, n, dtype):
    """The rooms of the boxes start over with every tile: a tile's last boxes
    have to be read before the next one's are written."""
    a, sa, [(w, sw)] = operands(m, k, n, seed=k)
    want, err = product64(a, sa, w, sw)
    for _ in range(3):
        assert near(fp8.matmul(a, sa, w, sw, dtype), want, err)


@pytest.mark.parametrize("m,k,n", GATED)
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_boxes_of_gated_results(m, k, n, dtype):
    a, sa, (gate, up) = operands(m, k, n, seed=k, mats=2)
    want, err = gated64(a, sa, gate, up, "gelu")
    for _ in range(3):
        assert near(fp8.gated_matmul(a, sa, *gate, *up, out_dtype=dtype), want, err)


@pytest.mark.parametrize("m,n", [(20001, 3), (20001, 1), (8002, 129), (8002, 257), (8002, 130)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("offset", [0, 2])
def test_residual_of_adjoining_rows(m, n, dtype, offset):
    """Rows without a gap, off the 16-byte boundary, some of them several to a
    block: the residual's own values and nothing of its neighbours."""
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
