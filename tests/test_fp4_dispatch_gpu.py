"""Which kernel a 4-bit product runs on, and calls that may not depend on it."""
import numpy as np
import pytest

import fp4_plain as F

pytestmark = pytest.mark.gpu

TYPES = [F.MXFP4, F.NVFP4]


def _weights(dev, rng, ty, rows, cols):
    codes = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
    sb = rng.integers(0x50, 0x58, (rows, cols // F.BLOCK[ty]), dtype=np.uint8) + np.uint8(40 if ty == F.MXFP4 else 0)
    d = dev.malloc(dev.lib.q4_cuda_fp4_bytes(ty, F.WEIGHTS, rows, cols))
    assert dev.lib.q4_cuda_fp4_put(ty, dev.upload(F.packed(codes)), dev.upload(sb), rows, cols, 1, d, 0)
    return F.values(ty, codes, sb), d


def _rows(dev, rng, ty, rows, cols):
    x = (rng.standard_normal((rows, cols)) * 30).astype(np.float32)
    d = dev.malloc(dev.lib.q4_cuda_fp4_bytes(ty, F.ROWS, rows, cols))
    assert dev.lib.q4_cuda_fp4_quantize(ty, F.ROWS, dev.upload(x), cols, 1.0, rows, cols, d)
    return F.values(ty, *F.quantise(ty, x.astype(np.float64))), d


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("stride", [0, 16, 1 << 41])
def test_the_stride_of_one_matrix_is_not_looked_at(dev, ty, rows, stride):
    rng = np.random.default_rng(rows)
    w, d_w = _weights(dev, rng, ty, 512, 512)
    x, d_x = _rows(dev, rng, ty, rows, 512)
    d_y = dev.malloc(rows * 512 * 4)
    d_b = dev.upload(np.array([0, rows], np.int32))
    assert dev.lib.q4_cuda_fp4_mul_id(ty, d_w, 512, 512, stride, 1, d_x, rows, None, d_b, rows, 1.0, None, d_y, 512)
    y = dev.download(d_y, (rows, 512), np.float32)
    assert (np.abs(y - x @ w.T) <= F.product_bound(x, w, 1.0, 512 // F.BLOCK[ty])).all()
    assert dev.lib.q4_cuda_device_error() == 0
