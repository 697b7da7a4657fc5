"""Scales of 4-bit floating point matrices that are unusual: every byte that a checkpoint may hold, on both sides of the line between
the products' kernels."""
import numpy as np
import pytest

import fp4_plain as F

pytestmark = pytest.mark.gpu

# rows of activations whose products with 512 x 512 weights are the CUDA cores' and the tensor cores'
FEW, MANY = 3, 300


def _put(dev, ty, codes, sb):
    rows, cols = codes.shape
    size = dev.lib.q4_cuda_fp4_bytes(ty, F.WEIGHTS, rows, cols)
    d = dev.upload(np.full(size, 0x55, np.uint8))
    assert dev.lib.q4_cuda_fp4_put(ty, dev.upload(F.packed(codes)), dev.upload(sb), rows, cols, 1, d, 0)
    return d, size


def test_negative_scales_of_a_checkpoint(dev):
    """All 256 bytes: the values are the signed ones, the buffer holds no sign (the tensor cores' e4m3 scales have none), and products
    with few rows and with many agree with the values."""
    lib, ty, w_rows, cols = dev.lib, F.NVFP4, 512, 512
    rng = np.random.default_rng(1)
    codes = rng.integers(0, 16, (w_rows, cols), dtype=np.uint8)
    sb = rng.integers(0, 256, (w_rows, cols // 16), dtype=np.uint8)
    sb[0, :] = np.arange(32) * 8 + 7                       # 0x7f and 0xff among them
    sb[1:9] = np.arange(256).reshape(8, 32)
    want = F.values(ty, codes, sb)
    d_w, size = _put(dev, ty, codes, sb)
    held = dev.download(d_w, (size,), np.uint8)[w_rows * cols // 2:]
    assert (held < 128).all()
    d_v = dev.malloc(w_rows * cols * 4)
    assert lib.q4_cuda_fp4_values(ty, F.WEIGHTS, d_w, w_rows, cols, d_v, cols)
    np.testing.assert_array_equal(dev.download(d_v, (w_rows, cols), np.float32), want.astype(np.float32))
    for rows in (FEW, MANY):
        x = rng.standard_normal((rows, cols)).astype(np.float32) * 30
        d_x = dev.malloc(lib.q4_cuda_fp4_bytes(ty, F.ROWS, rows, cols))
        assert lib.q4_cuda_fp4_quantize(ty, F.ROWS, dev.upload(x), cols, 1.0, rows, cols, d_x)
        d_y = dev.malloc(rows * w_rows * 4)
        assert lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_x, rows, 1.0, d_y, w_rows)
        y = dev.download(d_y, (rows, w_rows), np.float32)
        xv = F.values(ty, *F.quantise(ty, x.astype(np.float64)))
        nan = np.isnan(want).any(axis=1)
        assert nan.any() and not nan.all() and (np.isnan(y) == nan[None, :]).all()
        w = want[~nan]
        assert (np.abs(y[:, ~nan] - xv @ w.T) <= F.product_bound(xv, w, 1.0, cols // 16)).all()
    assert lib.q4_cuda_device_error() == 0
