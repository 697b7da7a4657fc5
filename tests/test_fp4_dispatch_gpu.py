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


def _ran(dev, before=None):
    n = np.zeros(3, np.uint64)
    dev.lib.q4_cuda_fp4_products(n.ctypes.data)
    return n if before is None else (n - before).tolist()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,w_rows,cols,kind", [
    (1, 4096, 2048, 0), (2, 4096, 2048, 0), (3, 4096, 2048, 1), (1, 33, 65536, 0), (3, 512, 512, 0), (300, 512, 512, 1), (777, 640, 352, 1),
    (140, 130, 65536, 1), (1300, 513, 32, 1), (700, 129, 352, 1), (1500, 257, 4096, 1), (4111, 6801, 96, 2), (4352, 7104, 320, 2), (4190, 7000, 32, 2)])
def test_products_run_where_they_should(dev, ty, rows, w_rows, cols, kind):
    """Codes of any block against any other's, all scales 1: every partial sum is a multiple of 1/4 below 2^22 (65536 products of at most 36),
    an fp32 number, so that the result is exact in whatever order it is added up; a lost block, or one that is taken twice, shows."""
    lib = dev.lib
    rng = np.random.default_rng(rows + cols)
    b = F.BLOCK[ty]

    def codes(n):
        c = rng.integers(0, 16, (n, cols), dtype=np.uint8)
        c[:, rng.integers(0, b):: b] = 7               # 6: the largest, and the scale 1, of every block
        return c

    cw, cx = codes(w_rows), codes(rows)
    one = np.uint8(127 if ty == F.MXFP4 else 0x38)
    d_w, d_x = (dev.malloc(lib.q4_cuda_fp4_bytes(ty, f, n, cols)) for f, n in ((F.WEIGHTS, w_rows), (F.ROWS, rows)))
    d_c, d_s, d_v = dev.upload(F.packed(cw)), dev.upload(np.full((w_rows, cols // b), one)), dev.upload(
        F.values(ty, cx, np.full((rows, cols // b), one)).astype(np.float32))
    assert lib.q4_cuda_fp4_put(ty, d_c, d_s, w_rows, cols, 1, d_w, 0)
    assert lib.q4_cuda_fp4_quantize(ty, F.ROWS, d_v, cols, 1.0, rows, cols, d_x)
    want = F.values(ty, cx, np.full((rows, cols // b), one)) @ F.values(ty, cw, np.full((w_rows, cols // b), one)).T
    d_y = dev.malloc(rows * w_rows * 4)
    d_b = dev.upload(np.array([0, rows], np.int32))
    before = _ran(dev)
    assert lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_x, rows, 1.0, d_y, w_rows)
    assert _ran(dev, before) == [int(i == kind) for i in range(3)]
    assert (dev.download(d_y, (rows, w_rows), np.float32) == want).all()
    assert lib.q4_hip_fill(d_y, float("nan"), rows * w_rows)
    before = _ran(dev)
    assert lib.q4_cuda_fp4_mul_id(ty, d_w, w_rows, cols, 0, 1, d_x, rows, None, d_b, rows, 1.0, None, d_y, w_rows)
    assert _ran(dev, before) == [int(i == min(kind, 1)) for i in range(3)]       # (pairs are for dense products)
    assert (dev.download(d_y, (rows, w_rows), np.float32) == want).all()
    for d in (d_w, d_x, d_c, d_s, d_v, d_y, d_b):
        dev.free(d)
    assert lib.q4_cuda_device_error() == 0


def test_refused_and_empty_products_are_not_counted(dev):
    lib, d = dev.lib, dev.malloc(1 << 16)
    before = _ran(dev)
    assert not lib.q4_cuda_fp4_mul(F.MXFP4, d, 64, 64, d, 4, 1.0, d, 63)
    assert lib.q4_cuda_fp4_mul_id(F.MXFP4, d, 64, 64, 0, 1, d, 4, None, d, 0, 1.0, None, d, 64)
    lib.q4_cuda_fp4_products(None)
    assert _ran(dev, before) == [0, 0, 0]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,kind", [(3, 0), (300, 1)])
def test_blocks_without_a_number(dev, ty, rows, kind):
    """A NaN block of the weights is in its column, one of the activations (a NaN or an infinity in a row) in its row, nothing beside them."""
    lib, w_rows, cols = dev.lib, 512, 512
    rng = np.random.default_rng(rows)
    codes = rng.integers(0, 16, (w_rows, cols), dtype=np.uint8)
    sb = rng.integers(0x50, 0x58, (w_rows, cols // F.BLOCK[ty]), dtype=np.uint8)
    for r, c in ((0, 0), (130, 7), (511, cols // F.BLOCK[ty] - 1)):
        sb[r, c] = 255 if ty == F.MXFP4 else 127
    codes[130, 7 * F.BLOCK[ty]:8 * F.BLOCK[ty]] = 0                 # NaN times nothing but zeros
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x[1, 77], x[rows - 1, 511] = np.nan, -np.inf
    d_w, d_x = (dev.malloc(lib.q4_cuda_fp4_bytes(ty, f, n, cols)) for f, n in ((F.WEIGHTS, w_rows), (F.ROWS, rows)))
    assert lib.q4_cuda_fp4_put(ty, dev.upload(F.packed(codes)), dev.upload(sb), w_rows, cols, 1, d_w, 0)
    assert lib.q4_cuda_fp4_quantize(ty, F.ROWS, dev.upload(x), cols, 8.0, rows, cols, d_x)
    d_y = dev.malloc(rows * w_rows * 4)
    before = _ran(dev)
    assert lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_x, rows, 1.0, d_y, w_rows)
    assert _ran(dev, before)[kind] == 1
    y = dev.download(d_y, (rows, w_rows), np.float32)
    with np.errstate(invalid="ignore"):
        xv = F.values(ty, *F.quantise(ty, (x * np.float32(8.0)).astype(np.float64)))
    wv = F.values(ty, codes, sb)
    want = xv @ wv.T
    nan = np.isnan(xv).any(axis=1)[:, None] | np.isnan(wv).any(axis=1)[None, :]
    assert nan.sum() == 2 * w_rows + 3 * rows - 6 and (np.isnan(y) == nan).all()
    bound = F.product_bound(np.nan_to_num(xv), np.nan_to_num(wv), 1.0, cols // F.BLOCK[ty])
    assert (np.abs(y - want)[~nan] <= bound[~nan]).all()


@pytest.mark.parametrize("w_rows,cols,rows,kind", [(64, 128, 32, 0), (64, 128, 1184, 1), (1000, 32, 9, 0), (1000, 32, 64, 1), (8192, 128, 1, 0), (8192, 128, 8, 1),
                                                   (1024, 1024, 8, 0), (1024, 1024, 12, 1), (128, 4096, 8, 0), (128, 4096, 75, 1)])
def test_narrow_matrices_leave_the_cuda_cores_in_time(dev, w_rows, cols, rows, kind):
    """A CTA of the CUDA cores' kernel costs about the same with 32 columns as with 2048: what counts is how many there are."""
    lib, ty = dev.lib, F.MXFP4
    rng = np.random.default_rng(rows)
    w, d_w = _weights(dev, rng, ty, w_rows, cols)
    x, d_x = _rows(dev, rng, ty, rows, cols)
    d_y = dev.malloc(rows * w_rows * 4)
    before = _ran(dev)
    assert lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_x, rows, 1.0, d_y, w_rows)
    assert _ran(dev, before) == [int(i == kind) for i in range(3)]
    y = dev.download(d_y, (rows, w_rows), np.float32)
    assert (np.abs(y - x @ w.T) <= F.product_bound(x, w, 1.0, cols // 32)).all()
    assert lib.q4_cuda_device_error() == 0
