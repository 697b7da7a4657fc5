"""4-bit floating point (MXFP4, NVFP4): quantisers, layouts and products against a plain implementation in 64 bits.

Quantised values are compared exactly.  Products: the bound of fp4_plain.product_bound, which counts the roundings."""
import numpy as np
import pytest

import fp4_plain as F

pytestmark = pytest.mark.gpu

TYPES = [F.MXFP4, F.NVFP4]
SENTINEL = np.float32(-12345.0)


def _buffer(dev, ty, form, rows, cols, n=1):
    size = dev.lib.q4_cuda_fp4_bytes(ty, form, rows, cols)
    assert size
    d = dev.malloc(n * size)
    assert dev.lib.q4_hip_fill(d, float("nan"), n * size // 4)      # whatever was there before
    return d, size


def _values(dev, ty, form, d, rows, cols, ld=None):
    ld = ld or cols
    d_out = dev.upload(np.full((rows, ld), SENTINEL, np.float32))
    assert dev.lib.q4_cuda_fp4_values(ty, form, d, rows, cols, d_out, ld)
    out = dev.download(d_out, (rows, ld), np.float32)
    assert (out[:, cols:] == SENTINEL).all()
    dev.free(d_out)
    return out[:, :cols]


def _weights(dev, rng, ty, n, rows, cols, spread=6):
    """n random matrices: their values in 64 bits, and the device buffer."""
    codes = rng.integers(0, 16, (n, rows, cols), dtype=np.uint8)
    mid = 120 if ty == F.MXFP4 else 0x50
    sb = rng.integers(mid, mid + spread, (n, rows, cols // F.BLOCK[ty]), dtype=np.uint8)
    d, size = _buffer(dev, ty, F.WEIGHTS, rows, cols, n)
    d_c, d_s = dev.upload(F.packed(codes)), dev.upload(sb)
    assert dev.lib.q4_cuda_fp4_put(ty, d_c, d_s, rows, cols, n, d, size)
    dev.sync()
    dev.free(d_c), dev.free(d_s)
    return F.values(ty, codes, sb), d, size


def _rows(dev, rng, ty, rows, cols, mul=1.0):
    """Random quantised activations: their values and the device buffer."""
    x = rng.standard_normal((rows, cols)).astype(np.float32) * rng.uniform(0.2, 4.0, (rows, 1)).astype(np.float32)
    d, _ = _buffer(dev, ty, F.ROWS, rows, cols)
    d_x = dev.upload(x)
    assert dev.lib.q4_cuda_fp4_quantize(ty, F.ROWS, d_x, cols, mul, rows, cols, d)
    dev.sync()
    dev.free(d_x)
    return F.values(ty, *F.quantise(ty, (x * np.float32(mul)).astype(np.float64))), d


def _hard_rows(rng, ty, rows, cols):
    """Random rows with blocks in which something can go wrong."""
    x = (rng.standard_normal((rows, cols)) * 10.0 ** rng.integers(-3, 4, (rows, cols // 32)).repeat(32, axis=1)).astype(np.float32)
    b = x.reshape(-1, 32)
    tie = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float32)
    special = [
        lambda v: v * 0, lambda v: v * 0 + np.float32(1e-45), lambda v: v * np.float32(1e-42), lambda v: v * 0 + np.float32(F.FMAX),
        lambda v: np.tile(tie, 4) * np.float32(2.0 ** -3), lambda v: -np.nextafter(np.tile(tie, 4), np.float32(9)),
        lambda v: np.nextafter(np.tile(tie, 4), np.float32(0)) * np.float32(6.5), lambda v: np.where(np.arange(32) == 5, np.nan, v),
        lambda v: np.where(np.arange(32) == 31, np.inf, v), lambda v: np.where(np.arange(32) == 0, -np.inf, v),
        lambda v: np.where(np.arange(32) == 17, np.float32(1e30), v), lambda v: v * 0 - np.float32(0.0), lambda v: v * 0 + np.float32(2.0 ** -126),
        lambda v: v * 0 + np.float32(7.999999), lambda v: v * 0 + np.float32(3.0 * 2.0 ** -10), lambda v: v * 0 + np.float32(6.0 * 17.0 / 16.0)]
    with np.errstate(invalid="ignore", over="ignore"):
        for i, f in enumerate(special):
            if i < len(b):
                b[(i * 7) % len(b)] = f(b[(i * 7) % len(b)])
    return b.reshape(rows, cols).astype(np.float32)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("form", [F.ROWS, F.WEIGHTS])
@pytest.mark.parametrize("rows,cols,extra,shift,mul", [(1, 32, 0, 0, 1.0), (3, 96, 4, 0, 1.0), (33, 256, 3, 1, 0.37), (130, 288, 0, 0, 224.0),
                                                     (7, 2048, 32, 2, -1.5), (260, 544, 0, 0, 1.0), (1, 65536, 0, 0, 1.0)])
def test_quantize_is_the_definition(dev, ty, form, rows, cols, extra, shift, mul):
    rng = np.random.default_rng(rows * cols)
    x = _hard_rows(rng, ty, rows, cols)
    ld = cols + extra
    flat = np.full(rows * ld + shift, 1e9, np.float32)
    flat[shift:].reshape(rows, ld)[:, :cols] = x
    d_x = dev.upload(flat)
    d, _ = _buffer(dev, ty, form, rows, cols)
    assert dev.lib.q4_cuda_fp4_quantize(ty, form, d_x + 4 * shift, ld, mul, rows, cols, d)
    with np.errstate(invalid="ignore", over="ignore"):
        want = F.values(ty, *F.quantise(ty, (x * np.float32(mul)).astype(np.float64))).astype(np.float32)
    got = _values(dev, ty, form, d, rows, cols, cols + (extra if extra != 4 else 0))
    np.testing.assert_array_equal(got, want)
    assert np.isnan(want).any() or rows * cols < 500
    dev.free(d), dev.free(d_x)


@pytest.mark.parametrize("ty", TYPES)
def test_quantize_takes_every_border_between_codes_and_scales(dev, ty):
    """The neighbours of every border in fp32, for every mantissa of the block's scale."""
    rows = []
    for top in np.concatenate([np.arange(64, 128), np.arange(64, 128) + 0.5]):       # largest of the block: 4 <= a < 8 in units
        top = np.float32(top / 16.0)
        unit = 1.0 if ty == F.MXFP4 else F.scale_values(ty, F.quantise(ty, np.full((1, 16), float(top)))[1])[0, 0]
        t = np.float32(unit) * np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
        b = np.concatenate([t, np.nextafter(t, np.float32(99)), np.nextafter(t, np.float32(0)), -t, np.zeros(4, np.float32)])
        for h in (b[:15], b[15:30]):     # a half of 16 with the largest in it, twice for the blocks of 32
            rows.append(np.concatenate([[top], h, [top], -h]))
    # ... and the borders between scales: six times those of e4m3, powers of two
    s = (F.E4M3[1:] + F.E4M3[:-1]) / 2 * 6.0 if ty == F.NVFP4 else 2.0 ** np.arange(-126, 128)
    for v in np.float32(s):
        for w in (v, np.nextafter(v, np.float32(0)), np.nextafter(v, np.float32(np.inf))):
            rows.append(np.where(np.arange(32) % 16 == 3, w, w * np.float32(0.31)))
    x = np.array(rows, np.float32)
    x = x[np.abs(x).max(axis=1) < np.inf]
    d, _ = _buffer(dev, ty, F.ROWS, len(x), 32)
    d_x = dev.upload(x)
    assert dev.lib.q4_cuda_fp4_quantize(ty, F.ROWS, d_x, 32, 1.0, len(x), 32, d)
    want = F.values(ty, *F.quantise(ty, x.astype(np.float64))).astype(np.float32)
    np.testing.assert_array_equal(_values(dev, ty, F.ROWS, d, len(x), 32), want)
    dev.free(d), dev.free(d_x)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n,rows,cols", [(1, 1, 32), (3, 129, 96), (5, 64, 512), (2, 300, 736)])
def test_put_and_values(dev, ty, n, rows, cols):
    rng = np.random.default_rng(n + rows)
    codes = rng.integers(0, 16, (n, rows, cols), dtype=np.uint8)
    sb = rng.integers(0, 256 if ty == F.MXFP4 else 128, (n, rows, cols // F.BLOCK[ty]), dtype=np.uint8)
    want = F.values(ty, codes, sb)
    d, size = _buffer(dev, ty, F.WEIGHTS, rows, cols, n)
    sources = [(dev.upload(F.packed(codes)), dev.upload(sb))]
    if ty == F.MXFP4:
        sources.append((dev.upload(F.ggml_blocks(codes, sb)), None))
    for d_c, d_s in sources:
        assert dev.lib.q4_hip_fill(d, float("nan"), n * size // 4)
        assert dev.lib.q4_cuda_fp4_put(ty, d_c, d_s, rows, cols, n, d, size)
        for i in range(n):
            with np.errstate(over="ignore"):
                np.testing.assert_array_equal(_values(dev, ty, F.WEIGHTS, d + i * size, rows, cols), want[i].astype(np.float32))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,n_ff,extra,mul", [(1, 32, 0, 1.0), (37, 96, 5, 224.0), (9, 512, 0, 1.0), (600, 1024, 0, 0.11)])
def test_swiglu_quantize_is_that_of_the_exact_values(dev, ty, rows, n_ff, extra, mul):
    rng = np.random.default_rng(rows + n_ff)
    gu = (rng.standard_normal((rows, 2 * n_ff)) * rng.uniform(0.3, 6.0, (rows, 1))).astype(np.float32)
    g, u = gu[:, :n_ff], gu[:, n_ff:]
    mul = float(np.float32(mul))
    hard = [(-88.0, 1.0), (-95.0, 1e20), (-104.0, 1e30), (np.nan, 1.0), (np.inf, 1.0), (1.0, -np.inf), (0.0, 5.0), (3e38, 0.9), (3e38, 7.0),
            (-120.0, 3.0), (1e-30, 1e-9), (1e-30, 1e-20), (-0.0, 2.0), (70.0, 6.0), (-np.inf, 1.0), (F.FMAX, 1.0), (F.FMAX, 0.999), (-60.0, F.FMAX)]
    for i, (a, b) in enumerate(hard):
        r, c = (i * 5) % rows, (i * 64) % n_ff
        if rows * n_ff > 32 * len(hard):
            if i % 2:
                g[r, c:c + 32], u[r, c:c + 32] = a, b      # a block of it
            else:
                g[r, c + 3], u[r, c + 3] = a, b            # one of a block
    ld = 2 * n_ff + extra
    src = np.full((rows, ld), 1e9, np.float32)
    src[:, :2 * n_ff] = gu
    d, _ = _buffer(dev, ty, F.ROWS, rows, n_ff)
    d_gu = dev.upload(src)
    assert dev.lib.q4_cuda_fp4_swiglu_quantize(ty, d_gu, ld, mul, rows, n_ff, d)
    with np.errstate(over="ignore"):
        want = F.values(ty, *F.quantise(ty, F.swiglu(gu, mul), exact=True)).astype(np.float32)
    np.testing.assert_array_equal(_values(dev, ty, F.ROWS, d, rows, n_ff), want)
    dev.free(d), dev.free(d_gu)


def _check(got, x, w, scale, ty):
    want = (x @ w.T) * scale
    bound = F.product_bound(x, w, scale, x.shape[-1] // F.BLOCK[ty])
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want)[bad][:5], bound[bad][:5])


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,w_rows,cols,extra", [
    (1, 1, 32, 0), (1, 128, 256, 0), (2, 31, 96, 3), (1, 4099, 2048, 0), (3, 129, 544, 0), (5, 200, 1024, 8), (8, 512, 2048, 0), (9, 130, 288, 1),
    (16, 1000, 64, 0), (17, 192, 256, 0), (33, 193, 320, 7), (64, 384, 2048, 0), (100, 65, 512, 0), (128, 448, 736, 0), (129, 1024, 1024, 0),
    (300, 513, 2560, 0), (777, 640, 352, 16), (1500, 257, 4096, 0), (1, 33, 65536, 0), (140, 130, 65536, 0),
    # more of the tensor cores' (calls of little work are the CUDA cores'): a column tile's and a row tile's end, few columns
    (1300, 513, 32, 0), (700, 129, 352, 1), (40, 1000, 544, 0), (9, 4099, 544, 0), (33, 2311, 320, 9), (127, 640, 96, 0), (600, 65, 512, 7),
    # enough tiles for pairs of CTAs: a last pair with and without rows for its second one, whole and ragged columns
    (4111, 6801, 96, 0), (4352, 7104, 320, 8), (4190, 7000, 32, 4)])
def test_mul(dev, ty, rows, w_rows, cols, extra):
    rng = np.random.default_rng(rows * 7 + cols)
    w, d_w, _ = _weights(dev, rng, ty, 1, w_rows, cols)
    x, d_x = _rows(dev, rng, ty, rows, cols, 1.0 if ty == F.MXFP4 else 30.0)
    ld = w_rows + extra
    d_y = dev.upload(np.full((rows + 1, ld), SENTINEL, np.float32))
    assert dev.lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_x, rows, 0.37, d_y, ld)
    y = dev.download(d_y, (rows + 1, ld), np.float32)
    assert (y[rows:] == SENTINEL).all() and (y[:, w_rows:] == SENTINEL).all()
    _check(y[:rows, :w_rows], x, w[0], float(np.float32(0.37)), ty)
    for d in (d_w, d_x, d_y):
        dev.free(d)
    assert dev.lib.q4_cuda_device_error() == 0


@pytest.mark.parametrize("rows", [1, 40, 200, 400])
def test_mul_scales_far_apart(dev, rows):
    """Powers of two whose product is an ordinary number although neither is, and NaN blocks: a row of the weights or of
    the activations, and nothing beside it."""
    lib, cols, w_rows, ty = dev.lib, 256, 192, F.MXFP4
    rng = np.random.default_rng(rows)
    for far in (0, 60, 100):
        codes = rng.integers(0, 16, (w_rows, cols), dtype=np.uint8)
        sb = np.full((w_rows, cols // 32), 127 + far, np.uint8)
        sb[5, 3] = 255
        d_w, _ = _buffer(dev, ty, F.WEIGHTS, w_rows, cols)
        assert lib.q4_cuda_fp4_put(ty, dev.upload(F.packed(codes)), dev.upload(sb), w_rows, cols, 1, d_w, 0)
        x = (rng.standard_normal((rows, cols)) * 2.0 ** -far).astype(np.float32)
        x[rows // 2, 77] = np.nan if rows > 1 else x[0, 77]
        d_x, _ = _buffer(dev, ty, F.ROWS, rows, cols)
        assert lib.q4_cuda_fp4_quantize(ty, F.ROWS, dev.upload(x), cols, 1.0, rows, cols, d_x)
        d_y = dev.malloc(rows * w_rows * 4)
        assert lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_x, rows, 1.0, d_y, w_rows)
        y = dev.download(d_y, (rows, w_rows), np.float32)
        xv, wv = F.values(ty, *F.quantise(ty, x.astype(np.float64))), F.values(ty, codes, sb)
        want = xv @ wv.T
        assert (np.isnan(y) == np.isnan(want)).all()
        ok = ~np.isnan(want)
        bound = F.product_bound(np.nan_to_num(xv), np.nan_to_num(wv), 1.0, cols // 32)
        assert (np.abs(y - want)[ok] <= bound[ok]).all()


CASES = [  # experts, w_rows, cols, rows of each expert
    (4, 128, 256, [1, 0, 2, 1]), (3, 200, 96, [0, 0, 5]), (6, 64, 512, [0, 3, 0, 0, 9, 0]), (2, 513, 544, [33, 130]), (5, 384, 1024, [128, 1, 129, 0, 64]),
    (9, 256, 288, [7, 300, 0, 2, 41, 1, 1, 16, 90]), (1, 192, 2048, [500]), (70, 192, 256, [i % 5 for i in range(70)]), (1024, 32, 32, [1] * 1024),
    # more of the tensor cores': few rows of large matrices, more tiles of rows than their table has
    (6, 2100, 1024, [0, 3, 0, 0, 9, 0]), (70, 640, 512, [i % 5 for i in range(70)]), (1024, 200, 64, [1 + i % 3 for i in range(1024)]),
    (3, 1500, 96, [0, 260, 131])]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_mul_id(dev, ty, gather, case):
    n, w_rows, cols, count = CASES[case]
    rng = np.random.default_rng(case)
    w, d_w, stride = _weights(dev, rng, ty, n, w_rows, cols)
    bounds = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    total = int(bounds[-1])
    x_rows = total if not gather else max(1, total // 3)
    x, d_x = _rows(dev, rng, ty, x_rows, cols, 1.0 if ty == F.MXFP4 else 30.0)
    pick = np.arange(total)
    if gather:
        pick = rng.integers(0, x_rows, total)
        pick[rng.random(total) < 0.05] = -1                 # a row that is not there
        pick[rng.random(total) < 0.02] = x_rows
    xv = np.where(((pick < 0) | (pick >= x_rows))[:, None], 0.0, x[np.clip(pick, 0, x_rows - 1)])
    each = rng.uniform(0.5, 2.0, n).astype(np.float32)
    d_rows, d_b, d_e = dev.upload(pick.astype(np.int32)), dev.upload(bounds), dev.upload(each)
    ld = w_rows + (5 if case % 2 else 0)
    for use_each in (False, True):
        d_y = dev.upload(np.full((total + 2, ld), SENTINEL, np.float32))
        assert dev.lib.q4_cuda_fp4_mul_id(ty, d_w, w_rows, cols, stride, n, d_x, x_rows, d_rows if gather else None, d_b, total, 0.5,
                                          d_e if use_each else None, d_y, ld)
        y = dev.download(d_y, (total + 2, ld), np.float32)
        assert (y[total:] == SENTINEL).all() and (y[:, w_rows:] == SENTINEL).all()
        for e in range(n):
            lo, hi = bounds[e], bounds[e + 1]
            if lo < hi:
                _check(y[lo:hi, :w_rows], xv[lo:hi], w[e], 0.5 * (float(each[e]) if use_each else 1.0), ty)
        dev.free(d_y)
    for d in (d_w, d_x, d_rows, d_b, d_e):
        dev.free(d)
    assert dev.lib.q4_cuda_device_error() == 0


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("first,last,total", [(3, 20, 30), (0, 30, 17), (5, 5, 12), (130, 270, 400)])
@pytest.mark.parametrize("w_rows,cols", [(160, 128), (4000, 512)])
def test_mul_id_leaves_rows_of_nobody_alone(dev, ty, first, last, total, w_rows, cols):
    """Bounds that begin behind row 0 or end before the last row, and rows behind total_rows."""
    rng = np.random.default_rng(first + total)
    n = 3
    w, d_w, stride = _weights(dev, rng, ty, n, w_rows, cols)
    rows = max(total, last)
    x, d_x = _rows(dev, rng, ty, rows, cols)
    bounds = np.array([first, first + (last - first) // 3, first + (last - first) // 3, last], np.int32)
    d_y = dev.upload(np.full((rows, w_rows), SENTINEL, np.float32))
    assert dev.lib.q4_cuda_fp4_mul_id(ty, d_w, w_rows, cols, stride, n, d_x, rows, None, dev.upload(bounds), total, 1.0, None, d_y, w_rows)
    y = dev.download(d_y, (rows, w_rows), np.float32)
    for r in range(rows):
        e = [i for i in range(n) if bounds[i] <= r < bounds[i + 1]]
        if e and r < total:
            _check(y[r:r + 1], x[r:r + 1], w[e[0]], 1.0, ty)
        else:
            assert (y[r] == SENTINEL).all(), r
    assert dev.lib.q4_cuda_device_error() == 0


@pytest.mark.parametrize("ty", TYPES)
def test_refusals(dev, ty):
    """Checks of arguments: false, and nothing is enqueued."""
    lib = dev.lib
    d = dev.malloc(1 << 20)
    d_b = dev.upload(np.array([0, 4], np.int32))
    size = lib.q4_cuda_fp4_bytes(ty, F.WEIGHTS, 64, 64)
    n0 = lib.q4_cuda_launch_count()
    for form, rows, cols in ((2, 4, 64), (0, 0, 64), (0, 4, 0), (0, 4, 48), (1, 4, 65568), (1, 1 << 31, 64)):
        assert lib.q4_cuda_fp4_bytes(ty, form, rows, cols) == 0
    assert lib.q4_cuda_fp4_bytes(21, 0, 4, 64) == 0
    no = [
        lib.q4_cuda_fp4_quantize(21, 0, d, 64, 1.0, 4, 64, d), lib.q4_cuda_fp4_quantize(ty, 2, d, 64, 1.0, 4, 64, d),
        lib.q4_cuda_fp4_quantize(ty, 0, d, 63, 1.0, 4, 64, d), lib.q4_cuda_fp4_quantize(ty, 0, None, 64, 1.0, 4, 64, d),
        lib.q4_cuda_fp4_quantize(ty, 0, d, 64, 1.0, 4, 64, d + 8), lib.q4_cuda_fp4_quantize(ty, 0, d + 2, 64, 1.0, 4, 64, d),
        lib.q4_cuda_fp4_quantize(ty, 0, d, 64, 1.0, 0, 64, d), lib.q4_cuda_fp4_quantize(ty, 0, d, 64, 1.0, 4, 40, d),
        lib.q4_cuda_fp4_swiglu_quantize(ty, d, 127, 1.0, 4, 64, d), lib.q4_cuda_fp4_swiglu_quantize(ty, d, 128, 1.0, 4, 64, None),
        lib.q4_cuda_fp4_values(ty, 0, d, 4, 64, d, 63), lib.q4_cuda_fp4_values(ty, 0, d + 4, 4, 64, d, 64),
        lib.q4_cuda_fp4_put(ty, d, d, 4, 64, 0, d, size), lib.q4_cuda_fp4_put(ty, d, d, 64, 64, 2, d, size - 16),
        lib.q4_cuda_fp4_put(ty, None, d, 4, 64, 1, d, 0), lib.q4_cuda_fp4_put(ty, d, d, 64, 64, 2, d, size + 8),
        lib.q4_cuda_fp4_mul(ty, d, 64, 64, d, 4, 1.0, d, 63), lib.q4_cuda_fp4_mul(ty, d, 64, 64, d, 0, 1.0, d, 64),
        lib.q4_cuda_fp4_mul(ty, d + 8, 64, 64, d, 4, 1.0, d, 64), lib.q4_cuda_fp4_mul(ty, d, 64, 64, None, 4, 1.0, d, 64),
        lib.q4_cuda_fp4_mul(20, d, 64, 64, d, 4, 1.0, d, 64), lib.q4_cuda_fp4_mul(ty, d, 64, 50, d, 4, 1.0, d, 64),
        lib.q4_cuda_fp4_mul_id(ty, d, 64, 64, size, 0, d, 4, None, d_b, 4, 1.0, None, d, 64),
        lib.q4_cuda_fp4_mul_id(ty, d, 64, 64, size, 1025, d, 4, None, d_b, 4, 1.0, None, d, 64),
        lib.q4_cuda_fp4_mul_id(ty, d, 64, 64, size - 256, 2, d, 4, None, d_b, 4, 1.0, None, d, 64),
        lib.q4_cuda_fp4_mul_id(ty, d, 64, 64, size, 1, d, 4, None, None, 4, 1.0, None, d, 64),
        lib.q4_cuda_fp4_mul_id(ty, d, 64, 64, size, 1, d, 4, None, d_b, 5, 1.0, None, d, 64),       # more rows than x has
        lib.q4_cuda_fp4_mul_id(ty, d, 64, 64, size, 1, d, 4, None, d_b, 4, 1.0, None, d, 63),
    ]
    if ty == F.NVFP4:
        no.append(lib.q4_cuda_fp4_put(ty, d, None, 4, 64, 1, d, 0))
    assert not any(no), no
    assert lib.q4_cuda_launch_count() == n0
    assert lib.q4_cuda_fp4_mul_id(ty, d, 64, 64, size, 1, d, 4, None, d_b, 0, 1.0, None, d, 64)       # no rows: nothing to do
    assert lib.q4_cuda_launch_count() == n0


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows", [1, 20, 150])
def test_captured_and_replayed_with_other_data(dev, ty, rows):
    """quantize + mul in a graph, replayed on new inputs, between eager calls of another size."""
    lib = dev.lib
    rng = np.random.default_rng(rows)
    cols, w_rows = 512, 300
    w, d_w, _ = _weights(dev, rng, ty, 1, w_rows, cols)
    other, d_o = _rows(dev, rng, ty, 77, cols)
    d_x, d_y, d_y2 = dev.malloc(rows * cols * 4), dev.malloc(rows * w_rows * 4), dev.malloc(77 * w_rows * 4)
    d_q, _ = _buffer(dev, ty, F.ROWS, rows, cols)
    dev.sync()
    assert lib.q4_hip_graph_begin() == 1
    ok = lib.q4_cuda_fp4_quantize(ty, F.ROWS, d_x, cols, 1.0, rows, cols, d_q) and lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_q, rows, 1.0, d_y, w_rows)
    g = lib.q4_hip_graph_end()
    assert ok and g
    for _ in range(3):
        x = rng.standard_normal((rows, cols)).astype(np.float32)
        dev.write(d_x, x)
        assert lib.q4_hip_graph_launch(g)
        assert lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_o, 77, 1.0, d_y2, w_rows)
        xv = F.values(ty, *F.quantise(ty, x.astype(np.float64)))
        _check(dev.download(d_y, (rows, w_rows), np.float32), xv, w[0], 1.0, ty)
        _check(dev.download(d_y2, (77, w_rows), np.float32), other, w[0], 1.0, ty)
    lib.q4_hip_graph_free(g)
    assert lib.q4_cuda_device_error() == 0


def test_nothing_is_written_behind_a_buffer(dev):
    """A buffer is q4_cuda_fp4_bytes bytes."""
    lib = dev.lib
    for ty in TYPES:
        for form in (F.ROWS, F.WEIGHTS):
            for rows, cols in ((1, 32), (5, 96), (129, 288)):
                size = lib.q4_cuda_fp4_bytes(ty, form, rows, cols)
                d = dev.upload(np.full(size + 512, 0xAB, np.uint8))
                x = np.ones((rows, cols), np.float32)
                assert lib.q4_cuda_fp4_quantize(ty, form, dev.upload(x), cols, 1.0, rows, cols, d)
                assert (dev.download(d, (size + 512,), np.uint8)[size:] == 0xAB).all()


@pytest.mark.parametrize("ty", TYPES)
def test_offsets_beyond_32_bits(dev, ty):
    """Rows whose place in the result, or in the values read back, is behind 2^31 elements; of each the last rows are looked at."""
    lib, cols, w_rows, rows = dev.lib, 64, 32768, 70000
    rng = np.random.default_rng(11)
    w, d_w, _ = _weights(dev, rng, ty, 1, w_rows, cols)
    x, d_x = _rows(dev, rng, ty, rows, cols)
    d_y = dev.malloc(4 * rows * w_rows)
    for gather in (False, True):
        assert lib.q4_hip_fill(d_y, 0.0, rows * w_rows)
        pick = np.arange(rows)[::-1] if gather else np.arange(rows)
        d_rows, d_b = dev.upload(pick.astype(np.int32)), dev.upload(np.array([0, rows], np.int32))
        if gather:
            ok = lib.q4_cuda_fp4_mul_id(ty, d_w, w_rows, cols, 0, 1, d_x, rows, d_rows, d_b, rows, 1.0, None, d_y, w_rows)
        else:
            ok = lib.q4_cuda_fp4_mul(ty, d_w, w_rows, cols, d_x, rows, 1.0, d_y, w_rows)
        assert ok
        for r in (0, 65535, 65536, 69990):
            got = dev.download(d_y + 4 * r * w_rows, (10, w_rows), np.float32)
            _check(got, x[pick[r:r + 10]], w[0], 1.0, ty)
        dev.free(d_rows), dev.free(d_b)
    # the result as a matrix of fp32 rows: quantised and read back
    n = 2048
    big = rows * w_rows // n
    d_q, _ = _buffer(dev, ty, F.ROWS, big, n)
    assert lib.q4_cuda_fp4_quantize(ty, F.ROWS, d_y, n, 1.0, big, n, d_q)
    tail = dev.download(d_y + 4 * (big - 7) * n, (7, n), np.float32)
    assert lib.q4_cuda_fp4_values(ty, F.ROWS, d_q, big, n, d_y, n)
    got = dev.download(d_y + 4 * (big - 7) * n, (7, n), np.float32)
    np.testing.assert_array_equal(got, F.values(ty, *F.quantise(ty, tail.astype(np.float64))).astype(np.float32))
    for d in (d_w, d_x, d_y, d_q):
        dev.free(d)
    assert lib.q4_cuda_device_error() == 0
