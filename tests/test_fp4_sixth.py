"""How far NVFP4's scale, the e4m3 number nearest to the product of a block's largest with fp32's 1/6, is from the one nearest to its sixth."""
import numpy as np
import pytest

import fp4_plain as F

SIXTH = np.float32(1.0 / 6.0)
# fp32's 1/6 is 2^-25 of it too large (its error is a third of a step of 2^-26), and the product is rounded by half a step, 2^-24 at most
OFF = 2.0 ** -25 + 2.0 ** -24
BORDERS = (F.E4M3[1:] + F.E4M3[:-1]) / 2


def _nearest(want):
    """Indices of the e4m3 numbers nearest to want (float64), ties to the even one."""
    up = np.clip(np.searchsorted(F.E4M3, np.minimum(want, 448.0)), 1, 126)
    lo, hi = np.minimum(want, 448.0) - F.E4M3[up - 1], F.E4M3[up] - np.minimum(want, 448.0)
    return np.where((lo < hi) | ((lo == hi) & (up % 2 == 1)), up - 1, up)


@pytest.mark.parametrize("binade", [-9, -8, -5, 0, 2, 3, 10])
def test_product_and_sixth_over_all_mantissas(binade):
    """They name the same scale for all fp32 numbers of a binade but one, at which both of its neighbours are equally near to the sixth to
    within the rounding of the two operations."""
    x = (np.arange(2 ** 23, dtype=np.uint32) + np.uint32((binade + 127) << 23)).view(np.float32)
    product = (x * SIXTH).astype(np.float64)
    sixth = x.astype(np.float64) / 6.0
    differ = np.flatnonzero(_nearest(product) != _nearest(sixth))
    assert len(differ) <= 1
    for i in differ:
        b = BORDERS[np.argmin(np.abs(BORDERS - sixth[i]))]
        assert abs(sixth[i] - b) <= OFF * sixth[i] and x[i] == np.nextafter(np.float32(7.125 * 2.0 ** (binade - 2)), np.float32(0))


@pytest.mark.gpu
@pytest.mark.parametrize("form", [F.ROWS, F.WEIGHTS])
def test_scales_near_every_border(dev, form):
    """64 fp32 numbers on both sides of six times every border between two e4m3 numbers: the scale is the one nearest to the sixth, or, nearer
    to the border than the product's rounding, the other neighbour."""
    at = (BORDERS * 6.0).astype(np.float32).view(np.uint32)[:, None] + np.arange(-64, 65)
    top = at.astype(np.uint32).view(np.float32).ravel()
    rows = -(-len(top) // 16)
    x = np.zeros((rows, 256), np.float32)
    x.reshape(-1, 16)[:len(top), 3] = top
    lib, ty = dev.lib, F.NVFP4
    d_x, d_v = dev.upload(x), dev.malloc(rows * 256 * 4)
    d = dev.malloc(lib.q4_cuda_fp4_bytes(ty, form, rows, 256))
    assert lib.q4_cuda_fp4_quantize(ty, form, d_x, 256, 1.0, rows, 256, d)
    assert lib.q4_cuda_fp4_values(ty, form, d, rows, 256, d_v, 256)
    got = dev.download(d_v, (rows, 256), np.float32).reshape(-1, 16)[:len(top), 3].astype(np.float64)
    sixth = top.astype(np.float64) / 6.0
    best = _nearest(sixth)
    near = np.abs(sixth - np.repeat(BORDERS, 129)) <= OFF * sixth

    def value(scale):
        s = F.E4M3[scale]
        code = F.e2m1(top / np.where(s > 0, s, 1.0))
        return np.where(s > 0, F.MAG[code] * s, 0.0)

    other = np.where(F.E4M3[best] > sixth, best - 1, np.minimum(best + 1, 126))
    assert ((got == value(best)) | (near & (got == value(other)))).all()
    assert near.sum() < 400
    for p in (d_x, d_v, d):
        dev.free(p)
