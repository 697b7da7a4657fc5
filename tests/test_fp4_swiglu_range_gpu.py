"""q4_cuda_fp4_swiglu_quantize over the whole range of its factor: scales and codes are those of the exact values also where gate, up or a
product on the way leaves fp32's normal numbers."""
import numpy as np
import pytest

import fp4_plain as F

pytestmark = pytest.mark.gpu


def _check(dev, ty, gu, mul):
    lib = dev.lib
    rows, n_ff = gu.shape[0], gu.shape[1] // 2
    d_gu = dev.upload(gu)
    d = dev.malloc(lib.q4_cuda_fp4_bytes(ty, F.ROWS, rows, n_ff))
    d_v = dev.malloc(rows * n_ff * 4)
    assert lib.q4_cuda_fp4_swiglu_quantize(ty, d_gu, 2 * n_ff, mul, rows, n_ff, d)
    assert lib.q4_cuda_fp4_values(ty, F.ROWS, d, rows, n_ff, d_v, n_ff)
    got = dev.download(d_v, (rows, n_ff), np.float32)
    for p in (d_gu, d, d_v):
        dev.free(p)
    with np.errstate(over="ignore", invalid="ignore"):
        want = F.values(ty, *F.quantise(ty, F.swiglu(gu, float(np.float32(mul))), exact=True)).astype(np.float32)
    np.testing.assert_array_equal(got, want)
    return want


@pytest.mark.parametrize("ty", [F.MXFP4, F.NVFP4])
@pytest.mark.parametrize("mul", [0.0, 1e-38, 1e-20, 1.0, 224.0, 8.5e7, 1e10, 1e18, -1e20, 1e30, 3e38])
def test_gate_and_up_of_every_size(dev, ty, mul):
    """Gate and up in every pair of magnitudes that fp32 has, a pair to a block: about equal within it, and as one value beside ordinary ones."""
    rng = np.random.default_rng(17)
    mags = 10.0 ** np.arange(-45, 39, 4.0)
    pairs = [(sign * g, u) for g in mags for u in mags for sign in ((1.0, -1.0) if g < 1e3 else (1.0,))]
    n = len(pairs)
    g = np.array([p[0] for p in pairs])[:, None] * rng.uniform(0.5, 2.0, (n, 64))
    u = np.array([p[1] for p in pairs])[:, None] * rng.uniform(0.5, 2.0, (n, 64)) * rng.choice([-1.0, 1.0], (n, 64))
    alone = np.arange(64) % 16 == 5
    g[:, 32:] = np.where(alone[32:], g[:, 32:], 1.0)
    u[:, 32:] = np.where(alone[32:], u[:, 32:], rng.standard_normal((n, 32)))
    _check(dev, ty, np.concatenate([g, u], axis=1).astype(np.float32), mul)


@pytest.mark.parametrize("ty", [F.MXFP4, F.NVFP4])
def test_products_that_lose_bits_before_the_factor(dev, ty):
    rng = np.random.default_rng(18)
    for g, u, mul in ((1.0, 1e-42, 1e18), (1.0, 1e-43, 1e20), (1e-30, 1e-20, 1e38), (3 * 2.0 ** -149, 2.0 ** 127, 1.0), (4.2e-45, 1.7e38, 1.0),
                      (-79.0, 1e-9, 1e30), (-80.5, 1e-9, 1e30), (1e-20, -1e-19, 1e37)):
        gu = np.concatenate([np.full((32, 64), g), u * rng.uniform(0.3, 1.0, (32, 64))], axis=1).astype(np.float32)
        assert (_check(dev, ty, gu, mul) != 0).any() or ty == F.NVFP4


@pytest.mark.parametrize("ty", [F.MXFP4, F.NVFP4])
def test_factor_of_zero_infinity_and_nan(dev, ty):
    gu = np.full((4, 128), 1e30, np.float32)         # gate * up is beyond fp32
    gu[1] = 0.0
    gu[2] = 1.5
    assert (_check(dev, ty, gu, 0.0) == 0).all()
    gu[3, :64] = np.inf
    for mul in (0.0, np.inf, np.nan, -np.inf):
        want = _check(dev, ty, gu, mul)
        assert np.isnan(want[3]).all() and (mul == 0.0 or np.isnan(want[2]).all())
