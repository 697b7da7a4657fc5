"""MXFP4 and NVFP4 written out plainly in numpy, in 64 bits: what the tests of the 4-bit floating point calls compare with."""
import numpy as np

MXFP4, NVFP4 = 39, 40
ROWS, WEIGHTS = 0, 1
NAMES = {MXFP4: "mxfp4", NVFP4: "nvfp4"}
BLOCK = {MXFP4: 32, NVFP4: 16}
MAG = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
FMAX = float(np.finfo(np.float32).max)


def e4m3_table():
    b = np.arange(127)
    e, m = b >> 3, b & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))


E4M3 = e4m3_table()


def scale_values(ty, b):
    b = np.asarray(b).astype(np.int64)
    if ty == MXFP4:
        return np.where(b == 255, np.nan, 2.0 ** (b - 127.0))
    v = E4M3[np.minimum(b & 127, 126)]
    return np.where((b & 127) == 127, np.nan, np.where(b >= 128, -v, v))


def e2m1(v):
    """Codes of the nearest values, ties to the even code."""
    a = np.minimum(np.abs(v), 6.0)
    up = np.clip(np.searchsorted(MAG, a), 1, 7)
    lo, hi = a - MAG[up - 1], MAG[up] - a
    code = np.where((lo < hi) | ((lo == hi) & (up % 2 == 1)), up - 1, up)
    return (code | np.where(np.signbit(v), 8, 0)).astype(np.uint8)


def quantise(ty, v, exact=False):
    """v (float64, what a row holds after its factor) -> codes [.., n], scale bytes [.., n / block].  A sixth of the largest is its
    fp32 product with fp32's 1/6, or, of values that are no fp32 numbers (exact), the quotient."""
    n = v.shape[-1]
    x = v.reshape(*v.shape[:-1], n // BLOCK[ty], BLOCK[ty])
    with np.errstate(invalid="ignore", over="ignore"):
        bad = ~(np.abs(x.astype(np.float32)) <= FMAX).all(axis=-1)
        x = np.where(bad[..., None], 0.0, x)
        top = np.abs(x).max(axis=-1)
        if ty == MXFP4:
            sb = np.clip(np.frexp(top)[1] - 3, -127, 127) + 127
            sb = np.where(top == 0, 0, sb)
            unit = 2.0 ** (sb - 127.0)
            nan = 255
        else:
            sixth = top / 6.0 if exact else (top.astype(np.float32) * np.float32(1.0 / 6.0)).astype(np.float64)
            want = np.minimum(sixth, 448.0)
            up = np.clip(np.searchsorted(E4M3, want), 1, 126)
            lo, hi = want - E4M3[up - 1], E4M3[up] - want
            sb = np.where((lo < hi) | ((lo == hi) & (up % 2 == 1)), up - 1, up)
            unit = E4M3[sb]
            nan = 127
        codes = e2m1(x / np.where(unit > 0, unit, 1.0)[..., None])
    codes = np.where((bad | (unit == 0))[..., None], 0, codes)
    return codes.reshape(v.shape).astype(np.uint8), np.where(bad, nan, sb).astype(np.uint8)


def values(ty, codes, sb):
    m = np.where(codes >= 8, -MAG[codes & 7], MAG[codes & 7])
    return m * np.repeat(scale_values(ty, sb), BLOCK[ty], axis=-1)


def packed(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def ggml_blocks(codes, sb):
    c = codes.reshape(*sb.shape, 32)
    return np.concatenate([sb[..., None], c[..., :16] | (c[..., 16:] << 4)], axis=-1).astype(np.uint8)


def swiglu(gu, mul):
    n = gu.shape[-1] // 2
    g, u = gu[..., :n].astype(np.float64), gu[..., n:].astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        return g / (1.0 + np.exp(-g)) * u * mul


def product_bound(x, w, scale, blocks):
    """|error| of a product whose code products are exact: every block's sum (at most 24 bits with its scales, exact) is added to
    a running fp32 sum, off by a step of it at most (2^-23 of the sum of magnitudes, also where a unit cuts instead of rounding),
    then come the factor and its product, half a step each."""
    return (blocks + 4) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) * abs(scale) + 1e-42
