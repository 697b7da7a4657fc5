"""The plain implementation of the 4-bit formats against their definitions' tables, and sizes and refusals that need no GPU."""
import numpy as np

import fp4_plain as F


def test_e4m3_and_e2m1_tables():
    assert F.E4M3[0] == 0 and F.E4M3[1] == 2.0 ** -9 and F.E4M3[8] == 2.0 ** -6 and F.E4M3[126] == 448.0
    v = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.3])
    assert F.e2m1(v).tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 9]


def test_quantised_values_are_nearest_of_all():
    rng = np.random.default_rng(3)
    for ty in (F.MXFP4, F.NVFP4):
        x = rng.standard_normal((50, 64)) * 3
        codes, sb = F.quantise(ty, x, exact=True)
        v = F.values(ty, codes, sb).reshape(-1)
        unit = np.repeat(F.scale_values(ty, sb), F.BLOCK[ty], axis=-1).reshape(-1)
        every = np.concatenate([-F.MAG[::-1], F.MAG])[None, :] * unit[:, None]
        best = np.abs(every - x.reshape(-1, 1)).min(axis=1)
        assert (np.abs(v - x.reshape(-1)) == best).all()
        # the codes again from the values: nothing more is lost
        if ty == F.MXFP4:
            assert (F.values(ty, *F.quantise(ty, v.reshape(50, 64))).reshape(-1) == v).all()


def test_blocks_that_hold_no_numbers():
    x = np.zeros((1, 32))
    for ty in (F.MXFP4, F.NVFP4):
        assert (F.values(ty, *F.quantise(ty, x)) == 0).all()
        for bad in (np.nan, np.inf, -np.inf):
            y = x + 1.0
            y[0, 3] = bad
            n = F.BLOCK[ty]
            v = F.values(ty, *F.quantise(ty, y))
            assert np.isnan(v[0, :n]).all() and not np.isnan(v[0, n:]).any()


def test_sizes(pkg):
    lib = pkg.capi.load()
    for ty, words in ((F.MXFP4, 2), (F.NVFP4, 4)):
        # codes on a 256-byte boundary, then words of scales for columns rounded up to 256; of four rows, or 128, at a time
        assert lib.q4_cuda_fp4_bytes(ty, F.ROWS, 1, 32) == 256 + 256
        assert lib.q4_cuda_fp4_bytes(ty, F.ROWS, 129, 2048) == 129 * 1024 + -(-132 * 8 * words * 4 // 256) * 256
        assert lib.q4_cuda_fp4_bytes(ty, F.WEIGHTS, 1, 32) == 256 + words * 512
        assert lib.q4_cuda_fp4_bytes(ty, F.WEIGHTS, 129, 288) == -(-129 * 144 // 256) * 256 + 2 * 2 * words * 512
        for form, rows, cols in ((2, 4, 64), (0, 0, 64), (0, 4, 0), (0, 4, 48), (1, 4, 65568), (1, 1 << 31, 64)):
            assert lib.q4_cuda_fp4_bytes(ty, form, rows, cols) == 0
    assert lib.q4_cuda_fp4_bytes(21, 0, 4, 64) == 0
