"""q4_cuda_route_balance: counts, mean probabilities, balance loss and its gradient against the formulas in 64 bits and against
differences of the loss."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def plain(logits, ids, valid, coef, gout=1.0):
    t, e = logits.shape
    k = ids.shape[1]
    live = np.ones(t, bool) if valid is None else valid != 0
    n = int(live.sum())
    x = np.where(live[:, None], logits.astype(np.float64), -np.inf)
    with np.errstate(invalid="ignore", over="ignore"):
        m = x.max(axis=1, keepdims=True)
        z = np.where(np.isneginf(m) & ~np.isnan(x), 0.0, np.exp(x - np.where(np.isneginf(m), 0.0, m)))
    s = z.sum(axis=1, keepdims=True)
    p = np.where(s == 0, 0.0, z / np.where(s == 0, 1.0, s))
    p[~live] = 0.0
    picked = ids[live].ravel()
    counts = np.bincount(picked[(picked >= 0) & (picked < e)], minlength=e)[:e]
    f = counts / max(n * k, 1)
    prob = p.sum(axis=0) / max(n, 1)
    grad = gout * coef * e / max(n, 1) * p * (f - (p @ f)[:, None])
    grad[~live] = 0.0
    return counts, prob, coef * e * float(f @ prob), grad, p, f


def call(dev, logits, ids, valid, coef, gout=None, in_place=False, want=("counts", "prob", "loss", "dlogits")):
    t, e = logits.shape
    d_l, d_i = dev.upload(logits), dev.upload(ids)
    d_v = dev.upload(valid) if valid is not None else None
    d_g = dev.upload(np.array([gout], np.float32)) if gout is not None else None
    fill = np.float32(-777.0)
    d_c, d_p, d_s = dev.upload(np.full(e, -5, np.int32)), dev.upload(np.full(e, fill)), dev.upload(np.full(1, fill))
    d_d = d_l if in_place else dev.upload(np.full((t, e), fill))
    assert dev.lib.q4_cuda_route_balance(d_l, d_i, d_v, t, e, ids.shape[1], coef, d_g, d_c if "counts" in want else None,
                                         d_p if "prob" in want else None, d_s if "loss" in want else None, d_d if "dlogits" in want else None)
    out = (dev.download(d_c, (e,), np.int32), dev.download(d_p, (e,), np.float32), dev.download(d_s, (1,), np.float32)[0],
           dev.download(d_d, (t, e), np.float32))
    for d in (d_l, d_i, d_c, d_p, d_s) + ((d_v,) if d_v else ()) + ((d_g,) if d_g else ()) + (() if in_place else (d_d,)):
        dev.free(d)
    return out


def inputs(rng, t, e, k, padding=True):
    logits = (rng.standard_normal((t, e)) + rng.standard_normal(e)).astype(np.float32)
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :k].astype(np.int32)
    valid = (rng.random(t) < 0.8).astype(np.uint8) * 7 if padding else None
    return logits, ids, valid


def check(got, logits, ids, valid, coef, gout=1.0):
    """Bounds by counting half steps (2^-24) of fp32.  A probability: the exponent x - max and its product with log2 e are off by
    |x - max| and as much again for the constant's rounding, at most a third of it (below -104 the exponential is 0 or below
    1e-45 either way); the exponential by 4; the sum of e of them, 32 lanes' and then five steps, by e / 32 + 5; its inverse and the
    product with it by 2; 5 for what is left.  A mean adds a warp's rows (n / 8 at most), 24 warps, 8 CTAs, 18 clusters and divides."""
    counts, prob, loss, grad, p, f = plain(logits, ids, valid, coef, gout)
    t, e = logits.shape
    live = np.ones(t, bool) if valid is None else valid != 0
    x = logits[live].astype(np.float64)
    with np.errstate(invalid="ignore"):
        d = np.nanmax(x, axis=1, keepdims=True, initial=-np.inf) - x
    spread = d[np.isfinite(d) & (d < 104)].max(initial=0.0)
    per_p = (1.34 * spread + e / 32 + 16) * EPS
    mean = (t / 8 + 55) * EPS
    assert (got[0] == counts).all()
    ok = ~np.isnan(prob)
    assert (np.isnan(got[1]) == np.isnan(prob)).all()
    assert (np.abs(got[1] - prob)[ok] <= (per_p + mean) * prob[ok] + 1e-44).all()
    if np.isnan(loss):
        assert np.isnan(got[2])
    else:      # e products, added up over 32 to 512 threads
        assert abs(got[2] - loss) <= (per_p + mean + (e / 32 + 20) * EPS) * abs(loss) + 1e-44
    # the gradient: p's error on both terms, the sum over e, five products and the difference
    size = abs(gout * coef) * e / max(live.sum(), 1) * p * (f + (p @ f)[:, None])
    bound = (2 * per_p + (e / 32 + 16) * EPS) * size + 1e-44
    assert (np.isnan(got[3]) == np.isnan(grad)).all()
    assert (np.abs(got[3] - grad) <= bound)[~np.isnan(grad)].all()


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 512, 10), (2, 33, 1), (7, 8, 8), (64, 512, 10), (65, 128, 4), (100, 129, 6), (300, 1000, 3), (777, 64, 2),
                                   (2048, 512, 10), (5000, 16, 2), (9, 1024, 64), (20000, 96, 3)])
def test_values_and_gradient(dev, t, e, k):
    rng = np.random.default_rng(t + e)
    for padding in (False, True):
        logits, ids, valid = inputs(rng, t, e, k, padding)
        check(call(dev, logits, ids, valid, 0.01, 0.5 if padding else None), logits, ids, valid, float(np.float32(0.01)), 0.5 if padding else 1.0)
    first = call(dev, logits, ids, valid, 0.01, 0.5)
    again = call(dev, logits, ids, valid, 0.01, 0.5, in_place=True)
    for a, b in zip(first, again):
        assert np.asarray(a).tobytes() == np.asarray(b).tobytes()
    assert dev.lib.q4_cuda_device_error() == 0


def test_gradient_is_that_of_differences(dev):
    rng = np.random.default_rng(5)
    logits, ids, valid = inputs(rng, 6, 12, 2)
    valid[:] = [1, 1, 0, 1, 1, 1]
    grad = call(dev, logits, ids, valid, 2.0)[3]
    h = 1e-5
    for t in range(6):
        for j in range(12):
            x = logits.astype(np.float64)
            x[t, j] += h
            hi = plain(x, ids, valid, 2.0)[2]
            x[t, j] -= 2 * h
            assert abs((hi - plain(x, ids, valid, 2.0)[2]) / (2 * h) - grad[t, j]) < 1e-6


def test_rows_that_are_empty_masked_or_no_numbers(dev):
    rng = np.random.default_rng(6)
    logits, ids, valid = inputs(rng, 40, 70, 3)
    valid[:] = 1
    logits[3] = -np.inf                       # a row whose mask leaves nothing
    logits[4, :69] = -np.inf                  # ... or one expert
    logits[5, 1::2] = -np.inf
    logits[6] = np.finfo(np.float32).min      # all equal, the type's lowest value
    logits[7, ::3] = np.finfo(np.float32).min
    logits[8] = 1e30
    ids[9] = [-1, 70, 2]                      # no picks
    ids[10] = [5, 5, 5]                       # the same one again
    valid[11] = 0
    logits[11] = np.nan                       # padding holds anything
    ids[11] = 2 ** 30
    got = call(dev, logits, ids, valid, 0.3)
    check(got, logits, ids, valid, float(np.float32(0.3)))
    counts = got[0]
    assert (got[3][3] == 0).all() and (got[3][11] == 0).all()
    logits[20, 7] = np.nan                    # a NaN stays in its row, and in the sums
    got = call(dev, logits, ids, valid, 0.3)
    assert np.isnan(got[3][20]).all() and not np.isnan(np.delete(got[3], 20, 0)).any()
    assert np.isnan(got[1]).all() and np.isnan(got[2]) and (got[0] == counts).all()


def test_no_token_counts(dev):
    rng = np.random.default_rng(7)
    logits, ids, valid = inputs(rng, 9, 20, 2)
    valid[:] = 0
    c, p, l, g = call(dev, logits, ids, valid, 1.0)
    assert (c == 0).all() and (p == 0).all() and l == 0 and (g == 0).all()


def test_outputs_that_nobody_wants(dev):
    rng = np.random.default_rng(8)
    logits, ids, valid = inputs(rng, 50, 40, 4)
    full = call(dev, logits, ids, valid, 0.1)
    for i, name in enumerate(("counts", "prob", "loss", "dlogits")):
        got = call(dev, logits, ids, valid, 0.1, want=(name,))
        for j in range(4):
            if i == j:
                assert np.asarray(got[j]).tobytes() == np.asarray(full[j]).tobytes()
            else:
                assert (np.asarray(got[j]) == (-5 if j == 0 else np.float32(-777.0))).all()


def test_refusals(dev):
    lib, d = dev.lib, dev.malloc(1 << 16)
    n0 = lib.q4_cuda_launch_count()
    for a in ((None, d, None, 4, 8, 2), (d, None, None, 4, 8, 2), (d, d, None, 0, 8, 2), (d, d, None, 4, 0, 2), (d, d, None, 4, 1025, 2),
              (d, d, None, 4, 8, 0), (d, d, None, 4, 8, 65), (d + 2, d, None, 4, 8, 2), (d, d, None, 1 << 23, 8, 2)):
        assert not lib.q4_cuda_route_balance(*a, 1.0, None, d, d, d, d)
    assert lib.q4_cuda_launch_count() == n0


def test_captured_and_replayed(dev):
    lib = dev.lib
    rng = np.random.default_rng(9)
    t, e, k = 70, 130, 5
    d_l, d_i, d_v = dev.malloc(t * e * 4), dev.malloc(t * k * 4), dev.malloc(t)
    d_c, d_p, d_s, d_d = dev.malloc(e * 4), dev.malloc(e * 4), dev.malloc(4), dev.malloc(t * e * 4)
    dev.sync()
    assert lib.q4_hip_graph_begin() == 1
    ok = lib.q4_cuda_route_balance(d_l, d_i, d_v, t, e, k, 0.1, None, d_c, d_p, d_s, d_d)
    g = lib.q4_hip_graph_end()
    assert ok and g
    for _ in range(3):
        logits, ids, valid = inputs(rng, t, e, k)
        dev.write(d_l, logits), dev.write(d_i, ids), dev.write(d_v, valid)
        assert lib.q4_hip_graph_launch(g)
        call(dev, logits[:3], ids[:3], valid[:3], 0.1)          # an eager call that uses the same scratch
        got = (dev.download(d_c, (e,), np.int32), dev.download(d_p, (e,), np.float32), dev.download(d_s, (1,), np.float32)[0],
               dev.download(d_d, (t, e), np.float32))
        check(got, logits, ids, valid, float(np.float32(0.1)))
    lib.q4_hip_graph_free(g)
