"""The 4-bit calls as an engine issues them for one MoE layer of a batch: routing, balance, row assignment, quantised tokens,
gate and up, SwiGLU, down, combine."""
import numpy as np
import pytest

import fp4_plain as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty", [F.MXFP4, F.NVFP4])
@pytest.mark.parametrize("n_tok,n_exp,topk,embd,ff", [(1, 8, 2, 64, 32), (5, 32, 4, 256, 96), (90, 24, 3, 512, 256), (700, 16, 6, 256, 128)])
def test_layer(dev, ty, n_tok, n_exp, topk, embd, ff):
    lib = dev.lib
    rng = np.random.default_rng(n_tok)
    k1, n_mat = topk + 1, n_exp + 1
    x = rng.standard_normal((n_tok, embd)).astype(np.float32)
    logits = rng.standard_normal((n_tok, n_exp)).astype(np.float32)
    mul = 1.0 if ty == F.MXFP4 else 64.0

    def matrix(rows, cols):
        w = (rng.standard_normal((n_mat, rows, cols)) * cols ** -0.5).astype(np.float32)
        size = lib.q4_cuda_fp4_bytes(ty, F.WEIGHTS, rows, cols)
        d = dev.malloc(n_mat * size)
        d_w = dev.upload(w)
        for e in range(n_mat):       # an fp32 checkpoint: the factor brings NVFP4's scales into e4m3's range
            assert lib.q4_cuda_fp4_quantize(ty, F.WEIGHTS, d_w + 4 * e * rows * cols, cols, mul, rows, cols, d + e * size)
        return F.values(ty, *F.quantise(ty, (w * np.float32(mul)).astype(np.float64))), d, size

    w_gu, d_gu_w, s_gu = matrix(2 * ff, embd)
    w_dn, d_dn_w, s_dn = matrix(embd, ff)
    rows = n_tok * k1
    d_x, d_log = dev.upload(x), dev.upload(logits)
    d_ids, d_wts = dev.malloc(4 * n_tok * topk), dev.malloc(4 * n_tok * topk)
    d_atok, d_rsrc, d_rw = dev.malloc(4 * rows), dev.malloc(4 * rows), dev.malloc(4 * rows)
    d_b, d_cnt, d_loss = dev.malloc(4 * (n_mat + 1)), dev.malloc(4 * n_exp), dev.malloc(4)
    d_q, d_hq = dev.malloc(lib.q4_cuda_fp4_bytes(ty, F.ROWS, n_tok, embd)), dev.malloc(lib.q4_cuda_fp4_bytes(ty, F.ROWS, rows, ff))
    d_gu, d_pd, d_y = dev.malloc(4 * rows * 2 * ff), dev.malloc(4 * rows * embd), dev.malloc(4 * n_tok * embd)

    def layer():
        return (lib.q4_hip_route_pf(d_log, d_ids, d_wts, n_tok, n_exp, topk)
                and lib.q4_cuda_route_balance(d_log, d_ids, None, n_tok, n_exp, topk, 1.0, None, d_cnt, None, d_loss, None)
                and lib.q4_cuda_assign_local(d_ids, d_wts, d_atok, d_rsrc, d_rw, d_b, n_tok, topk, 0, n_exp, 1, 0, n_tok)
                and lib.q4_cuda_fp4_quantize(ty, F.ROWS, d_x, embd, mul, n_tok, embd, d_q)
                and lib.q4_cuda_fp4_mul_id(ty, d_gu_w, 2 * ff, embd, s_gu, n_mat, d_q, n_tok, d_atok, d_b, rows, 1.0 / mul ** 2, None, d_gu, 2 * ff)
                and lib.q4_cuda_fp4_swiglu_quantize(ty, d_gu, 2 * ff, mul, rows, ff, d_hq)
                and lib.q4_cuda_fp4_mul_id(ty, d_dn_w, embd, ff, s_dn, n_mat, d_hq, rows, None, d_b, rows, 1.0 / mul ** 2, None, d_pd, embd)
                and lib.q4_cuda_expert_reduce_set(d_y, d_pd, d_rsrc, d_rw, n_tok, k1, embd))

    def check():
        ids, wts = dev.download(d_ids, (n_tok, topk), np.int32), dev.download(d_wts, (n_tok, topk), np.float32)
        bounds = dev.download(d_b, (n_mat + 1,), np.int32)
        assert (np.diff(bounds)[:n_exp] == dev.download(d_cnt, (n_exp,), np.int32)).all()
        xq = F.values(ty, *F.quantise(ty, (dev.download(d_x, (n_tok, embd), np.float32) * np.float32(mul)).astype(np.float64)))
        atok = dev.download(d_atok, (rows,), np.int32)
        gu, pd = dev.download(d_gu, (rows, 2 * ff), np.float32), dev.download(d_pd, (rows, embd), np.float32)
        hq = F.values(ty, *F.quantise(ty, F.swiglu(gu, mul), exact=True))       # of the gate and up values that the device has
        scale = 1.0 / mul ** 2
        for e in range(n_mat):
            lo, hi = bounds[e], bounds[e + 1]
            a, h = xq[atok[lo:hi]], hq[lo:hi]
            assert (np.abs(gu[lo:hi] - a @ w_gu[e].T * scale) <= F.product_bound(a, w_gu[e], scale, embd // F.BLOCK[ty])).all()
            assert (np.abs(pd[lo:hi] - h @ w_dn[e].T * scale) <= F.product_bound(h, w_dn[e], scale, ff // F.BLOCK[ty])).all()
        # the layer as a whole, from the picks and the weights.  The device's gate and up values are fp32 sums, up to 1e-6 off, and a
        # value of h so near to a border falls on its other side: some four in a million, of half a million values at most, and
        # each moves one of n_ff values of a row by a third at most.  Three of them in one row of 128: 3 / 3 / sqrt(128) of its norm,
        # an eighth of the picks' share of one token of 700; of one token alone none is expected, and one would be 1 / 3 / sqrt(32).
        y = dev.download(d_y, (n_tok, embd), np.float32)
        want = np.zeros((n_tok, embd))
        for t in range(n_tok):
            for e, w in list(zip(ids[t], wts[t])) + [(n_exp, 1.0)]:
                h = F.values(ty, *F.quantise(ty, F.swiglu((xq[t] @ w_gu[e].T * scale)[None].astype(np.float32), mul), exact=True))[0]
                want[t] += float(w) * (h @ w_dn[e].T * scale)
        assert np.linalg.norm(y - want) <= 1e-2 * np.linalg.norm(want)
        return y

    assert layer()
    first = check()
    dev.sync()
    assert lib.q4_hip_graph_begin() == 1
    ok = layer()
    g = lib.q4_hip_graph_end()
    assert ok and g and lib.q4_hip_graph_launch(g)
    assert (check() == first).all()                              # the same bits
    dev.write(d_x, rng.standard_normal((n_tok, embd)).astype(np.float32))
    dev.write(d_log, rng.standard_normal((n_tok, n_exp)).astype(np.float32))
    assert lib.q4_hip_graph_launch(g)
    check()
    lib.q4_hip_graph_free(g)
    assert lib.q4_cuda_device_error() == 0
