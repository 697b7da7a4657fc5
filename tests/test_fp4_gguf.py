"""MXFP4 experts of a GGUF file: the host's reader sizes and slices them, and a layer runs from the file."""
import ctypes as C

import numpy as np
import pytest

import fp4_plain as F
import test_gguf as G

NAMES = ("ffn_gate", "ffn_up", "ffn_down")


def _model(path, rng, n_embd, n_ff, n_exp):
    """A file with one layer; the codes and scales of its matrices, the shared expert's last."""
    shapes = ((n_ff, n_embd), (n_ff, n_embd), (n_embd, n_ff))
    codes = [rng.integers(0, 16, (n_exp + 1, r, c), dtype=np.uint8) for r, c in shapes]
    sb = [rng.integers(121, 124, (n_exp + 1, r, c // 32), dtype=np.uint8) for r, c in shapes]
    tensors = [("token_embd.weight", G.F32, (8, 4), rng.bytes(128))]
    for i, name in enumerate(NAMES):
        r, c = shapes[i]
        blocks = F.ggml_blocks(codes[i], sb[i])
        tensors.append(("blk.0.%s_exps.weight" % name, F.MXFP4, (c, r, n_exp), blocks[:n_exp].tobytes()))
        tensors.append(("blk.0.%s_shexp.weight" % name, F.MXFP4, (c, r), blocks[n_exp].tobytes()))
    G.write_gguf(path, tensors, alignment=32)
    return codes, sb


def _parts(lib, g):
    v = [C.c_uint64() for _ in range(4)]
    n = C.c_uint32()
    t = [C.POINTER(G.Tensor)() for _ in range(3)]
    ok = lib.q4b_gguf_expert_parts(C.byref(g), 0, *(C.byref(x) for x in t), *(C.byref(x) for x in v), C.byref(n))
    return ok and ([x.value for x in v], n.value, [x.contents.type for x in t])


def test_reader_sizes_and_slices_mxfp4(tmp_path):
    lib = G._lib(False)
    n_embd, n_ff, n_exp = 96, 64, 3
    codes, sb = _model(str(tmp_path / "m.gguf"), np.random.default_rng(1), n_embd, n_ff, n_exp)
    assert lib.q4b_gguf_row_bytes(F.MXFP4, C.c_uint64(96)) == 51 and lib.q4b_gguf_row_bytes(F.MXFP4, C.c_uint64(80)) == 0
    assert lib.q4b_gguf_row_bytes(F.NVFP4, C.c_uint64(128)) == 0            # a type that it cannot size
    g = G.Gguf()
    assert lib.q4b_gguf_open(C.byref(g), str(tmp_path / "m.gguf").encode())
    part = n_ff * n_embd // 32 * 17
    assert _parts(lib, g) == ([0, part, 2 * part, 3 * part], n_exp, [F.MXFP4] * 3)
    host = np.zeros(3 * part, np.uint8)
    for e in range(n_exp + 1):
        got = (lib.q4b_gguf_read_pack(C.byref(g), 0, e, C.c_void_p(host.ctypes.data)) if e < n_exp else
               lib.q4b_gguf_read_shared_pack(C.byref(g), 0, C.c_void_p(host.ctypes.data), C.c_uint64(3 * part)))
        assert got == 3 * part
        assert np.array_equal(host, np.concatenate([F.ggml_blocks(codes[i][e], sb[i][e]).ravel() for i in range(3)]))
    lib.q4b_gguf_close(C.byref(g))


def test_arenas_do_not_take_mxfp4(tmp_path, pkg):
    """No layer call multiplies MXFP4 packs out of an arena: loading them into one is refused."""
    lib = G._lib(True)
    lib.q4b_moe_layer_load_gguf.restype = C.c_bool
    _model(str(tmp_path / "m.gguf"), np.random.default_rng(2), 256, 256, 2)
    g, layer = G.Gguf(), G.Layer()
    assert lib.q4b_gguf_open(C.byref(g), str(tmp_path / "m.gguf").encode())
    assert not lib.q4b_moe_layer_load_gguf(C.byref(layer), 3, C.byref(g), 0)
    lib.q4b_gguf_close(C.byref(g))
    text = open(G.os.path.join(G.PKG, "host", "q4_moe_b200.c")).read()
    body = text[text.index("bool q4b_moe_layer_load_gguf"):]
    assert body.index("Q4_T_MXFP4") < body.index("q4_hip_host_alloc_coh")       # before anything is allocated


@pytest.mark.gpu
def test_layer_from_a_file(tmp_path, dev):
    host_lib, lib, ty = G._lib(True), dev.lib, F.MXFP4
    rng = np.random.default_rng(3)
    n_embd, n_ff, n_exp, topk, n_tok = 256, 96, 6, 2, 21
    codes, sb = _model(str(tmp_path / "m.gguf"), rng, n_embd, n_ff, n_exp)
    g = G.Gguf()
    assert host_lib.q4b_gguf_open(C.byref(g), str(tmp_path / "m.gguf").encode())
    (_, _, od, total), n, _ = _parts(host_lib, g)
    assert n == n_exp
    sg, sd = lib.q4_cuda_fp4_bytes(ty, F.WEIGHTS, 2 * n_ff, n_embd), lib.q4_cuda_fp4_bytes(ty, F.WEIGHTS, n_embd, n_ff)
    w_gu, w_dn, pack = dev.malloc((n_exp + 1) * sg), dev.malloc((n_exp + 1) * sd), dev.malloc(total)
    host = np.zeros(total, np.uint8)
    at = C.c_void_p(host.ctypes.data)
    for e in range(n_exp + 1):
        assert (host_lib.q4b_gguf_read_pack(C.byref(g), 0, e, at) if e < n_exp else
                host_lib.q4b_gguf_read_shared_pack(C.byref(g), 0, at, C.c_uint64(total))) == total
        assert lib.q4_hip_h2d(pack, host.ctypes.data, total)
        assert lib.q4_cuda_fp4_put(ty, pack, None, 2 * n_ff, n_embd, 1, w_gu + e * sg, 0)
        assert lib.q4_cuda_fp4_put(ty, pack + od, None, n_embd, n_ff, 1, w_dn + e * sd, 0)
        assert lib.q4_hip_stream_sync()
    host_lib.q4b_gguf_close(C.byref(g))

    rows = n_tok * (topk + 1)
    x = rng.standard_normal((n_tok, n_embd)).astype(np.float32)
    d_x, d_log = dev.upload(x), dev.upload(rng.standard_normal((n_tok, n_exp)).astype(np.float32))
    ids, wts, counts = dev.malloc(4 * n_tok * topk), dev.malloc(4 * n_tok * topk), dev.malloc(4 * n_exp)
    atok, rsrc, rw, bounds = dev.malloc(4 * rows), dev.malloc(4 * rows), dev.malloc(4 * rows), dev.malloc(4 * (n_exp + 2))
    xq, hq = dev.malloc(lib.q4_cuda_fp4_bytes(ty, F.ROWS, n_tok, n_embd)), dev.malloc(lib.q4_cuda_fp4_bytes(ty, F.ROWS, rows, n_ff))
    gu, pd, y = dev.malloc(4 * rows * 2 * n_ff), dev.malloc(4 * rows * n_embd), dev.malloc(4 * n_tok * n_embd)
    assert lib.q4_hip_route_pf(d_log, ids, wts, n_tok, n_exp, topk)
    assert lib.q4_cuda_route_balance(d_log, ids, None, n_tok, n_exp, topk, 0.0, None, counts, None, None, None)
    assert lib.q4_cuda_assign_local(ids, wts, atok, rsrc, rw, bounds, n_tok, topk, 0, n_exp, 1, 0, n_tok)
    assert lib.q4_cuda_fp4_quantize(ty, F.ROWS, d_x, n_embd, 1.0, n_tok, n_embd, xq)
    assert lib.q4_cuda_fp4_mul_id(ty, w_gu, 2 * n_ff, n_embd, sg, n_exp + 1, xq, n_tok, atok, bounds, rows, 1.0, None, gu, 2 * n_ff)
    assert lib.q4_cuda_fp4_swiglu_quantize(ty, gu, 2 * n_ff, 1.0, rows, n_ff, hq)
    assert lib.q4_cuda_fp4_mul_id(ty, w_dn, n_embd, n_ff, sd, n_exp + 1, hq, rows, None, bounds, rows, 1.0, None, pd, n_embd)
    assert lib.q4_cuda_expert_reduce_set(y, pd, rsrc, rw, n_tok, topk + 1, n_embd)

    b = dev.download(bounds, (n_exp + 2,), np.int32)
    tok = dev.download(atok, (rows,), np.int32)
    picks, weight = dev.download(ids, (n_tok, topk), np.int32), dev.download(wts, (n_tok, topk), np.float32)
    gu_d, pd_d = dev.download(gu, (rows, 2 * n_ff), np.float32), dev.download(pd, (rows, n_embd), np.float32)
    w = [F.values(ty, codes[i], sb[i]) for i in range(3)]
    xv = F.values(ty, *F.quantise(ty, x.astype(np.float64)))
    hv = F.values(ty, *F.quantise(ty, F.swiglu(gu_d, 1.0), exact=True))
    want = np.zeros((n_tok, n_embd))
    for e in range(n_exp + 1):
        lo, hi = b[e], b[e + 1]
        a, both = xv[tok[lo:hi]], np.concatenate([w[0][e], w[1][e]])
        assert (np.abs(gu_d[lo:hi] - a @ both.T) <= F.product_bound(a, both, 1.0, n_embd // 32)).all()
        assert (np.abs(pd_d[lo:hi] - hv[lo:hi] @ w[2][e].T) <= F.product_bound(hv[lo:hi], w[2][e], 1.0, n_ff // 32)).all()
        for p in range(lo, hi):
            t = tok[p]
            want[t] += (1.0 if e == n_exp else float(weight[t][list(picks[t]).index(e)])) * pd_d[p]
    # three products and their sum, rounded to fp32 each: 4 half steps of the magnitudes, which the rows of pd bound
    size = np.zeros_like(want)
    for p in range(rows):
        size[tok[p]] += np.abs(pd_d[p])
    assert (np.abs(dev.download(y, (n_tok, n_embd), np.float32) - want) <= 6 * 2.0 ** -24 * size + 1e-42).all()
    assert (dev.download(counts, (n_exp,), np.int32) == np.diff(b)[:n_exp]).all()
    assert lib.q4_cuda_device_error() == 0
