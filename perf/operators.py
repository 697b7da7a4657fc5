"""Workloads for the 4-bit floating point operators and the balance loss of the router: their plain forms in elementary
torch operations, the calls that a program makes of libq4cuda.so, and the values from the definitions in 64 bits.

Two formats.  MXFP4: blocks of 32 values share a power of two (one byte, 127 + exponent); NVFP4: blocks of 16 share an
e4m3 number.  A value is a sign and a magnitude out of 0, 1/2, 1, 3/2, 2, 3, 4, 6, two to a byte (the even one low).

Kinds of cases:
  linear   rows of fp32 are quantised and multiplied with a quantised matrix (a dense projection)
  gate_up  tokens are quantised once; every expert multiplies the rows of the tokens that picked it (gathered)
  down     SwiGLU of gate and up rows, quantised in one step, and the experts' second product
  store    rows are quantised and read back as the values that they stand for
  balance  counts per expert, mean probabilities, balance loss and its gradient with respect to the router logits

Shapes are those of the benchmark and the tests: hidden 2048, expert width 512, 512 experts, top-10 plus one shared
expert that every token takes, and widths around them.
"""
import math

import torch

own = False

TILE = 128                                          # rows of an expert that the plain form multiplies at a time
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)   # between neighbours; a value on one goes to the even code
TYPE = {"mxfp4": 39, "nvfp4": 40}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
ROWS, WEIGHTS = 0, 1                                # the library's two orders of a quantised matrix


def listed():
    model = {"experts": 512, "topk": 10, "embd": 2048, "ff": 512}
    return [
        # a projection of one decoded token
        {"name": "linear 1 token", "kind": "linear", "type": "mxfp4", "tokens": 1, "rows": 4096, "embd": 2048},
        # a verify window of speculative decoding
        {"name": "linear 7 tokens", "kind": "linear", "type": "nvfp4", "tokens": 7, "rows": 4096, "embd": 2048},
        # a ragged last chunk of a prompt and an odd number of matrix rows (a vocabulary slice)
        {"name": "linear 777 tokens", "kind": "linear", "type": "mxfp4", "tokens": 777, "rows": 4099, "embd": 2560},
        # a long prompt
        {"name": "linear 8192 tokens", "kind": "linear", "type": "nvfp4", "tokens": 8192, "rows": 4096, "embd": 2048},
        # the experts' first product: one decoded token, the benchmark's batch, a long prompt with skewed popularity
        dict(model, name="gate/up 1 token", kind="gate_up", type="mxfp4", tokens=1, skew=0.0),
        dict(model, name="gate/up 64 tokens", kind="gate_up", type="nvfp4", tokens=64, skew=0.0),
        dict(model, name="gate/up 8192 skewed", kind="gate_up", type="mxfp4", tokens=8192, skew=0.7),
        # the second product: a small odd batch, the benchmark's prompt chunk
        dict(model, name="down 33 tokens", kind="down", type="mxfp4", tokens=33, skew=0.0),
        dict(model, name="down 2048 tokens", kind="down", type="nvfp4", tokens=2048, skew=0.7),
        # activations of a prompt kept in 4 bits and read back
        {"name": "store 4096 rows", "kind": "store", "type": "nvfp4", "tokens": 4096, "embd": 2048},
        # the load of the experts for a decode batch, and for a long padded prompt with the gradient
        {"name": "balance 64 tokens", "kind": "balance", "tokens": 64, "experts": 512, "topk": 10},
        {"name": "balance 8192 tokens", "kind": "balance", "tokens": 8192, "experts": 512, "topk": 10},
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "gate_up", "gate_up", "gate_up", "down", "down", "store", "balance"])
    case = {"kind": kind, "tokens": log_int(rng, 1, 8192)}
    if kind == "balance":
        case["topk"] = rng.randint(1, 10)
        case["experts"] = log_int(rng, case["topk"] + 1, 512)
        return case
    case["type"] = rng.choice(["mxfp4", "nvfp4"])
    case["embd"] = 32 * log_int(rng, 4, 80)
    if kind == "store":
        return case
    if kind == "linear":
        case["rows"] = log_int(rng, 64, 8192)
        case["tokens"] = min(case["tokens"], 8192 * 4096 * 2048 // (case["rows"] * case["embd"]))
        return case
    case["topk"] = rng.randint(1, 10)
    case["experts"] = log_int(rng, case["topk"] + 1, 512)
    case["ff"] = 32 * rng.randint(2, 20)
    case["tokens"] = max(1, min(case["tokens"], 8192 * 11 * 2048 * 512 // ((case["topk"] + 1) * case["embd"] * case["ff"])))
    if kind == "down":
        case["tokens"] = min(case["tokens"], 4096)
    case["skew"] = rng.choice([0.0, 0.7])
    return case


# ------------------------------------------------------------------ sizes

def matrix(case):
    """Rows and columns of one weight matrix."""
    if case["kind"] == "linear":
        return case["rows"], case["embd"]
    return (2 * case["ff"], case["embd"]) if case["kind"] == "gate_up" else (case["embd"], case["ff"])


def stored(ty, values):
    return values // 2 + values // BLOCK[ty]


def popularity(case):
    e = case["experts"]
    p = torch.arange(1, e + 1, dtype=torch.float64) ** -case["skew"]
    return p / p.sum()


def work(case):
    t, kind = case["tokens"], case["kind"]
    if kind == "balance":
        e, k = case["experts"], case["topk"]
        return {"bytes": t * (8 * e + 4 * k + 1) + 8 * e, "flops": 9.0 * t * e}
    if kind == "store":
        n = t * case["embd"]
        return {"bytes": 8 * n + stored(case["type"], n), "flops": 4.0 * n}
    m, k = matrix(case)
    if kind == "linear":
        return {"bytes": stored(case["type"], m * k) + 4 * t * (k + m), "flops": 2.0 * t * m * k}
    rows = t * (case["topk"] + 1)
    # expected number of matrices that are read: an expert is in a token's picks about topk * p times (at most once)
    used = 1.0 + float((1 - (1 - (case["topk"] * popularity(case)).clamp(max=1.0)) ** t).sum())
    read = 4 * t * k + 4 * rows if kind == "gate_up" else 8 * rows * k
    return {"bytes": used * stored(case["type"], m * k) + read + 4 * rows * m, "flops": 2.0 * rows * m * k}


# ------------------------------------------------------------------ what a program has in hand

_lib = None


def library():
    global _lib
    if _lib is None:
        import __graft_entry__ as entry
        _lib = entry.load_package().capi.load()
        if not _lib.q4_hip_init():
            raise RuntimeError("q4_hip_init failed")
    return _lib


def must(ok, what):
    if not ok:
        raise RuntimeError(what + " refused")


class State:
    pass


def random_codes(gen, *shape):
    """4-bit codes, two to a byte, as often as a block of normal values has them after division by its scale."""
    # the largest of 16 to 32 normal values, some 2.2 sigma, comes to 4 to 6: sigma is about 2.2 units of the block's scale
    below = torch.erf(torch.tensor(BORDERS, dtype=torch.float64) / (2.2 * math.sqrt(2.0)))
    share = torch.diff(torch.cat([torch.zeros(1, dtype=torch.float64), below, torch.ones(1, dtype=torch.float64)]))
    counts = torch.diff(torch.round(torch.cumsum(torch.cat([torch.zeros(1, dtype=torch.float64), share]), 0) * 128)).long()
    mag = torch.repeat_interleave(torch.arange(8), counts)
    table = torch.cat([mag, mag + 8]).to(torch.uint8).cuda()
    low = table[torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=gen).int()]
    high = table[torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=gen).int()]
    return low | (high << 4)


def weights(s, case, gen, n):
    """n matrices as a checkpoint holds them: codes, and a scale byte for each block."""
    m, k = matrix(case)
    s.codes = random_codes(gen, n, m, k // 2)
    shape = (n, m, k // BLOCK[case["type"]])
    if case["type"] == "mxfp4":      # 2^-9 to 2^-6
        s.scales = torch.randint(118, 122, shape, dtype=torch.uint8, device="cuda", generator=gen)
    else:                            # e4m3: 8 to 60, with a factor for the whole matrix beside them
        s.scales = torch.randint(0x50, 0x68, shape, dtype=torch.uint8, device="cuda", generator=gen)


def lay_out(s, case, lib, n):
    """The weights in the library's order, once; the checkpoint's form is then let go."""
    ty = TYPE[case["type"]]
    m, k = matrix(case)
    s.stride = lib.q4_cuda_fp4_bytes(ty, WEIGHTS, m, k)
    must(s.stride, "q4_cuda_fp4_bytes")
    s.w = torch.empty(n * s.stride, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    must(lib.q4_cuda_fp4_put(ty, s.codes.data_ptr(), s.scales.data_ptr(), m, k, n, s.w.data_ptr(), s.stride), "q4_cuda_fp4_put")
    lib.q4_hip_sync()
    s.codes = s.scales = None


def activations(gen, t, n):
    """Token rows: normal, with a few channels that carry much larger values."""
    x = torch.randn(t, n, device="cuda", generator=gen)
    loud = torch.rand(n, device="cuda", generator=gen) < 0.01
    return torch.where(loud, 8.0 * x, x)


def route(s, case, gen):
    """Which tokens every expert takes: rows sorted by expert, the shared expert (all tokens) last."""
    t, e, k = case["tokens"], case["experts"], case["topk"]
    logits = torch.log(popularity(case)).float().cuda() + torch.empty(t, e, device="cuda").exponential_(generator=gen).log_().neg_()
    picks = torch.topk(logits, k, dim=1).indices
    expert = torch.cat([picks.flatten(), torch.full((t,), e, device="cuda", dtype=torch.int64)])
    token = torch.cat([torch.arange(t, device="cuda").repeat_interleave(k), torch.arange(t, device="cuda")])
    order = torch.argsort(expert, stable=True)
    s.token = token[order].int()
    count = torch.bincount(expert, minlength=e + 1)
    s.bounds = torch.zeros(e + 1 + 1, dtype=torch.int32, device="cuda")
    s.bounds[1:] = torch.cumsum(count, 0).int()
    # the plain form's plan: tiles of at most TILE rows of one expert
    tiles = (count + TILE - 1) // TILE
    s.tile_expert = torch.repeat_interleave(torch.arange(e + 1, device="cuda"), tiles)
    within = torch.arange(len(s.tile_expert), device="cuda") - torch.repeat_interleave(torch.cumsum(tiles, 0) - tiles, tiles)
    at = s.bounds[:-1].long()[s.tile_expert] + within * TILE
    s.tile_row = at[:, None] + torch.arange(TILE, device="cuda")[None, :]
    s.tile_live = s.tile_row < s.bounds[1:].long()[s.tile_expert][:, None]
    s.tile_row = torch.where(s.tile_live, s.tile_row, torch.zeros_like(s.tile_row))


def data(case, seed):
    s = State()
    s.case = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, t = case["kind"], case["tokens"]
    if kind == "balance":
        e = case["experts"]
        # popular experts have a larger bias; a few rows are padding behind a batch's shorter sequences
        s.logits = torch.randn(t, e, device="cuda", generator=gen) + 0.7 * torch.randn(e, device="cuda", generator=gen)
        s.ids = torch.topk(s.logits, case["topk"], dim=1).indices.int().contiguous()
        s.valid = (torch.rand(t, device="cuda", generator=gen) < 0.95).to(torch.uint8)
        s.valid[0] = 1
        s.coef, s.gout = 0.01, torch.full((1,), 0.5, device="cuda")
        return s
    # NVFP4 rows are brought into the range of their scales by a calibrated factor, which the product takes out again
    s.mul = 1.0 if case["type"] == "mxfp4" else 224.0
    if kind == "store":
        s.x = activations(gen, t, case["embd"])
        return s
    s.scale = 1.0 if case["type"] == "mxfp4" else 2.0 ** -11 / 224.0
    n = 1 if kind == "linear" else case["experts"] + 1
    weights(s, case, gen, n)
    if kind == "linear":
        s.x = activations(gen, t, case["embd"])
        return s
    route(s, case, gen)
    s.each = None
    if case["type"] == "nvfp4":      # the matrices' own factors
        s.each = torch.rand(n, device="cuda", generator=gen) + 0.5
    if kind == "gate_up":
        s.x = activations(gen, t, case["embd"])
    else:
        s.gu = torch.randn(len(s.token), 2 * case["ff"], device="cuda", generator=gen)
    return s


def prepare(case, seed):
    s = data(case, seed)
    if not own:
        return s
    lib, kind, t = library(), case["kind"], case["tokens"]

    def out(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    def buffer(rows, cols):
        return out(lib.q4_cuda_fp4_bytes(TYPE[case["type"]], ROWS, rows, cols), dtype=torch.uint8)

    if kind == "balance":
        e = case["experts"]
        s.out = {"counts": out(e, dtype=torch.int32), "prob": out(e), "loss": out(1), "dlogits": out(t, e)}
        s.calls = [(lib.q4_cuda_route_balance, (s.logits.data_ptr(), s.ids.data_ptr(), s.valid.data_ptr(), t, e, s.ids.shape[1], s.coef,
                                                s.gout.data_ptr(), s.out["counts"].data_ptr(), s.out["prob"].data_ptr(),
                                                s.out["loss"].data_ptr(), s.out["dlogits"].data_ptr()))]
        torch.cuda.synchronize()
        return s
    ty = TYPE[case["type"]]
    if kind == "store":
        n = case["embd"]
        s.q, s.out = buffer(t, n), {"values": out(t, n)}
        s.calls = [(lib.q4_cuda_fp4_quantize, (ty, ROWS, s.x.data_ptr(), n, s.mul, t, n, s.q.data_ptr())),
                   (lib.q4_cuda_fp4_values, (ty, ROWS, s.q.data_ptr(), t, n, s.out["values"].data_ptr(), n))]
        torch.cuda.synchronize()
        return s
    m, k = matrix(case)
    if kind == "linear":
        lay_out(s, case, lib, 1)
        s.q, s.out = buffer(t, k), {"y": out(t, m)}
        s.calls = [(lib.q4_cuda_fp4_quantize, (ty, ROWS, s.x.data_ptr(), k, s.mul, t, k, s.q.data_ptr())),
                   (lib.q4_cuda_fp4_mul, (ty, s.w.data_ptr(), m, k, s.q.data_ptr(), t, s.scale, s.out["y"].data_ptr(), m))]
        torch.cuda.synchronize()
        return s
    n, rows = case["experts"] + 1, len(s.token)
    lay_out(s, case, lib, n)
    s.out = {"y": out(rows, m)}
    each = s.each.data_ptr() if s.each is not None else None
    if kind == "gate_up":
        s.q = buffer(t, k)
        s.calls = [(lib.q4_cuda_fp4_quantize, (ty, ROWS, s.x.data_ptr(), k, s.mul, t, k, s.q.data_ptr())),
                   (lib.q4_cuda_fp4_mul_id, (ty, s.w.data_ptr(), m, k, s.stride, n, s.q.data_ptr(), t, s.token.data_ptr(), s.bounds.data_ptr(),
                                             rows, s.scale, each, s.out["y"].data_ptr(), m))]
    else:
        s.q = buffer(rows, k)
        s.calls = [(lib.q4_cuda_fp4_swiglu_quantize, (ty, s.gu.data_ptr(), 2 * k, s.mul, rows, k, s.q.data_ptr())),
                   (lib.q4_cuda_fp4_mul_id, (ty, s.w.data_ptr(), m, k, s.stride, n, s.q.data_ptr(), rows, None, s.bounds.data_ptr(),
                                             rows, s.scale, each, s.out["y"].data_ptr(), m))]
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ one pass

def e2m1(v):
    """Nearest of the eight magnitudes, ties to the even code, 6 for all beyond it; keeps v's sign and type."""
    a = v.abs()
    code = torch.zeros(v.shape, dtype=torch.int32, device=v.device)
    for i, b in enumerate(BORDERS):
        code += (a >= b) if i % 2 else (a > b)
    return torch.copysign(torch.tensor(MAGNITUDES, dtype=v.dtype, device=v.device)[code], v)


def quantised(v, ty):
    """The values that v's rows stand for after quantisation, in 32 bits."""
    blocks = v.view(*v.shape[:-1], -1, BLOCK[ty])
    top = blocks.abs().amax(dim=-1, keepdim=True)
    if ty == "mxfp4":    # the power of two that brings the largest into [4, 8)
        power = (torch.frexp(top).exponent - 3).clamp(-127, 127)
        scale = torch.where(top > 0, torch.exp2(power.double()), torch.full_like(top, 2.0 ** -127, dtype=torch.float64)).to(v.dtype)
    else:                # a sixth of the largest, as e4m3: three bits behind the point, smallest step 2^-9
        want = (top / 6.0).double()
        step = torch.exp2((torch.frexp(want).exponent - 1).clamp(min=-6).double() - 3.0)
        scale = (torch.round(want / step) * step).clamp(max=448.0).to(v.dtype)
    codes = e2m1(blocks / torch.where(scale > 0, scale, torch.ones_like(scale)))
    return torch.where(scale > 0, codes * scale, torch.zeros_like(codes)).view(v.shape).float()


def dequantised(codes, scales, ty):
    """Matrices of a checkpoint as 32-bit values."""
    both = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    v = torch.stack([both[(codes & 15).int()], both[(codes >> 4).int()]], dim=-1).flatten(-2)
    s = torch.exp2(scales.float() - 127.0) if ty == "mxfp4" else scales.view(torch.float8_e4m3fn).float()
    return (v.view(*s.shape, BLOCK[ty]) * s[..., None]).view(v.shape)


def grouped(s, rows):
    """Every expert's matrix with its rows."""
    tiles = torch.bmm(rows[s.tile_row], dequantised(s.codes[s.tile_expert], s.scales[s.tile_expert], s.case["type"]).transpose(1, 2))
    tiles = tiles * s.scale
    if s.each is not None:
        tiles = tiles * s.each[s.tile_expert][:, None, None]
    y = torch.empty(len(s.token), tiles.shape[2], device=rows.device)
    y[s.tile_row[s.tile_live]] = tiles[s.tile_live]
    return {"y": y}


def run(s):
    if own:
        for call, args in s.calls:
            must(call(*args), call.__name__)
        return s.out
    kind, ty = s.case["kind"], s.case.get("type")
    if kind == "balance":
        t, e = s.logits.shape
        live = s.valid[:, None] != 0
        n = live.sum().float().clamp(min=1.0)
        z = torch.exp(s.logits - s.logits.amax(dim=1, keepdim=True))
        p = torch.where(live, z / z.sum(dim=1, keepdim=True), torch.zeros_like(z))
        counts = torch.zeros(e, dtype=torch.int32, device=p.device)
        counts.index_add_(0, s.ids.flatten(), live.int().expand(-1, s.ids.shape[1]).flatten())
        share = counts.float() / (n * s.ids.shape[1])
        prob = p.sum(dim=0) / n
        loss = s.coef * e * (share * prob).sum()
        inner = (p * share).sum(dim=1, keepdim=True)
        dlogits = s.gout * (s.coef * e / n) * p * (share - inner)
        return {"counts": counts, "prob": prob, "loss": loss.view(1), "dlogits": dlogits}
    if kind == "store":
        return {"values": quantised(s.x * s.mul, ty)}
    if kind == "linear":
        return {"y": quantised(s.x * s.mul, ty) @ dequantised(s.codes[0], s.scales[0], ty).T * s.scale}
    if kind == "gate_up":
        return grouped(s, quantised(s.x * s.mul, ty)[s.token])
    g, u = s.gu.double().chunk(2, dim=1)       # in 64 bits: a value next to a border falls on its right side
    return grouped(s, quantised(g / (1.0 + torch.exp(-g)) * u * s.mul, ty))


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = data(case, seed)
    kind = case["kind"]
    if kind == "balance":
        live = torch.nonzero(s.valid).flatten()
        n, e, k = len(live), case["experts"], s.ids.shape[1]
        x = s.logits.double()[live]
        p = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
        counts = torch.bincount(s.ids[live].long().flatten(), minlength=e)
        f = counts.double() / (n * k)
        g = torch.zeros(s.logits.shape, dtype=torch.float64, device="cuda")
        # loss = c sum_e f_e mean_t p_te, dp_te / dlogit_tj = p_te ([e = j] - p_tj)
        c = case["experts"] * s.coef
        g[live] = (p * f - p * (p @ f)[:, None]) * (c / n * float(s.gout))
        return {"counts": None, "prob": p.mean(dim=0), "loss": c * (f @ p.mean(dim=0)).view(1), "dlogits": g}
    ty, b = case["type"], BLOCK[case["type"]]

    def nearest(v):
        """v's blocks rounded to the format: of all its scales and codes the ones that the definition names."""
        v = v.reshape(-1, b)
        top = v.abs().max(dim=1).values
        if ty == "mxfp4":
            e = torch.floor(torch.log2(top))
            e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))
            scale = torch.exp2((e - 2).clamp(-127, 127))
        else:
            grid = torch.arange(0, 127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
            want = top / 6.0
            hi = torch.searchsorted(grid, want).clamp(1, 126)
            up, down = grid[hi] - want, want - grid[hi - 1]
            scale = grid[torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)]
        unit = torch.where(scale > 0, scale, 1.0)[:, None]
        a = (v.abs() / unit).clamp(max=6.0)
        # within a binade the numbers are a step apart; half to even, by torch.round
        step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
        return torch.round(a / step) * step * torch.sign(v) * scale[:, None]

    def values(q, sc):
        c = torch.stack([q & 15, q >> 4], dim=-1).reshape(q.shape[0], -1).int()
        e, m = (c >> 1) & 3, (c & 1).double()
        a = torch.where(e == 0, m * 0.5, (1.0 + m * 0.5) * torch.exp2((e - 1).double()))
        u = torch.exp2(sc.double() - 127.0) if ty == "mxfp4" else sc.view(torch.float8_e4m3fn).double()
        return torch.where(c >= 8, -a, a) * u.repeat_interleave(b, dim=1)

    if kind == "down":
        half = case["ff"]
        g, u = s.gu[:, :half].double(), s.gu[:, half:].double()
        rows = nearest(g * torch.sigmoid(g) * u * s.mul).view(g.shape)
    else:
        rows = nearest((s.x * s.mul).double()).view(s.x.shape)
    if kind == "store":
        return {"values": rows}
    if kind == "linear":
        return {"y": rows @ values(s.codes[0], s.scales[0]).T * s.scale}
    if kind == "gate_up":
        rows = rows[s.token.long()]
    m, _ = matrix(case)
    y = torch.empty(len(s.token), m, dtype=torch.float64, device="cuda")
    bounds = s.bounds.tolist()
    for e in range(case["experts"] + 1):
        lo, hi = bounds[e], bounds[e + 1]
        if lo < hi:
            y[lo:hi] = rows[lo:hi] @ values(s.codes[e], s.scales[e]).T * (s.scale * (1.0 if s.each is None else float(s.each[e])))
    return {"y": y}
