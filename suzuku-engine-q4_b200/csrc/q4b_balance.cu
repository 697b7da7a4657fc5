// How evenly a router spreads its tokens: picks per expert, mean probabilities, the balance loss and its gradient.
// Part of the single translation unit q4cuda.cu.
//
// With n tokens that count, k picks each, E experts and p_t = softmax(logits_t):
//   f_e = (picks of e) / (n k),  P_e = (1 / n) sum_t p_te,  loss = c E sum_e f_e P_e
//   d loss / d logits_tj = (c E / n) p_tj (f_j - sum_e f_e p_te)      (the picks are integers: f has no derivative)
// f is known before the logits are looked at, so that loss and gradient are one pass over them.
namespace balance {

constexpr uint32_t MAX_E = 1024u;
struct Args {
    const float *logits;
    const int32_t *ids;
    const uint8_t *valid;
    uint32_t n_tok, n_exp, topk;
    float coef;
    const float *gout;
    int32_t *counts;
    float *prob, *loss, *dlogits;
    int32_t *hist;        // [count CTA][1 + n_exp]: tokens that count, picks of every expert
    uint32_t n_hist;      // 0: the one CTA of rows_k counts by itself
    float *part;          // [CTA][n_exp] sums of probabilities
    uint32_t *done;       // CTAs of rows_k that are through
};

// Picks of a slice of the tokens, with shared-memory counters; returns after a barrier.
__device__ __forceinline__ void count(const Args &a, uint32_t cta, uint32_t ctas, int32_t *hist, int32_t *n_live) {
    for (uint32_t i = threadIdx.x; i < a.n_exp; i += blockDim.x) hist[i] = 0;
    if (threadIdx.x == 0) *n_live = 0;
    __syncthreads();
    const uint32_t n = a.n_tok * a.topk, step = ctas * blockDim.x, at = cta * blockDim.x + threadIdx.x;       // below 2^29
    for (uint32_t i = at; i < n; i += step) {
        const int32_t e = a.ids[i];
        if ((uint32_t)e < a.n_exp && (!a.valid || a.valid[i / a.topk])) atomicAdd(&hist[e], 1);
    }
    int32_t live = 0;
    for (uint32_t t = at; t < a.n_tok; t += step) live += !a.valid || a.valid[t];
    live = __reduce_add_sync(0xffffffffu, live);
    if ((threadIdx.x & 31u) == 0 && live) atomicAdd(n_live, live);
    __syncthreads();
}
__global__ void __launch_bounds__(1024) count_k(const Args a) {
    __shared__ int32_t hist[MAX_E], n_live;
    q4b_pdl_wait();
    count(a, blockIdx.x, gridDim.x, hist, &n_live);
    int32_t *o = a.hist + (uint64_t)blockIdx.x * (1u + a.n_exp);
    if (threadIdx.x == 0) o[0] = n_live;
    for (uint32_t i = threadIdx.x; i < a.n_exp; i += blockDim.x) o[1u + i] = hist[i];
}

// A warp takes a token's row at a time, 32 NV experts in registers (VEC: four neighbours a lane and load); its sums of
// probabilities stay there too.  They are added up in a fixed order: over the warps of a CTA in shared memory, over the CTAs by
// the last one to come to its end.  Bound by the reads of the logits and the writes of the gradient: 32 warps an SM have
// a row each in flight.
template <int NV, bool VEC> __global__ void __launch_bounds__(NV > 16 ? 512 : 1024) rows_k(const Args a) {
    constexpr uint32_t W = NV > 16 ? 16u : 32u, N = NV * 32u;
    __shared__ __align__(16) float f[N];
    __shared__ __align__(16) float sum[W / 2u][N];
    __shared__ int32_t hist[N], n_live;
    __shared__ float red[W];
    __shared__ bool last;
    q4b_pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    auto at = [&](int i) { return VEC ? (uint32_t)(i >> 2) * 128u + lane * 4u + (i & 3u) : (uint32_t)i * 32u + lane; };   // expert of register i
    if (a.n_hist) {
        for (uint32_t e = threadIdx.x; e <= a.n_exp; e += blockDim.x) {
            int32_t s = 0;
#pragma unroll 8
            for (uint32_t c = 0; c < a.n_hist; c++) s += a.hist[(uint64_t)c * (1u + a.n_exp) + e];
            if (e == 0) n_live = s;
            else hist[e - 1u] = s;
        }
        __syncthreads();
    } else {
        count(a, 0, 1, hist, &n_live);
    }
    const float inv_n = n_live ? 1.f / (float)n_live : 0.f, share = n_live ? 1.f / ((float)n_live * (float)a.topk) : 0.f;
    for (uint32_t i = threadIdx.x; i < N; i += blockDim.x) f[i] = i < a.n_exp ? (float)hist[i] * share : 0.f;
    __syncthreads();
    const float g = (a.gout ? *a.gout : 1.f) * a.coef * (float)a.n_exp * inv_n;
    float acc[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) acc[i] = 0.f;
    for (uint32_t t = blockIdx.x * W + warp; t < a.n_tok; t += gridDim.x * W) {
        const float *row = a.logits + (uint64_t)t * a.n_exp;
        const bool live = !a.valid || a.valid[t];
        float p[NV], m = -INFINITY;
        if (VEC) {
#pragma unroll
            for (int i = 0; i < NV; i += 4) {
                float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (live && at(i) < a.n_exp) v = *reinterpret_cast<const float4 *>(row + at(i));
                p[i] = v.x, p[i + 1] = v.y, p[i + 2] = v.z, p[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++) p[i] = live && at(i) < a.n_exp ? row[at(i)] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) m = fmaxf(m, p[i]);
        m = q4b_warp_max(m);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            p[i] = m == -INFINITY && p[i] == p[i] ? 0.f : expf(p[i] - m);      // a row without any expert has no probabilities
            s += p[i];
        }
        s = q4b_warp_sum(s);
        const float inv = s == 0.f ? 0.f : 1.f / s;
        float inner = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            p[i] *= inv;
            acc[i] += p[i];
            inner = fmaf(p[i], f[at(i)], inner);
        }
        if (!a.dlogits) continue;
        inner = q4b_warp_sum(inner);
        float *d = a.dlogits + (uint64_t)t * a.n_exp;
#pragma unroll
        for (int i = 0; i < NV; i++) p[i] = live ? g * p[i] * (f[at(i)] - inner) : 0.f;
        if (VEC) {
#pragma unroll
            for (int i = 0; i < NV; i += 4)
                if (at(i) < a.n_exp) *reinterpret_cast<float4 *>(d + at(i)) = make_float4(p[i], p[i + 1], p[i + 2], p[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (at(i) < a.n_exp) d[at(i)] = p[i];
        }
    }
    if (warp >= W / 2u) {
#pragma unroll
        for (int i = 0; i < NV; i++) sum[warp - W / 2u][at(i)] = acc[i];
    }
    __syncthreads();
    if (warp < W / 2u) {
#pragma unroll
        for (int i = 0; i < NV; i++) sum[warp][at(i)] += acc[i];
    }
    __syncthreads();
    const bool alone = gridDim.x == 1u;
    for (uint32_t e = threadIdx.x; e < a.n_exp; e += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < W / 2u; w++) s += sum[w][e];
        if (alone) sum[0][e] = s;           // (a column is one thread's)
        else a.part[(uint64_t)blockIdx.x * a.n_exp + e] = s;
    }
    if (!alone) {
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last = atomicInc(a.done, gridDim.x - 1u) == gridDim.x - 1u;     // back at 0 behind the last one
        __syncthreads();
        if (!last) return;
        __threadfence();
        // W / 2 groups of threads add up a run of the CTAs' sums each, then the groups' are added
        const uint32_t grp = warp >> 1, run = (gridDim.x + W / 2u - 1u) / (W / 2u), c0 = grp * run, c1 = min(c0 + run, gridDim.x);
        for (uint32_t e = (warp & 1u) * 32u + lane; e < a.n_exp; e += 64u) {
            float s = 0.f;
#pragma unroll 10
            for (uint32_t c = c0; c < c1; c++) s += __ldcg(a.part + (uint64_t)c * a.n_exp + e);
            sum[grp][e] = s;
        }
    }
    __syncthreads();
    float l = 0.f;
    for (uint32_t e = threadIdx.x; e < a.n_exp; e += blockDim.x) {
        float s = sum[0][e];
        if (!alone)
#pragma unroll
            for (uint32_t w = 1; w < W / 2u; w++) s += sum[w][e];
        const float p = s * inv_n;
        if (a.counts) a.counts[e] = hist[e];
        if (a.prob) a.prob[e] = p;
        l = fmaf(f[e], p, l);
    }
    l = q4b_warp_sum(l);
    if (lane == 0) red[warp] = l;
    __syncthreads();
    if (warp == 0) {
        l = q4b_warp_sum(lane < W ? red[lane] : 0.f);
        if (lane == 0 && a.loss) *a.loss = a.coef * (float)a.n_exp * l;
    }
}

constexpr uint32_t MAX_HIST = 32u;
static int32_t *g_hist = nullptr;
static uint32_t *g_done = nullptr;
static float *g_part = nullptr;
}  // namespace balance

// The sums' scratch, once: calls come one after another on the library's stream.
bool q4b_balance_warm() {
    using namespace balance;
    if (g_hist) return true;
    Q4B_CHECK(cudaMalloc(&g_done, 256));
    Q4B_CHECK(cudaMemset(g_done, 0, 256));
    Q4B_CHECK(cudaMalloc(&g_part, (size_t)g_q4b.n_sm * MAX_E * sizeof(float)));
    Q4B_CHECK(cudaMalloc(&g_hist, (size_t)MAX_HIST * (1u + MAX_E) * sizeof(int32_t)));
    return true;
}
void q4b_balance_shutdown() {
    using namespace balance;
    cudaFree(g_hist);
    cudaFree(g_done);
    cudaFree(g_part);
    g_hist = nullptr;
    g_done = nullptr;
    g_part = nullptr;
}

extern "C" bool q4_cuda_route_balance(const float *d_logits, const int32_t *d_ids, const uint8_t *d_valid, uint32_t n_tok, uint32_t n_exp, uint32_t topk,
                                      float coef, const float *d_gout, int32_t *d_counts, float *d_prob, float *d_loss, float *d_dlogits) {
    using namespace balance;
    if (!g_q4b.ok || !g_hist || !d_logits || !d_ids || !n_tok || n_tok > 0x7fffffu || !n_exp || n_exp > MAX_E || !topk || topk > 64u ||
        (((uintptr_t)d_logits | (uintptr_t)d_ids | (uintptr_t)d_gout | (uintptr_t)d_counts | (uintptr_t)d_prob | (uintptr_t)d_loss | (uintptr_t)d_dlogits) & 3u))
        return false;
    fp4::OnDevice dev;
    Args a = {d_logits, d_ids, d_valid, n_tok, n_exp, topk, coef, d_gout, d_counts, d_prob, d_loss, d_dlogits, g_hist, 0u, g_part, g_done};
    const uint32_t sm = (uint32_t)g_q4b.n_sm, warps = n_exp > 512u ? 16u : 32u;
    uint32_t ctas = (n_tok + warps - 1u) / warps;
    if (ctas > sm) ctas = sm;
    if (n_tok <= 4u * warps) ctas = 1;       // up to four rows a warp: one CTA, one launch
    if (ctas > 1u) {
        a.n_hist = (n_tok * topk + 2047u) / 2048u;
        if (a.n_hist > MAX_HIST) a.n_hist = MAX_HIST;
        q4b_launch(count_k, dim3(a.n_hist), dim3(1024), 0, g_q4b.stream, a);
        g_q4b_launches++;
    }
    const bool vec = n_exp % 4u == 0 && (((uintptr_t)d_logits | (uintptr_t)d_dlogits) & 15u) == 0;
    auto go = [&](auto k) { q4b_launch(k, dim3(ctas), dim3(32u * warps), 0, g_q4b.stream, a); };
    if (n_exp <= 128u) vec ? go(rows_k<4, true>) : go(rows_k<4, false>);
    else if (n_exp <= 512u) vec ? go(rows_k<16, true>) : go(rows_k<16, false>);
    else vec ? go(rows_k<32, true>) : go(rows_k<32, false>);
    g_q4b_launches++;
    return q4b_launch_ok("route balance");
}
