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
    int32_t *work;        // [0] tokens that count, [16 ..] picks of every expert
    float *part;          // [CTA][n_exp] sums of probabilities
};

__global__ void __launch_bounds__(256) clear_k(const Args a) {
    q4b_pdl_wait();
    for (uint32_t i = threadIdx.x; i < 16u + a.n_exp; i += blockDim.x) a.work[i] = 0;
}
__global__ void __launch_bounds__(256) count_k(const Args a) {
    __shared__ int32_t hist[MAX_E], n_live;
    q4b_pdl_wait();
    for (uint32_t i = threadIdx.x; i < a.n_exp; i += blockDim.x) hist[i] = 0;
    if (threadIdx.x == 0) n_live = 0;
    __syncthreads();
    const uint64_t n = (uint64_t)a.n_tok * a.topk, step = (uint64_t)gridDim.x * blockDim.x, at = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (uint64_t i = at; i < n; i += step) {
        const int32_t e = a.ids[i];
        if ((uint32_t)e < a.n_exp && (!a.valid || a.valid[i / a.topk])) atomicAdd(&hist[e], 1);
    }
    int32_t live = 0;
    for (uint64_t t = at; t < a.n_tok; t += step) live += !a.valid || a.valid[t];
    if (live) atomicAdd(&n_live, live);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.n_exp; i += blockDim.x)
        if (hist[i]) atomicAdd(&a.work[16u + i], hist[i]);
    if (threadIdx.x == 0 && n_live) atomicAdd(&a.work[0], n_live);
}

// A warp takes a token's row at a time, NV x 32 experts in registers; its sums of probabilities stay there too.
template <int NV> __global__ void __launch_bounds__(256) rows_k(const Args a) {
    __shared__ float f[MAX_E], sum[8][NV * 32];
    q4b_pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const int32_t n = a.work[0];
    const float inv_n = n ? 1.f / (float)n : 0.f, share = n ? 1.f / ((float)n * (float)a.topk) : 0.f;
    for (uint32_t i = threadIdx.x; i < NV * 32u; i += blockDim.x) f[i] = i < a.n_exp ? (float)a.work[16u + i] * share : 0.f;
    __syncthreads();
    const float g = (a.gout ? *a.gout : 1.f) * a.coef * (float)a.n_exp * inv_n;
    float acc[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) acc[i] = 0.f;
    for (uint32_t t = blockIdx.x * 8u + warp; t < a.n_tok; t += gridDim.x * 8u) {
        const float *row = a.logits + (uint64_t)t * a.n_exp;
        const bool live = !a.valid || a.valid[t];
        float p[NV], m = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const uint32_t e = i * 32u + lane;
            p[i] = live && e < a.n_exp ? row[e] : -INFINITY;
            m = fmaxf(m, p[i]);
        }
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
            inner = fmaf(p[i], f[i * 32u + lane], inner);
        }
        inner = q4b_warp_sum(inner);
        if (a.dlogits) {
            float *d = a.dlogits + (uint64_t)t * a.n_exp;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const uint32_t e = i * 32u + lane;
                if (e < a.n_exp) d[e] = live ? g * p[i] * (f[e] - inner) : 0.f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) sum[warp][i * 32u + lane] = acc[i];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.n_exp; e += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; w++) s += sum[w][e];
        a.part[(uint64_t)blockIdx.x * a.n_exp + e] = s;
    }
}

__global__ void __launch_bounds__(1024) finish_k(const Args a, uint32_t n_part) {
    __shared__ float red[32];
    q4b_pdl_wait();
    const int32_t n = a.work[0];
    const float inv_n = n ? 1.f / (float)n : 0.f, share = n ? 1.f / ((float)n * (float)a.topk) : 0.f;
    float l = 0.f;
    for (uint32_t e = threadIdx.x; e < a.n_exp; e += blockDim.x) {
        float s = 0.f;
        for (uint32_t c = 0; c < n_part; c++) s += a.part[(uint64_t)c * a.n_exp + e];
        const float p = s * inv_n;
        const int32_t c = a.work[16u + e];
        if (a.counts) a.counts[e] = c;
        if (a.prob) a.prob[e] = p;
        l = fmaf((float)c * share, p, l);
    }
    l = q4b_warp_sum(l);
    if ((threadIdx.x & 31u) == 0) red[threadIdx.x >> 5] = l;
    __syncthreads();
    if (threadIdx.x < 32u) {
        l = q4b_warp_sum(threadIdx.x < (blockDim.x >> 5) ? red[threadIdx.x] : 0.f);
        if (threadIdx.x == 0 && a.loss) *a.loss = a.coef * (float)a.n_exp * l;
    }
}

static int32_t *g_work = nullptr;
static float *g_part = nullptr;
}  // namespace balance

// The sums' scratch, once: calls come one after another on the library's stream.
bool q4b_balance_warm() {
    using namespace balance;
    if (g_work) return true;
    Q4B_CHECK(cudaMalloc(&g_work, (16u + MAX_E) * sizeof(int32_t)));
    Q4B_CHECK(cudaMalloc(&g_part, (size_t)g_q4b.n_sm * MAX_E * sizeof(float)));
    return true;
}
void q4b_balance_shutdown() {
    using namespace balance;
    if (g_work) cudaFree(g_work);
    if (g_part) cudaFree(g_part);
    g_work = nullptr;
    g_part = nullptr;
}

extern "C" bool q4_cuda_route_balance(const float *d_logits, const int32_t *d_ids, const uint8_t *d_valid, uint32_t n_tok, uint32_t n_exp, uint32_t topk,
                                      float coef, const float *d_gout, int32_t *d_counts, float *d_prob, float *d_loss, float *d_dlogits) {
    using namespace balance;
    if (!g_q4b.ok || !g_work || !d_logits || !d_ids || !n_tok || n_tok > 0x7fffffu || !n_exp || n_exp > MAX_E || !topk || topk > 64u ||
        (((uintptr_t)d_logits | (uintptr_t)d_ids | (uintptr_t)d_gout | (uintptr_t)d_counts | (uintptr_t)d_prob | (uintptr_t)d_loss | (uintptr_t)d_dlogits) & 3u))
        return false;
    fp4::OnDevice dev;
    const Args a = {d_logits, d_ids, d_valid, n_tok, n_exp, topk, coef, d_gout, d_counts, d_prob, d_loss, d_dlogits, g_work, g_part};
    const uint32_t sm = (uint32_t)g_q4b.n_sm;
    const uint32_t want = (n_tok * topk + 1023u) / 1024u;
    q4b_launch(clear_k, dim3(1), dim3(256), 0, g_q4b.stream, a);
    q4b_launch(count_k, dim3(want < sm ? want : sm), dim3(256), 0, g_q4b.stream, a);
    const uint32_t ctas = (n_tok + 7u) / 8u < sm ? (n_tok + 7u) / 8u : sm;
    auto go = [&](auto k) { q4b_launch(k, dim3(ctas), dim3(256), 0, g_q4b.stream, a); };
    if (n_exp <= 128u) go(rows_k<4>);
    else if (n_exp <= 512u) go(rows_k<16>);
    else go(rows_k<32>);
    q4b_launch(finish_k, dim3(1), dim3(1024), 0, g_q4b.stream, a, ctas);
    g_q4b_launches += 4;
    return q4b_launch_ok("route balance");
}
