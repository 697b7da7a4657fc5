// How evenly a router spreads its tokens: picks per expert, mean probabilities, the balance loss and its gradient.
// Part of the single translation unit q4cuda.cu.
//
// With n tokens that count, k picks each, E experts and p_t = softmax(logits_t):
//   f_e = (picks of e) / (n k),  P_e = (1 / n) sum_t p_te,  loss = c E sum_e f_e P_e
//   d loss / d logits_tj = (c E / n) p_tj (f_j - sum_e f_e p_te)      (the picks are integers: f has no derivative)
// f is known before the logits are looked at, so that loss and gradient are one pass over them.
namespace balance {

constexpr uint32_t MAX_E = 1024u, CL = 8u;      // experts; CTAs of a cluster
struct Args {
    const float *logits;
    const int32_t *ids;
    const uint8_t *valid;
    uint32_t n_tok, n_exp, topk;
    float coef;
    const float *gout;
    int32_t *counts;
    float *prob, *loss, *dlogits;
    float *part;          // [cluster][n_exp] sums of probabilities
    uint32_t *done;       // CTAs that are through
};

// Picks of a slice of the tokens, with shared-memory counters; returns after a barrier.
__device__ __forceinline__ void count(const Args &a, uint32_t cta, uint32_t ctas, int32_t *hist, int32_t *n_live) {
    for (uint32_t i = threadIdx.x; i < a.n_exp; i += blockDim.x) hist[i] = 0;
    if (threadIdx.x == 0) *n_live = 0;
    __syncthreads();
    int32_t live = 0;
    const uint32_t step = ctas * blockDim.x;
    for (uint32_t t0 = cta * blockDim.x + threadIdx.x; t0 < a.n_tok; t0 += 2u * step)        // two tokens' loads at a time
        for (uint32_t k0 = 0; k0 < a.topk; k0 += 16u) {
            int32_t e[2][16];
            bool ok[2];
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                const uint32_t t = t0 + h * step;
                ok[h] = t < a.n_tok;
#pragma unroll
                for (uint32_t k = 0; k < 16u; k++) e[h][k] = ok[h] && k0 + k < a.topk ? a.ids[(uint64_t)t * a.topk + k0 + k] : -1;
                if (ok[h] && a.valid) ok[h] = a.valid[t] != 0;
            }
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                live += ok[h] && k0 == 0;
#pragma unroll
                for (uint32_t k = 0; k < 16u; k++)
                    if (ok[h] && (uint32_t)e[h][k] < a.n_exp) atomicAdd(&hist[e[h][k]], 1);
            }
        }
    live = __reduce_add_sync(0xffffffffu, live);
    if ((threadIdx.x & 31u) == 0 && live) atomicAdd(n_live, live);
    __syncthreads();
}
// A value of another CTA's shared memory, by this CTA's address of it.
__device__ __forceinline__ uint32_t peer_word(const void *p, uint32_t cta) {
    uint32_t a, v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 2^x to 2 steps of 2^-23; x is a rounded multiple of log2(e), off by |x| 2^-24: a probability that matters has a small one.
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// One launch.  Every cluster of eight CTAs counts all picks, an eighth a CTA, and adds the eighths up through distributed shared
// memory.  Then a warp takes a token's row at a time, 32 NV experts in registers (VEC: four neighbours a lane and load); its sums
// of probabilities stay there too.  They are added up in a fixed order: over the warps of a CTA in shared memory, over the
// CTAs of a cluster (each takes an eighth of the experts), over the clusters by the last CTA to come to its end.  A chain of
// short steps: 8192 x 512, top-10, 16.1 us with inputs in the L2 and 17.5 with three sets of inputs in turn, of them counts 3, rows 5.8
// (5.8 TB/s), sums and their barriers 5; 64 x 512 8.4.  (Four launches, with counts by global atomics, took 33.6 and 10.5.)
// Warps of a CTA: as many as have registers for a row and its sums.
__host__ __device__ constexpr uint32_t warps(int nv) { return nv > 16 ? 16u : nv > 4 ? 24u : 32u; }
template <int NV, bool VEC> __global__ void __launch_bounds__(32u * warps(NV)) rows_k(const Args a) {
    constexpr uint32_t W = warps(NV), N = NV * 32u;
    __shared__ __align__(16) float f[N];
    __shared__ __align__(16) float sum[W / 2u][N];
    __shared__ int32_t hist[N], total[N], n_here;
    __shared__ float red[W];
    __shared__ bool last;
    q4b_pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    auto at = [&](int i) { return VEC ? (uint32_t)(i >> 2) * 128u + lane * 4u + (i & 3u) : (uint32_t)i * 32u + lane; };   // expert of register i
    float p[NV];
    auto load = [&](uint32_t t) {             // (padding is read, too: nobody waits for its mark)
        if (t >= a.n_tok) return;
        const float *row = a.logits + (uint64_t)t * a.n_exp;
        if (VEC) {
#pragma unroll
            for (int i = 0; i < NV; i += 4) {
                float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (at(i) < a.n_exp) v = *reinterpret_cast<const float4 *>(row + at(i));
                p[i] = v.x, p[i + 1] = v.y, p[i + 2] = v.z, p[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++) p[i] = at(i) < a.n_exp ? row[at(i)] : -INFINITY;
        }
    };
    const uint32_t rank = blockIdx.x % CL, clusters = gridDim.x / CL, step = gridDim.x * W;
    uint32_t t = blockIdx.x * W + warp;
    load(t);                                  // the first row comes while the picks are counted
    count(a, rank, CL, hist, &n_here);
    cluster_sync();
    int32_t n_live = 0;
#pragma unroll
    for (uint32_t c = 0; c < CL; c++) n_live += (int32_t)peer_word(&n_here, c);
    // (quotients, not products with rounded inverses: one an expert, and one a launch; no token that counts: 0 / 1)
    const float n_f = n_live ? (float)n_live : 1.f, picks = n_f * (float)a.topk;
    for (uint32_t i = threadIdx.x; i < N; i += blockDim.x) {
        int32_t n = 0;
        if (i < a.n_exp)
#pragma unroll
            for (uint32_t c = 0; c < CL; c++) n += (int32_t)peer_word(&hist[i], c);
        total[i] = n;
        f[i] = n_live ? __fdiv_rn((float)n, picks) : 0.f;
    }
    __syncthreads();
    const float g = __fdiv_rn((a.gout ? *a.gout : 1.f) * a.coef * (float)a.n_exp, n_f);
    float acc[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) acc[i] = 0.f;
    for (; t < a.n_tok; t += step, load(t)) {
        const bool live = !a.valid || a.valid[t];
        float *d = a.dlogits + (uint64_t)t * a.n_exp;
        if (live) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < NV; i++) m = fmaxf(m, p[i]);
            m = q4b_warp_max(m);
            if (m == -INFINITY) m = 0.f;              // a row without any expert: all exponentials are 0
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                p[i] = exp2_approx((p[i] - m) * 1.4426950408889634f);
                s += p[i];
            }
            s = q4b_warp_sum(s);
            const float inv = s == 0.f ? 0.f : __fdiv_rn(1.f, s);
            float inner = 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                p[i] *= inv;
                acc[i] += p[i];
                inner = fmaf(p[i], f[at(i)], inner);
            }
            if (!a.dlogits) continue;
            inner = q4b_warp_sum(inner);
#pragma unroll
            for (int i = 0; i < NV; i++) p[i] = g * p[i] * (f[at(i)] - inner);
        } else {
            if (!a.dlogits) continue;
#pragma unroll
            for (int i = 0; i < NV; i++) p[i] = 0.f;
        }
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
    for (uint32_t e = threadIdx.x; e < a.n_exp; e += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < W / 2u; w++) s += sum[w][e];
        sum[0][e] = s;           // (a column is one thread's)
    }
    cluster_sync();
    const bool alone = clusters == 1u;
    const uint32_t slice = (a.n_exp + CL - 1u) / CL, e0 = alone ? 0u : rank * slice, e1 = alone ? (rank ? 0u : a.n_exp) : min(e0 + slice, a.n_exp);
    for (uint32_t e = e0 + threadIdx.x; e < e1; e += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (uint32_t c = 0; c < CL; c++) s += __uint_as_float(peer_word(&sum[0][e], c));
        if (alone) sum[1][e] = s;
        else a.part[(uint64_t)(blockIdx.x / CL) * a.n_exp + e] = s;
    }
    if (!alone) {
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last = atomicInc(a.done, gridDim.x - 1u) == gridDim.x - 1u;     // back at 0 behind the last one
    }
    cluster_sync();              // nobody reads a CTA that has gone
    if (alone ? rank != 0u : !last) return;
    __threadfence();
    float l = 0.f;
    for (uint32_t e = threadIdx.x; e < a.n_exp; e += blockDim.x) {
        float s = alone ? sum[1][e] : 0.f;
        if (!alone)
            for (uint32_t c0 = 0; c0 < clusters; c0 += 16u) {
                float p[16];
#pragma unroll
                for (uint32_t c = 0; c < 16u; c++) p[c] = c0 + c < clusters ? __ldcg(a.part + (uint64_t)(c0 + c) * a.n_exp + e) : 0.f;
#pragma unroll
                for (uint32_t c = 0; c < 16u; c++) s += p[c];
            }
        const float p = __fdiv_rn(s, n_f);
        if (a.counts) a.counts[e] = total[e];
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

static uint32_t *g_done = nullptr;
static float *g_part = nullptr;
static uint32_t g_clusters = 0;       // that run at a time

template <int NV, bool VEC> bool launch(const Args &a, uint32_t clusters, uint32_t *most) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CL * clusters);
    cfg.blockDim = dim3(32u * warps(NV));
    cfg.stream = g_q4b.stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CL, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    if (most) {
        int n = 0;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, rows_k<NV, VEC>, &cfg) != cudaSuccess || n < 1) return false;
        *most = (uint32_t)n;
        return true;
    }
    (void)cudaLaunchKernelEx(&cfg, rows_k<NV, VEC>, a);
    g_q4b_launches++;
    return q4b_launch_ok("route balance");
}
}  // namespace balance

// The sums' scratch, once: calls come one after another on the library's stream.  Where it cannot be had, the rest of the library
// works without: nothing is held, no error is left, and the call refuses.
void q4b_balance_shutdown() {
    using namespace balance;
    cudaFree(g_done);
    cudaFree(g_part);
    g_done = nullptr;
    g_part = nullptr;
}
bool q4b_balance_warm() {
    using namespace balance;
    if (g_done) return true;
    uint32_t n = 0;
    if (launch<16, true>(Args{}, 1u, &n) && cudaMalloc(&g_part, (size_t)n * MAX_E * sizeof(float)) == cudaSuccess &&
        cudaMalloc(&g_done, 256) == cudaSuccess && cudaMemset(g_done, 0, 256) == cudaSuccess) {
        g_clusters = n;
        return true;
    }
    q4b_balance_shutdown();
    cudaGetLastError();
    return false;
}

extern "C" bool q4_cuda_route_balance(const float *d_logits, const int32_t *d_ids, const uint8_t *d_valid, uint32_t n_tok, uint32_t n_exp, uint32_t topk,
                                      float coef, const float *d_gout, int32_t *d_counts, float *d_prob, float *d_loss, float *d_dlogits) {
    using namespace balance;
    if (!g_q4b.ok || !g_done || !d_logits || !d_ids || !n_tok || n_tok > 0x7fffffu || !n_exp || n_exp > MAX_E || !topk || topk > 64u ||
        (((uintptr_t)d_logits | (uintptr_t)d_ids | (uintptr_t)d_gout | (uintptr_t)d_counts | (uintptr_t)d_prob | (uintptr_t)d_loss | (uintptr_t)d_dlogits) & 3u))
        return false;
    fp4::OnDevice dev;
    const Args a = {d_logits, d_ids, d_valid, n_tok, n_exp, topk, coef, d_gout, d_counts, d_prob, d_loss, d_dlogits, g_part, g_done};
    const uint32_t rows = CL * (n_exp > 512u ? warps(32) : n_exp > 128u ? warps(16) : warps(4)), want = (n_tok + rows - 1u) / rows, n = want < g_clusters ? want : g_clusters;
    const bool vec = n_exp % 4u == 0 && (((uintptr_t)d_logits | (uintptr_t)d_dlogits) & 15u) == 0;
    if (n_exp <= 128u) return vec ? launch<4, true>(a, n, nullptr) : launch<4, false>(a, n, nullptr);
    if (n_exp <= 512u) return vec ? launch<16, true>(a, n, nullptr) : launch<16, false>(a, n, nullptr);
    return vec ? launch<32, true>(a, n, nullptr) : launch<32, false>(a, n, nullptr);
}
