// The product of MXFP4 and NVFP4 matrices on the tensor cores.  Part of the single translation unit q4cuda.cu.
//
// tcgen05.mma.kind::mxf4 / mxf4nvf4 multiplies the codes and their scales as they are stored: 128 rows of x times BN rows of W,
// 64 values of k an instruction, fp32 sums in tensor memory.  The kernel is persistent; a CTA takes tiles of
// 128 x BN of the result (an expert's rows begin at any row; its last tile has fewer), and its warps have a task each:
//   warp 0     copies: codes of x and W (TMA, 128-byte swizzle: 256 values of a row a stage), W's scales (bulk).  Gathered rows
//              of x come by four (tile::gather4)
//   warp 2     the scales of x: words of [word][row] that land where the tensor memory's layout wants them (cp.async)
//   warp 1     brings a stage's scales to tensor memory (tcgen05.cp) and issues its MMAs
//   warps 4-7  read a finished accumulator, apply the factor, transpose 32 x 32 in shared memory and store whole lines, while
//              the MMAs fill the other one
// Scales in tensor memory: 128 rows' words are 4 columns (row r in lane r % 32 of column r / 32, copied to the four lane
// quarters), a word serves 128 values of k in MXFP4 (two MMAs, told apart in the instruction descriptor), 64 in NVFP4.
namespace fp4 {

using mmqtc::elect_one;
using mmqtc::mbar_arrive;
using mmqtc::mbar_expect_tx;
using mmqtc::mbar_init;
using mmqtc::mbar_look;
using mmqtc::mma_commit;
using mmqtc::smem_desc_sw128;
using mmqtc::smem_u32;
using mmqtc::tc_fence_after;
using mmqtc::tc_fence_before;
using mmqtc::tma_load_2d;
using mmqtc::tmem_ld_wait;

constexpr uint32_t ERR_FP4 = 1u << 20;
constexpr uint32_t BM = 128u, KSTAGE = 256u;
constexpr uint32_t MAX_EXPERTS = 1024u;

template <bool NVF, uint32_t BN> struct Cfg {
    static constexpr uint32_t WPS = NVF ? 4u : 2u;                 // scale words of a row a stage
    static constexpr uint32_t ATOMS = BN > 128u ? 2u : 1u;         // 128-row blocks of W's scales under a tile
    static constexpr uint32_t A = BM * 128u, B = BN * 128u, SA = WPS * 512u, SB = WPS * ATOMS * 512u;
    static constexpr uint32_t STAGE = A + B + SA + SB;
    static constexpr uint32_t FIXED = 24u * 1024u;                 // barriers, tile table, the epilogue's transpose
    static constexpr uint32_t NS = (227u * 1024u - FIXED) / STAGE > 8u ? 8u : (227u * 1024u - FIXED) / STAGE;
    static constexpr uint32_t SMEM = FIXED + NS * STAGE;
    static constexpr uint32_t SF_COLS = WPS * 4u * (1u + ATOMS);   // tensor memory columns of a stage's scales
    static constexpr uint32_t SF_AT = 2u * BN;
    static_assert(SF_AT + 2u * SF_COLS <= 512u && NS >= 4u && STAGE % 1024u == 0u, "layout");
};
struct TcSmem {
    unsigned long long full[8], empty[8], acc_full[2], acc_empty[2];
    uint32_t tmem, warp_sum[8];
    uint32_t first[MAX_EXPERTS + 1];       // tiles of rows before every expert
    __align__(16) uint8_t out[4][4096];    // the epilogue warps' 32 x 32 blocks
};
static_assert(sizeof(TcSmem) <= 24u * 1024u, "shared memory layout");
struct TcMaps {
    CUtensorMap x, xg, w;                  // 32 rows of x; one row of x (gather); BN rows of an expert's W
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, unsigned long long *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, unsigned long long *bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_gather4(void *dst, const CUtensorMap *map, unsigned long long *bar, int c0, const int *r) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(c0), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(smem_u32(bar))
        : "memory");
}
// 512 bytes (32 lanes x 4 columns, for all four lane quarters) from shared to tensor memory
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint32_t smem) {
    // no swizzle; groups of 8 x 16 bytes 128 bytes apart
    const uint64_t d = (uint64_t)((smem >> 4) & 0x3fffu) | ((uint64_t)8u << 32) | (1ull << 46);
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}
template <bool NVF> __device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    if (NVF)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *f) {
    uint32_t *v = reinterpret_cast<uint32_t *>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
          "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(taddr)
        : "memory");
}

struct Tile {
    uint32_t e, n0;
    int32_t m0, rows;      // first row of the result, rows
};

template <bool NVF, uint32_t BN> __global__ void __launch_bounds__(256, 1) tc_k(const MArgs a, const __grid_constant__ TcMaps maps) {
    using C = Cfg<NVF, BN>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *const ring = smem_raw;                                 // stages: codes of x, codes of W, scales of x, scales of W
    TcSmem &s = *reinterpret_cast<TcSmem *>(smem_raw + C::NS * C::STAGE);
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    q4b_pdl_wait();
    if (tid == 0) {
        for (uint32_t i = 0; i < C::NS; i++) mbar_init(&s.full[i], 2), mbar_init(&s.empty[i], 1);
        for (uint32_t i = 0; i < 2u; i++) mbar_init(&s.acc_full[i], 1), mbar_init(&s.acc_empty[i], 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // rows of every expert in tiles of 128, summed up
    auto first_row = [&](uint32_t e) { return min(max(a.bounds[e], 0), (int32_t)a.total); };
    uint32_t m_tiles;
    if (a.bounds) {
        uint32_t c[4], sum = 0;
        for (uint32_t i = 0; i < 4u; i++) {
            const uint32_t e = tid * 4u + i;
            c[i] = e < a.n_expert ? (uint32_t)(max(first_row(e + 1u) - first_row(e), 0) + 127) / 128u : 0u;
            sum += c[i];
        }
        uint32_t inc = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += t;
        }
        if (lane == 31u) s.warp_sum[warp] = inc;
        __syncthreads();
        uint32_t at = inc - sum;
        m_tiles = 0;
        for (uint32_t w = 0; w < 8u; w++) {
            if (w < warp) at += s.warp_sum[w];
            m_tiles += s.warp_sum[w];
        }
        for (uint32_t i = 0; i < 4u; i++) {
            if (tid * 4u + i <= a.n_expert) s.first[tid * 4u + i] = at;
            at += c[i];
        }
        if (tid == 255u && a.n_expert == MAX_EXPERTS) s.first[MAX_EXPERTS] = at;
    } else {
        m_tiles = (uint32_t)((a.total + 127u) / 128u);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    const uint32_t n_tiles = (a.w_rows + BN - 1u) / BN, n_ks = (a.cols + KSTAGE - 1u) / KSTAGE, all = m_tiles * n_tiles;
    auto tile_of = [&](uint32_t t) {
        Tile r;
        const uint32_t m = t / n_tiles;
        r.n0 = (t - m * n_tiles) * BN;
        r.e = 0;
        if (a.bounds) {
            uint32_t lo = 0, hi = a.n_expert;        // the last expert whose first tile is not behind m: one that has rows
            while (hi - lo > 1u) {
                const uint32_t k = (lo + hi) >> 1;
                if (s.first[k] <= m) lo = k; else hi = k;
            }
            r.e = lo;
            r.m0 = first_row(lo) + (int32_t)(m - s.first[lo]) * 128;
            r.rows = min(first_row(lo + 1u) - r.m0, 128);
        } else {
            r.m0 = (int32_t)(m * 128u);
            r.rows = min((int32_t)a.total - r.m0, 128);
        }
        return r;
    };
    // Bounded: half a second, then the error word, and from there on short waits.
    unsigned long long patience = 500000000ull;
    auto wait = [&](unsigned long long *bar, uint32_t parity) {
        unsigned long long t0 = 0;
        for (uint32_t n = 0; !mbar_look(bar, parity); n++) {
            if ((n & 255u) != 255u) continue;
            unsigned long long t;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
            if (t0 == 0) t0 = t;
            if (t - t0 > patience) {
                atomicOr(a.err, ERR_FP4);
                patience = 10000ull;
                return;
            }
        }
    };

    if (warp == 0) {
        // ---- copies ----
        uint32_t it = 0;
        for (uint32_t t = blockIdx.x; t < all; t += gridDim.x) {
            const Tile tl = tile_of(t);
            const uint32_t n_rows = (uint32_t)max(tl.rows, 1);
            int idx[4];
            if (a.rows)
                for (int i = 0; i < 4; i++) {
                    const int32_t r = (int32_t)lane * 4 + i;
                    const int32_t x = r < tl.rows ? a.rows[tl.m0 + r] : 0;
                    idx[i] = (uint32_t)x < (uint32_t)a.x_rows ? x : 0;
                }
            const uint32_t n_box = a.rows ? (n_rows + 3u) / 4u : (n_rows + 31u) / 32u;
            const uint32_t a0 = tl.n0 >> 7, blocks = (a.w_rows + 127u) >> 7, atoms = min(C::ATOMS, blocks - a0);
            const uint32_t bytes = n_box * (a.rows ? 512u : 4096u) + C::B + atoms * C::WPS * 512u;
            const uint8_t *ws = a.w + tl.e * a.stride + a.w_off + (uint64_t)a0 * a.words * 512u;
            for (uint32_t k = 0; k < n_ks; k++, it++) {
                const uint32_t sl = it % C::NS;
                uint8_t *st = ring + sl * C::STAGE;
                if (it >= C::NS) wait(&s.empty[sl], (it / C::NS - 1u) & 1u);
                __syncwarp();
                if (lane == 0) {
                    mbar_expect_tx(&s.full[sl], bytes);
                    tma_load_3d(st + C::A, &maps.w, &s.full[sl], (int)(k * 128u), (int)tl.n0, (int)tl.e);
                    for (uint32_t i = 0; i < atoms; i++)
                        bulk_load(smem_u32(st + C::A + C::B + C::SA + i * C::WPS * 512u), ws + ((uint64_t)i * a.words + k * C::WPS) * 512u, C::WPS * 512u,
                                  &s.full[sl]);
                    if (!a.rows)
                        for (uint32_t i = 0; i < n_box; i++) tma_load_2d(st + i * 4096u, &maps.x, &s.full[sl], (int)(k * 128u), tl.m0 + (int)(i * 32u));
                }
                __syncwarp();
                if (a.rows && lane < n_box) tma_gather4(st + lane * 512u, &maps.xg, &s.full[sl], (int)(k * 128u), idx);
            }
        }
    } else if (warp == 1) {
        // ---- scales to tensor memory, MMAs ----
        if (elect_one()) {
            const uint32_t idesc0 = (1u << 7) | (1u << 10) | ((BN >> 3) << 17) | ((NVF ? 0u : 1u) << 23) | (1u << 27);
            const uint64_t d0 = smem_desc_sw128(smem_u32(ring));
            uint32_t it = 0, n = 0;
            for (uint32_t t = blockIdx.x; t < all; t += gridDim.x, n++) {
                const uint32_t acc = n & 1u, n0 = (t % n_tiles) * BN;
                if (n >= 2u) wait(&s.acc_empty[acc], (n / 2u - 1u) & 1u);
                tc_fence_after();
                for (uint32_t k = 0; k < n_ks; k++, it++) {
                    const uint32_t sl = it % C::NS, at = sl * C::STAGE;
                    wait(&s.full[sl], (it / C::NS) & 1u);
                    tc_fence_after();
                    const uint32_t sf = tmem + C::SF_AT + (it & 1u) * C::SF_COLS, sfb = sf + C::WPS * 4u;
                    const uint32_t sa = smem_u32(ring) + at + C::A + C::B;
#pragma unroll
                    for (uint32_t w = 0; w < C::WPS; w++) scales_to_tmem(sf + w * 4u, sa + w * 512u);
#pragma unroll
                    for (uint32_t i = 0; i < C::ATOMS; i++)
#pragma unroll
                        for (uint32_t w = 0; w < C::WPS; w++)
                            scales_to_tmem(sfb + (w * C::ATOMS + i) * 4u, sa + C::SA + (i * C::WPS + w) * 512u);
                    const uint32_t left = a.cols - k * KSTAGE, n_mma = left >= KSTAGE ? 4u : (left + 63u) / 64u;
                    const uint64_t da = d0 + (at >> 4), db = da + (C::A >> 4);
                    for (uint32_t j = 0; j < n_mma; j++) {
                        const uint32_t w = NVF ? j : j >> 1, id = NVF ? 0u : (j & 1u) * 2u;
                        mma_fp4<NVF>(tmem + acc * BN, da + j * 2u, db + j * 2u, idesc0 | (id << 4) | (id << 29), sf + w * 4u,
                                     sfb + w * C::ATOMS * 4u + ((n0 & 127u) >> 5), (k | j) ? 1u : 0u);
                    }
                    mma_commit(&s.empty[sl]);
                }
                mma_commit(&s.acc_full[acc]);
            }
        }
    } else if (warp == 2) {
        // ---- the scales of x: lane l brings rows l, l + 32, l + 64, l + 96; a stage is handed on when those of two later ones
        // are under way ----
        constexpr uint32_t LAG = 2u;
        uint32_t it = 0;
        auto hand_on = [&](uint32_t i) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.full[i % C::NS]);
        };
        for (uint32_t t = blockIdx.x; t < all; t += gridDim.x) {
            const Tile tl = tile_of(t);
            const uint8_t *src[4];
            uint32_t size[4];
            for (int j = 0; j < 4; j++) {
                const int32_t r = (int32_t)lane + 32 * j;
                uint32_t x = 0;
                bool ok = r < tl.rows;
                if (ok) {
                    x = (uint32_t)(a.rows ? a.rows[tl.m0 + r] : tl.m0 + r);
                    ok = x < (uint32_t)a.x_rows;
                }
                src[j] = a.xs + (ok ? (uint64_t)x : 0u) * 4u;
                size[j] = ok ? 4u : 0u;
            }
            for (uint32_t k = 0; k < n_ks; k++, it++) {
                const uint32_t sl = it % C::NS;
                if (it >= C::NS) wait(&s.empty[sl], (it / C::NS - 1u) & 1u);
                const uint32_t dst = smem_u32(ring) + sl * C::STAGE + C::A + C::B + lane * 16u;
#pragma unroll
                for (uint32_t w = 0; w < C::WPS; w++)
#pragma unroll
                    for (uint32_t j = 0; j < 4u; j++)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + w * 512u + j * 4u),
                                     "l"(src[j] + (uint64_t)(k * C::WPS + w) * a.x_pitch * 4u), "r"(size[j])
                                     : "memory");
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (it >= LAG) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
                    hand_on(it - LAG);
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        for (uint32_t i = it > LAG ? it - LAG : 0u; i < it; i++) hand_on(i);
    } else if (warp >= 4u) {
        // ---- finished accumulators ----
        const uint32_t q = warp & 3u;
        uint8_t *const buf = s.out[q];
        const bool vec = ((uintptr_t)a.dst & 15u) == 0 && (a.ld & 3u) == 0;
        uint32_t n = 0;
        for (uint32_t t = blockIdx.x; t < all; t += gridDim.x, n++) {
            const Tile tl = tile_of(t);
            const uint32_t acc = n & 1u;
            const float f0 = a.each ? a.scale * a.each[tl.e] : a.scale;
            const int32_t mine = tl.rows - (int32_t)(32u * q);      // rows of this warp
            bool there = (int32_t)lane < mine;
            if (there && a.rows) there = (uint32_t)a.rows[tl.m0 + (int32_t)(32u * q + lane)] < (uint32_t)a.x_rows;
            wait(&s.acc_full[acc], (n / 2u) & 1u);
            tc_fence_after();
            float *const base = a.dst + (uint64_t)(tl.m0 + (int32_t)(32u * q)) * a.ld;
            const uint32_t cols = min(BN, a.w_rows - tl.n0);
            if (mine > 0)
                for (uint32_t c0 = 0; c0 < cols; c0 += 32u) {
                    float v[32];
                    tmem_ld32(tmem + ((32u * q) << 16) + acc * BN + c0, v);
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++)
                        *reinterpret_cast<float4 *>(buf + lane * 128u + ((i ^ (lane & 7u)) << 4)) =
                            there ? make_float4(v[4 * i] * f0, v[4 * i + 1] * f0, v[4 * i + 2] * f0, v[4 * i + 3] * f0) : make_float4(0.f, 0.f, 0.f, 0.f);
                    __syncwarp();
                    const uint32_t col = tl.n0 + c0;
                    if (vec && col + 32u <= a.w_rows) {
#pragma unroll
                        for (uint32_t i = 0; i < 8u; i++) {
                            const uint32_t r = i * 4u + (lane >> 3), c = lane & 7u;
                            const float4 o = *reinterpret_cast<const float4 *>(buf + r * 128u + ((c ^ (r & 7u)) << 4));
                            if ((int32_t)r < mine) *reinterpret_cast<float4 *>(base + (uint64_t)r * a.ld + col + 4u * c) = o;
                        }
                    } else {
                        for (uint32_t r = 0; r < 32u && (int32_t)r < mine; r++) {
                            const float o = *reinterpret_cast<const float *>(buf + r * 128u + (((lane >> 2) ^ (r & 7u)) << 4) + (lane & 3u) * 4u);
                            if (col + lane < a.w_rows) base[(uint64_t)r * a.ld + col + lane] = o;
                        }
                    }
                    __syncwarp();
                }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.acc_empty[acc]);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <bool NVF, uint32_t BN> bool tc_launch(const MArgs &a, uint64_t m_tiles) {
    using C = Cfg<NVF, BN>;
    TcMaps maps;
    auto encode = [](CUtensorMap *m, uint32_t rank, const void *p, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
        const cuuint32_t es[3] = {1, 1, 1};
        return mmqtc::g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, (void *)p, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    const cuuint64_t xd[2] = {a.cols / 2u, a.x_rows}, xs[1] = {a.cols / 2u};
    const cuuint64_t wd[3] = {a.cols / 2u, a.w_rows, a.n_expert}, ws[2] = {a.cols / 2u, a.stride ? a.stride : code_bytes(a.w_rows, a.cols)};
    const cuuint32_t xb[2] = {128, 32}, gb[2] = {128, 1}, wb[3] = {128, BN, 1};
    if (!encode(&maps.x, 2, a.x, xd, xs, xb) || !encode(&maps.xg, 2, a.x, xd, xs, gb) || !encode(&maps.w, 3, a.w, wd, ws, wb)) return false;
    const uint64_t tiles = m_tiles * ((a.w_rows + BN - 1u) / BN);
    q4b_launch(tc_k<NVF, BN>, dim3((unsigned)(tiles < (uint64_t)g_q4b.n_sm ? tiles : (uint64_t)g_q4b.n_sm)), dim3(256), C::SMEM, g_q4b.stream, a, maps);
    g_q4b_launches++;
    return q4b_launch_ok("fp4 product");
}

static bool g_tc_ready = false;
template <bool NVF, uint32_t BN> bool tc_attr() {
    return cudaFuncSetAttribute(tc_k<NVF, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<NVF, BN>::SMEM) == cudaSuccess;
}
bool tc_warm() {
    if (g_tc_ready) return true;
    if (!mmqtc::warm()) return false;
    g_tc_ready = tc_attr<false, 64>() && tc_attr<true, 64>() && tc_attr<false, 128>() && tc_attr<true, 128>() && tc_attr<false, 192>() && tc_attr<true, 192>();
    return g_tc_ready;
}

// Tiles of 64, 128 or 192 rows of W: the one with which the busiest CTA has least to do.
bool tc_product(bool nv, const MArgs &a) {
    const uint64_t m_tiles = a.bounds ? (a.total < a.n_expert ? a.total : a.n_expert) + a.total / 128u : (a.total + 127u) / 128u;
    if (!g_tc_ready || m_tiles * ((a.w_rows + 63u) / 64u) > 0x7fffffffull) return false;
    uint64_t best = ~0ull;
    uint32_t bn = 128;
    for (uint32_t c = 192u; c >= 64u; c -= 64u) {
        const uint64_t tiles = m_tiles * ((a.w_rows + c - 1u) / c), cost = (tiles + g_q4b.n_sm - 1u) / g_q4b.n_sm * (c + 32u);
        if (cost < best) best = cost, bn = c;
    }
    if (bn == 64u) return nv ? tc_launch<true, 64>(a, m_tiles) : tc_launch<false, 64>(a, m_tiles);
    if (bn == 128u) return nv ? tc_launch<true, 128>(a, m_tiles) : tc_launch<false, 128>(a, m_tiles);
    return nv ? tc_launch<true, 192>(a, m_tiles) : tc_launch<false, 192>(a, m_tiles);
}

}  // namespace fp4

bool q4b_fp4_warm() { return fp4::tc_warm(); }
