// The product of MXFP4 and NVFP4 matrices on the tensor cores.  Part of the single translation unit q4cuda.cu.
//
// tcgen05.mma.kind::mxf4 / mxf4nvf4 multiplies the codes and their scales as they are stored: 128 rows of x times BN rows of W,
// 64 values of k an instruction, fp32 sums in tensor memory.  The kernel is persistent; a CTA takes tiles of
// 128 x BN of the result (an expert's rows begin at any row; its last tile has fewer), and its warps have a task each:
//   warp 0      copies of W: codes (TMA, 128-byte swizzle: 256 values of a row a stage), scales (bulk)
//   warps 2, 3  x: codes by TMA, or where rows are gathered by cp.async (tile::gather4 took 50 cycles for four of them: 466 us where
//               this takes 205); scales word by word (cp.async)
//   warp 1      sees that a stage is there
//   warp 12     brings a stage's scales to tensor memory (tcgen05.cp) and issues its MMAs
//   warps 4-11  read a finished accumulator, apply the factor and store, while the MMAs fill the other one: 32 x 32 at a time
//               through shared memory (TMA), of fewer rows from the registers
// What bounds it: with few rows an expert the reads of W (64 tokens, top-10 of 512 experts, 1024 x 2048, NVFP4: 71 to 73 us, 5.9 TB/s,
// in a short run of calls; 80 over 0.3 s, which the power cap slows down); with many the loads of a stage, 35 to 45 KB that arrive
// at some 45 bytes a cycle and SM, beside the stores of fp32 results (8192 x 4096 x 2048, NVFP4: 47 to 48 us in a short run, 2.9
// PFLOP/s, tensor pipe 39 %; 55 over 0.3 s), hence tiles as large as two accumulators and the scales leave room for.
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

constexpr uint32_t ERR_FP4 = 1u << 20;
constexpr uint32_t KSTAGE = 256u;
constexpr uint32_t MAX_EXPERTS = 1024u, MAX_MAP = 512u;
constexpr uint32_t THREADS = 416u;

struct TcSmem {
    unsigned long long full[8], ready[8], empty[8], acc_full[2], acc_empty[2];
    uint32_t tmem, warp_sum[8];
    uint32_t first[MAX_EXPERTS + 1];       // tiles of rows before every expert
    int32_t row[MAX_EXPERTS + 1];          // its first row
    uint16_t of[MAX_MAP];                  // the expert of a tile of rows
};
constexpr uint32_t OUT = 8u * 4096u;       // in front of it: the epilogue warps' 32 x 32 blocks
template <bool NVF, uint32_t BN, bool PAIR> struct Cfg {
    static constexpr uint32_t UM = PAIR ? 256u : 128u;             // rows of a tile
    static constexpr uint32_t BH = PAIR ? BN / 2u : BN;            // rows of W that a CTA brings
    static constexpr uint32_t WPS = NVF ? 4u : 2u;                 // scale words of a row a stage
    static constexpr uint32_t ATOMS = BN > 128u ? 2u : 1u;         // 128-row blocks of W's scales under a tile
    static constexpr uint32_t A = 128u * 128u, B = BH * 128u, SA = WPS * 512u, SB = WPS * ATOMS * 512u;
    static constexpr uint32_t STAGE = A + B + SA + SB;
    static constexpr uint32_t FIXED = OUT + (uint32_t)((sizeof(TcSmem) + 1023u) & ~1023u);
    static constexpr uint32_t NS = (227u * 1024u - FIXED) / STAGE > 8u ? 8u : (227u * 1024u - FIXED) / STAGE;
    static constexpr uint32_t SMEM = FIXED + NS * STAGE;
    static constexpr uint32_t SF_COLS = WPS * 4u * (1u + ATOMS);   // tensor memory columns of a stage's scales
    static constexpr uint32_t SF_AT = 2u * BN;
    static_assert(SF_AT + 2u * SF_COLS <= 512u && NS >= 4u && STAGE % 1024u == 0u, "layout");
};
struct TcMaps {
    CUtensorMap x, x32, w, y;              // 128 and 32 rows of x; BH rows of an expert's W; 32 x 32 of the result
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
// 512 bytes (32 lanes x 4 columns, for all four lane quarters) from shared to tensor memory; PAIR: in both CTAs
template <bool PAIR> __device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint32_t smem) {
    // no swizzle; groups of 8 x 16 bytes 128 bytes apart
    const uint64_t d = (uint64_t)((smem >> 4) & 0x3fffu) | ((uint64_t)8u << 32) | (1ull << 46);
    if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}
template <bool NVF, bool PAIR>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
#define Q4B_FP4_MMA(group, kind)                                                                             \
    asm volatile(                                                                                            \
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                    \
        "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),   \
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)                                               \
        : "memory")
    if (NVF) {
        if (PAIR) Q4B_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
        else Q4B_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
    } else {
        if (PAIR) Q4B_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
        else Q4B_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
    }
#undef Q4B_FP4_MMA
}
// 32 columns of a lane's row, and the wait for them (in one statement, so that nothing is computed from them before)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *f) {
    uint32_t *v = reinterpret_cast<uint32_t *>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
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

template <bool NVF, uint32_t BN, bool PAIR> __global__ void __launch_bounds__(THREADS, 1) tc_k(const MArgs a, const __grid_constant__ TcMaps maps, bool vec) {
    using C = Cfg<NVF, BN, PAIR>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *const ring = smem_raw;                                 // stages: codes of x, codes of W, scales of x, scales of W
    TcSmem &s = *reinterpret_cast<TcSmem *>(smem_raw + C::NS * C::STAGE + OUT);
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t rank = PAIR ? blockIdx.x & 1u : 0u, unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, units = PAIR ? gridDim.x >> 1 : gridDim.x;
    if (tid == 0) {
        for (uint32_t i = 0; i < C::NS; i++) mbar_init(&s.full[i], (a.rows ? 1 : 2) + 64), mbar_init(&s.ready[i], PAIR ? 2 : 1), mbar_init(&s.empty[i], 1);
        for (uint32_t i = 0; i < 2u; i++) mbar_init(&s.acc_full[i], 1), mbar_init(&s.acc_empty[i], PAIR ? 16 : 8);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (!a.bounds && warp == 1u && elect_one()) {       // a dense product's first stages of W, into the L2, before the kernel ahead is waited for
        const uint32_t n = (a.w_rows + BN - 1u) / BN, stages = min((a.cols + KSTAGE - 1u) / KSTAGE, C::NS);
        for (uint32_t k = 0; k < stages; k++)
            asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(&maps.w), "r"((int)(k * 128u)),
                         "r"((int)(unit % n * BN + rank * C::BH)), "r"(0)
                         : "memory");
    }
    // Rows that a tile does not have are multiplied all the same: by zeros while no tile had them, which takes less power than by what
    // shared memory holds, and a card at its power limit lowers its clock (64 tokens, top-10 of 512 experts: 78.5 us instead of 82).
    for (uint32_t i = 0; i < C::NS; i++)
        for (uint32_t k = tid; k < C::A / 16u; k += THREADS) *reinterpret_cast<uint4 *>(ring + i * C::STAGE + k * 16u) = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    q4b_pdl_wait();
    if (warp == 0) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    // the rows of every expert in tiles, summed up
    uint32_t m_tiles;
    if (a.bounds) {
        auto clipped = [&](uint32_t e) { return min(max(a.bounds[min(e, a.n_expert)], 0), (int32_t)a.total); };
        uint32_t c[4], sum = 0;                 // four experts a thread: the first 256 threads have all of them
        int32_t r = clipped(tid * 4u);
        for (uint32_t i = 0; i < 4u; i++) {
            const uint32_t e = tid * 4u + i;
            const int32_t next = clipped(e + 1u);
            if (e <= a.n_expert) s.row[e] = r;
            c[i] = (uint32_t)(max(next - r, 0) + (int32_t)C::UM - 1) / C::UM;
            sum += c[i];
            r = next;
        }
        if (tid == 255u) s.row[MAX_EXPERTS] = r;
        uint32_t inc = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += t;
        }
        if (lane == 31u && warp < 8u) s.warp_sum[warp] = inc;
        __syncthreads();
        uint32_t at = inc - sum;
        m_tiles = 0;
        for (uint32_t w = 0; w < 8u; w++) {
            if (w < warp) at += s.warp_sum[w];
            m_tiles += s.warp_sum[w];
        }
        for (uint32_t i = 0; i < 4u; i++) {
            const uint32_t e = tid * 4u + i;
            if (e <= a.n_expert) s.first[e] = at;
            for (uint32_t k = at; k < at + c[i] && k < MAX_MAP; k++) s.of[k] = (uint16_t)e;
            at += c[i];
        }
        if (tid == 255u) s.first[MAX_EXPERTS] = at;
    } else {
        m_tiles = (uint32_t)((a.total + C::UM - 1u) / C::UM);
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) mmqtc::cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    const uint32_t n_tiles = (a.w_rows + BN - 1u) / BN, n_ks = (a.cols + KSTAGE - 1u) / KSTAGE, all = m_tiles * n_tiles;
    auto tile_of = [&](uint32_t t) {
        Tile r;
        const uint32_t m = t / n_tiles;
        r.n0 = (t - m * n_tiles) * BN;
        r.e = 0;
        if (a.bounds) {
            if (m < MAX_MAP) {
                r.e = s.of[m];
            } else {             // the last expert whose first tile is not behind m: one that has rows
                uint32_t lo = 0, hi = a.n_expert;
                while (hi - lo > 1u) {
                    const uint32_t k = (lo + hi) >> 1;
                    if (s.first[k] <= m) lo = k; else hi = k;
                }
                r.e = lo;
            }
            r.m0 = s.row[r.e] + (int32_t)((m - s.first[r.e]) * C::UM);
            r.rows = s.row[r.e + 1u] - r.m0;
        } else {
            r.m0 = (int32_t)(m * C::UM);
            r.rows = (int32_t)a.total - r.m0;
        }
        // this CTA's 128 of them
        r.m0 += (int32_t)(rank * 128u);
        r.rows = max(min(r.rows - (int32_t)(rank * 128u), 128), 0);
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
        // ---- copies of W ----
        if (elect_one()) {
            uint32_t it = 0;
            for (uint32_t t = unit; t < all; t += units) {
                const Tile tl = tile_of(t);
                const uint32_t a0 = tl.n0 >> 7, atoms = min(C::ATOMS, ((a.w_rows + 127u) >> 7) - a0);
                const uint8_t *ws = a.w + tl.e * a.stride + a.w_off + (uint64_t)a0 * a.words * 512u;
                for (uint32_t k = 0; k < n_ks; k++, it++, ws += C::WPS * 512u) {
                    const uint32_t sl = it % C::NS;
                    uint8_t *st = ring + sl * C::STAGE;
                    if (it >= C::NS) wait(&s.empty[sl], (it / C::NS - 1u) & 1u);
                    mbar_expect_tx(&s.full[sl], C::B + atoms * C::WPS * 512u);
                    tma_load_3d(st + C::A, &maps.w, &s.full[sl], (int)(k * 128u), (int)(tl.n0 + rank * C::BH), (int)tl.e);
                    for (uint32_t i = 0; i < atoms; i++)
                        bulk_load(smem_u32(st + C::A + C::B + C::SA + i * C::WPS * 512u), ws + (uint64_t)i * a.words * 512u, C::WPS * 512u, &s.full[sl]);
                }
            }
        }
    } else if (warp == 1) {
        // ---- a stage is there: its copies and the scales' are seen by this thread, made visible to the tensor cores and reported
        // to the warp that issues the MMAs (of a pair, in the first CTA), which so waits for one barrier a stage and needs no fence ----
        if (elect_one()) {
            uint32_t it = 0;
            for (uint32_t t = unit; t < all; t += units)
                for (uint32_t k = 0; k < n_ks; k++, it++) {
                    wait(&s.full[it % C::NS], (it / C::NS) & 1u);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    tc_fence_after();
                    tc_fence_before();
                    if (PAIR) mmqtc::mbar_arrive_cluster(mmqtc::leader_addr(&s.ready[it % C::NS]));
                    else mbar_arrive(&s.ready[it % C::NS]);
                }
        }
    } else if (warp < 4u) {
        // ---- x: scales of 64 rows a warp, word by word to their places; codes.  A lane arrives when its copies have landed ----
        auto copies = [&](auto gathered) {
            constexpr bool G = decltype(gathered)::value;
            const uint32_t half = (warp & 1u) * 64u;
            uint32_t it = 0;
            for (uint32_t t = unit; t < all; t += units) {
                const Tile tl = tile_of(t);
                const int32_t mine = tl.rows - (int32_t)half;          // rows of this warp; what is behind them may hold anything
                // lane l: scales of rows l and l + 32, sixteen bytes l % 8 of the codes of rows 4 i + l / 8
                const uint8_t *src[2];
                uint32_t size[2], code_row[16];
#pragma unroll
                for (uint32_t j = 0; j < 2u; j++) {
                    const int32_t r = (int32_t)(lane + 32u * j);
                    uint32_t x = 0;
                    bool ok = r < mine;
                    if (ok) {
                        x = (uint32_t)(tl.m0 + (int32_t)half + r);
                        if (G) x = (uint32_t)a.rows[x];
                        ok = x < (uint32_t)a.x_rows;
                    }
                    src[j] = a.xs + (ok ? (uint64_t)x : 0u) * 4u;
                    size[j] = ok ? 4u : 0u;
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++)
                        if (G) code_row[j * 8u + i] = __shfl_sync(0xffffffffu, ok ? x : 0xffffffffu, i * 4u + (lane >> 3));
                }
                for (uint32_t k = 0; k < n_ks; k++, it++) {
                    const uint32_t sl = it % C::NS, st = smem_u32(ring) + sl * C::STAGE, dst = st + C::A + C::B + lane * 16u + (half >> 3);
                    if (it >= C::NS) wait(&s.empty[sl], (it / C::NS - 1u) & 1u);
#pragma unroll
                    for (uint32_t w = 0; w < C::WPS; w++)
#pragma unroll
                        for (uint32_t j = 0; j < 2u; j++)
                            if ((int32_t)(32u * j) < mine)
                                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + w * 512u + j * 4u),
                                             "l"(src[j] + (uint64_t)(k * C::WPS + w) * a.x_pitch * 4u), "r"(size[j])
                                             : "memory");
                    if (G) {
                        const uint32_t c = k * 128u + (lane & 7u) * 16u;
                        const bool in = c < (a.cols >> 1);
#pragma unroll
                        for (uint32_t i = 0; i < 16u; i++) {
                            const uint32_t r = half + i * 4u + (lane >> 3);
                            const bool ok = in && code_row[i] != 0xffffffffu;
                            if ((int32_t)(4u * i) < mine)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(st + r * 128u + (((lane & 7u) ^ (r & 7u)) << 4)),
                                             "l"(a.x + (ok ? (uint64_t)code_row[i] * (a.cols >> 1) + c : 0u)), "r"(ok ? 16u : 0u)
                                             : "memory");
                        }
                    } else if (warp == 3u && elect_one()) {
                        uint8_t *const to = ring + sl * C::STAGE;
                        const uint32_t boxes = tl.rows > 96 ? 4u : ((uint32_t)tl.rows + 31u) / 32u;
                        mbar_expect_tx(&s.full[sl], boxes * 4096u);
                        if (boxes == 4u) tma_load_2d(to, &maps.x, &s.full[sl], (int)(k * 128u), tl.m0);
                        else
                            for (uint32_t i = 0; i < boxes; i++) tma_load_2d(to + i * 4096u, &maps.x32, &s.full[sl], (int)(k * 128u), tl.m0 + (int)(i * 32u));
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&s.full[sl])) : "memory");
                }
            }
        };
        if (a.rows) copies(std::true_type());
        else copies(std::false_type());
    } else if (warp == 12u) {
        // ---- scales to tensor memory, MMAs ----
        if (rank == 0 && elect_one()) {
            const uint32_t idesc0 = (1u << 7) | (1u << 10) | ((BN >> 3) << 17) | ((NVF ? 0u : 1u) << 23) | ((PAIR ? 2u : 1u) << 27);
            const uint64_t d0 = smem_desc_sw128(smem_u32(ring));
            uint32_t n = 0, sl = 0, par = 0, odd = 0;       // tiles; the stage's slot, its parity, its half of the scales' columns
            for (uint32_t t = unit; t < all; t += units, n++) {
                const uint32_t acc = n & 1u, n0 = (t % n_tiles) * BN;
                if (n >= 2u) wait(&s.acc_empty[acc], (n / 2u - 1u) & 1u);
                tc_fence_after();
                for (uint32_t k = 0; k < n_ks; k++) {
                    const uint32_t at = sl * C::STAGE;
                    wait(&s.ready[sl], par);
                    tc_fence_after();
                    const uint32_t sf = tmem + C::SF_AT + odd * C::SF_COLS, sfb = sf + C::WPS * 4u;
                    const uint32_t sa = smem_u32(ring) + at + C::A + C::B;
#pragma unroll
                    for (uint32_t w = 0; w < C::WPS; w++) scales_to_tmem<PAIR>(sf + w * 4u, sa + w * 512u);
#pragma unroll
                    for (uint32_t i = 0; i < C::ATOMS; i++)
#pragma unroll
                        for (uint32_t w = 0; w < C::WPS; w++)
                            scales_to_tmem<PAIR>(sfb + (w * C::ATOMS + i) * 4u, sa + C::SA + (i * C::WPS + w) * 512u);
                    const uint32_t left = a.cols - k * KSTAGE, n_mma = left >= KSTAGE ? 4u : (left + 63u) / 64u;
                    const uint64_t da = d0 + (at >> 4), db = da + (C::A >> 4);
#pragma unroll
                    for (uint32_t j = 0; j < 4u; j++) {
                        if (j >= n_mma) break;
                        const uint32_t w = NVF ? j : j >> 1, id = NVF ? 0u : (j & 1u) * 2u;
                        mma_fp4<NVF, PAIR>(tmem + acc * BN, da + j * 2u, db + j * 2u, idesc0 | (id << 4) | (id << 29), sf + w * 4u,
                                           sfb + w * C::ATOMS * 4u + ((n0 & 127u) >> 5), (k | j) ? 1u : 0u);
                    }
                    if (PAIR) mmqtc::mma_commit2(&s.empty[sl]);
                    else mma_commit(&s.empty[sl]);
                    odd ^= 1u;
                    if (++sl == C::NS) sl = 0, par ^= 1u;
                }
                if (PAIR) mmqtc::mma_commit2(&s.acc_full[acc]);
                else mma_commit(&s.acc_full[acc]);
            }
        }
    } else {
        // ---- finished accumulators: two warps to a quarter of the rows, every second 32 columns each ----
        const uint32_t q = warp & 3u, set = (warp - 4u) >> 2;
        uint8_t *const buf = smem_raw + C::NS * C::STAGE + (warp - 4u) * 4096u;
        const uint32_t free0 = PAIR ? mmqtc::leader_addr(&s.acc_empty[0]) : 0u;
        bool busy = false;           // a copy out of the buffer may be under way
        uint32_t n = 0;
        for (uint32_t t = unit; t < all; t += units, n++) {
            const Tile tl = tile_of(t);
            const uint32_t acc = n & 1u;
            const float f0 = a.each ? a.scale * a.each[tl.e] : a.scale;
            const int32_t row0 = tl.m0 + (int32_t)(32u * q), mine = tl.rows - (int32_t)(32u * q);      // rows of this warp
            bool there = (int32_t)lane < mine;
            if (there && a.rows) there = (uint32_t)a.rows[row0 + (int32_t)lane] < (uint32_t)a.x_rows;
            const float f = there ? f0 : 0.f;
            float *const base = a.dst + (uint64_t)row0 * a.ld;
            const uint32_t cols = min(BN, a.w_rows - tl.n0);
            wait(&s.acc_full[acc], (n / 2u) & 1u);
            tc_fence_after();
            for (uint32_t c0 = 32u * set; mine > 0 && c0 < cols; c0 += 64u) {
                const uint32_t col = tl.n0 + c0;
                float v[32];
                tmem_ld32(tmem + ((32u * q) << 16) + acc * BN + c0, v);
#pragma unroll
                for (uint32_t i = 0; i < 32u; i++) v[i] = there ? v[i] * f : 0.f;
                if (mine < 32 && vec && col + 32u <= a.w_rows) {       // fewer rows: each from its lane, in whole sectors
                    if ((int32_t)lane < mine) {
                        float *o = base + (uint64_t)lane * a.ld + col;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++)
                            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o + 8 * i), "f"(v[8 * i]), "f"(v[8 * i + 1]),
                                         "f"(v[8 * i + 2]), "f"(v[8 * i + 3]), "f"(v[8 * i + 4]), "f"(v[8 * i + 5]), "f"(v[8 * i + 6]), "f"(v[8 * i + 7])
                                         : "memory");
                    }
                    continue;
                }
                if (busy) {
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
                    busy = false;
                }
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++)
                    *reinterpret_cast<float4 *>(buf + lane * 128u + ((i ^ (lane & 7u)) << 4)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                if (mine >= 32 && vec && (col + 32u <= a.w_rows || (a.w_rows & 3u) == 0)) {     // (a copy is cut at 16 bytes)
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&maps.y), "r"((int)col), "r"(row0),
                                     "r"(smem_u32(buf))
                                     : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                    busy = true;
                    continue;
                }
                __syncwarp();
                const bool in = col + lane < a.w_rows;
#pragma unroll 8
                for (uint32_t r = 0; r < 32u; r++) {
                    const float o = *reinterpret_cast<const float *>(buf + r * 128u + (((lane >> 2) ^ (r & 7u)) << 4) + (lane & 3u) * 4u);
                    if (in && (int32_t)r < mine) base[(uint64_t)r * a.ld + col + lane] = o;
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) mmqtc::mbar_arrive_cluster_relaxed(free0 + 8u * acc);
                else mbar_arrive(&s.acc_empty[acc]);
            }
        }
        if (busy && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (PAIR) mmqtc::cluster_sync();
    tc_fence_after();
    if (warp == 0) {
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <bool NVF, uint32_t BN, bool PAIR> bool tc_launch(const MArgs &a, uint64_t m_tiles) {
    using C = Cfg<NVF, BN, PAIR>;
    TcMaps maps;
    auto encode = [](CUtensorMap *m, CUtensorMapDataType type, uint32_t rank, const void *p, const cuuint64_t *dims, const cuuint64_t *strides,
                     const cuuint32_t *box) {
        const cuuint32_t es[3] = {1, 1, 1};
        return mmqtc::g_encode(m, type, rank, (void *)p, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    const cuuint64_t xd[2] = {a.cols / 2u, a.x_rows}, xs[1] = {a.cols / 2u};
    const cuuint64_t wd[3] = {a.cols / 2u, a.w_rows, a.n_expert}, ws[2] = {a.cols / 2u, a.n_expert > 1u ? a.stride : code_bytes(a.w_rows, a.cols)};
    const cuuint32_t xb[2] = {128, 128}, x32b[2] = {128, 32}, wb[3] = {128, C::BH, 1};
    const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    if (!encode(&maps.x, u8, 2, a.x, xd, xs, xb) || !encode(&maps.x32, u8, 2, a.x, xd, xs, x32b) || !encode(&maps.w, u8, 3, a.w, wd, ws, wb)) return false;
    const bool vec = aligned(a.dst, 32) && a.ld % 8u == 0 && a.ld * 4u < (1ull << 40);      // whole sectors of the result
    maps.y = maps.x;
    const cuuint64_t yd[2] = {a.w_rows, a.total}, ys[1] = {a.ld * 4u};
    const cuuint32_t yb[2] = {32, 32};
    if (vec && !encode(&maps.y, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, a.dst, yd, ys, yb)) return false;
    const uint64_t tiles = m_tiles * ((a.w_rows + BN - 1u) / BN), most = (uint64_t)g_q4b.n_sm / (PAIR ? 2u : 1u), units = tiles < most ? tiles : most;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * (PAIR ? 2u : 1u)));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = g_q4b.stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 2, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = PAIR ? 2 : 1;
    (void)cudaLaunchKernelEx(&cfg, tc_k<NVF, BN, PAIR>, a, maps, vec);
    g_q4b_launches++;
    g_ran[PAIR ? 2 : 1]++;
    return q4b_launch_ok("fp4 product");
}

template <uint32_t BN, bool PAIR> bool tc_attr() {
    return cudaFuncSetAttribute(tc_k<false, BN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<false, BN, PAIR>::SMEM) == cudaSuccess &&
           cudaFuncSetAttribute(tc_k<true, BN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<true, BN, PAIR>::SMEM) == cudaSuccess;
}
bool tc_warm() {
    if (g_tc_ready) return true;
    if (!mmqtc::warm()) return false;
    g_tc_ready = tc_attr<64, false>() && tc_attr<128, false>() && tc_attr<192, false>() && tc_attr<192, true>();
    if (!g_tc_ready) cudaGetLastError();       // the products stay on the CUDA cores; the next launch's check is its own
    return g_tc_ready;
}

template <uint32_t BN, bool PAIR> bool tc_go(bool nv, const MArgs &a, uint64_t m_tiles) {
    return nv ? tc_launch<true, BN, PAIR>(a, m_tiles) : tc_launch<false, BN, PAIR>(a, m_tiles);
}
// The tile of 64, 128 or 192 rows of W with which the busiest SM has least to do: its rows and 96 for a tile's beginning and end
// (short runs; of 64 / 128 / 192, us: 777 rows x 4099 x 2560 17 / 13.6 / 15.5; 64 tokens, top-10 of 512 experts, 1024 x 2048 127 / 75 / 73;
// one token of them 8.7 / 6.8 / 8.0; 8192 tokens 380 / 243 / 209).  Pairs of CTAs, which halve the reads of W, for dense products of
// four rounds of tiles and more: 8192 x 4096 x 2048 47.1 us, by single CTAs 52.0.  Of experts with fewer than 256 rows half a pair
// idles (the 8192 tokens above: 259 us).
bool tc_product(bool nv, const MArgs &a) {
    const uint64_t m_tiles = a.bounds ? (a.total < a.n_expert ? a.total : a.n_expert) + a.total / 128u : (a.total + 127u) / 128u;
    if (m_tiles * ((a.w_rows + 63u) / 64u) > 0x7fffffffull) return false;
    const uint64_t pairs = (a.total + 255u) / 256u;
    if (!a.bounds && pairs * ((a.w_rows + 191u) / 192u) >= 4u * (uint64_t)g_q4b.n_sm) return tc_go<192, true>(nv, a, pairs);
    uint64_t best = ~0ull;
    uint32_t bn = 192;
    for (uint32_t c = 192u; c >= 64u; c -= 64u) {
        const uint64_t tiles = m_tiles * ((a.w_rows + c - 1u) / c), cost = (tiles + g_q4b.n_sm - 1u) / g_q4b.n_sm * (c + 96u);
        if (cost < best) best = cost, bn = c;
    }
    return bn == 192u ? tc_go<192, false>(nv, a, m_tiles) : bn == 128u ? tc_go<128, false>(nv, a, m_tiles) : tc_go<64, false>(nv, a, m_tiles);
}

}  // namespace fp4

bool q4b_fp4_warm() { return fp4::tc_warm(); }
void q4b_fp4_shutdown() { fp4::g_tc_ready = false; }      // (the limits are a device's: the next init asks for its own)
