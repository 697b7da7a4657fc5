// Microscaled 4-bit floating point (MXFP4, NVFP4): quantisers, layouts and the product on the CUDA cores.
// Part of the single translation unit q4cuda.cu.
//
// A value is a sign and a magnitude out of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (E2M1) times its block's scale:
//   MXFP4  32 values share 2^(b - 127), one byte b (255 = NaN)
//   NVFP4  16 values share an e4m3 number without its sign, one byte (0x7f = NaN)
// A quantised [rows][cols] matrix begins with the codes, row after row, value 2 i in the low half of byte i.  Behind them (on the
// next 256-byte boundary) stand the scales as words of four bytes, the four blocks of a row that follow one another (128
// values in MXFP4, 64 in NVFP4), for cols rounded up to a multiple of 256 (zero bytes there):
//   rows     [word][row]: a product's tiles of activations begin at any row, or gather their rows
//   weights  [row / 128][word][row % 32][row / 32 % 4]: 512 bytes that go to tensor memory as they are
#include <atomic>
#include <type_traits>

namespace fp4 {

constexpr uint32_t MX = 39u, NV = 40u;      // ggml type ids
constexpr uint32_t ROWS = 0u, WEIGHTS = 1u;

__host__ __device__ constexpr uint32_t n_words(bool nv, uint32_t cols) { return (cols + 255u) / 256u * (nv ? 4u : 2u); }
__host__ __device__ inline uint64_t up256(uint64_t v) { return (v + 255u) & ~(uint64_t)255u; }
__host__ __device__ inline uint64_t code_bytes(uint64_t rows, uint32_t cols) { return up256(rows * (cols / 2u)); }
__host__ __device__ inline uint64_t row_pitch(uint64_t rows) { return (rows + 3u) & ~(uint64_t)3u; }   // words of a line of the rows order
inline uint64_t bytes(bool nv, uint32_t form, uint64_t rows, uint32_t cols) {
    return code_bytes(rows, cols) + up256((form == WEIGHTS ? (rows + 127u) / 128u * 128u : row_pitch(rows)) * n_words(nv, cols) * 4u);
}
// Byte offset, from the scales' beginning, of word w of a row.
template <bool WF> __device__ __forceinline__ uint64_t word_at(uint64_t row, uint32_t w, uint32_t words, uint64_t pitch) {
    if (WF) return ((row >> 7) * words + w) * 512u + ((uint32_t)row & 31u) * 16u + ((uint32_t)(row >> 5) & 3u) * 4u;
    return (w * pitch + row) * 4u;
}

// ---- arithmetic of the formats ----
// Two magnitudes' worth: the eight E2M1 magnitudes times two, as the bytes of two words.
constexpr uint32_t MAG_LO = 0x03020100u, MAG_HI = 0x0c080604u;

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(s));
    return r;
}
// Eight values to eight codes, v[0] in the lowest four bits.  To the nearest, ties to the even code, 6 for all beyond it.
__device__ __forceinline__ uint32_t encode8(const float *v) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
__device__ __forceinline__ float e4m3_value(uint32_t b) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)b));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}
__device__ __forceinline__ uint32_t e4m3_nearest(float v) {   // v >= 0; 448 for all beyond it
    uint16_t h;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(0.f), "f"(v));
    return h & 0xffu;
}
// 2^(b - 127); b = 0 is a subnormal fp32, 255 is no number
__device__ __forceinline__ float e8m0_value(uint32_t b) {
    return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7fc00000u : b << 23);
}
template <bool NVF> __device__ __forceinline__ float scale_value(uint32_t b) { return NVF ? e4m3_value(b) : e8m0_value(b); }

// The scale byte of a block whose largest magnitude is a.  MXFP4: the power of two that brings a into [4, 8); NVFP4: a sixth
// of a, rounded to e4m3.  The sixth is the fp32 product with fp32's 1/6, off by 1.5 * 2^-24 at most, as fp32 frameworks divide by a
// constant on a GPU: rows that one of them quantises get the same bytes.  A quotient would name another scale for one fp32 number a
// binade, 7.125 less a step times a power of two, whose sixth lies between two e4m3 numbers to within that rounding.
template <bool NVF> __device__ __forceinline__ uint32_t scale_byte(float a) {
    if (!(a <= 3.402823466e38f)) return NVF ? 0x7fu : 255u;
    if (NVF) return e4m3_nearest(a * (1.f / 6.f));
    const int e = (int)(__float_as_uint(a) >> 23) - 2;      // 127 + floor(log2 a) - 2 for a normal a, at most 252
    return (uint32_t)max(e, 0);
}
// What a block's values are multiplied with to become units of its scale: exact in MXFP4 (a power of two), rounded in NVFP4; 0 where
// the scale is 0 or NaN, whose codes are 0.
template <bool NVF> __device__ __forceinline__ float inverse(uint32_t sb) {
    if (NVF) return sb == 0u || sb == 0x7fu ? 0.f : __frcp_rn(e4m3_value(sb));
    return sb == 255u ? 0.f : __uint_as_float((254u - sb) << 23);
}
// Eight values of a block with that scale to codes.  MXFP4: the product with the inverse power of two is exact.  NVFP4: the quotient
// by the scale is rounded correctly (Markstein 1990: a product with the rounded inverse, corrected once by its exact remainder), and then
// falls on a border between two codes only where the exact one does: the scale has four bits and a border three, so a border's value
// is an fp32 number, and one that is not on it is a step of fp32 away at least.
template <bool NVF> __device__ __forceinline__ uint32_t codes8(const float *v, uint32_t sb) {
    const float inv = inverse<NVF>(sb);
    float t[8];
    if (NVF) {
        if (inv == 0.f) return 0u;
        const float s = e4m3_value(sb);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float q = v[i] * inv;
            t[i] = fmaf(fmaf(-q, s, v[i]), inv, q);
        }
    } else {
        if (inv == 0.f) return 0u;
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = v[i] * inv;
    }
    return encode8(t);
}
__device__ __forceinline__ float max_nan(float a, float b) {      // NaN where one of them is none
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max8(const float *v) {
    float a = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 8; i++) a = max_nan(a, fabsf(v[i]));
    return a;
}
// Largest of the lanes that hold a block (two with 16 values, four with 32), NaN if one is: as the bits of magnitudes,
// whose order is the numbers' and in which NaN is largest.
template <bool NVF> __device__ __forceinline__ float block_max(float a) {
    uint32_t u = __float_as_uint(a) & 0x7fffffffu;
    u = max(u, __shfl_xor_sync(0xffffffffu, u, 1));
    if (!NVF) u = max(u, __shfl_xor_sync(0xffffffffu, u, 2));
    return __uint_as_float(u);
}

// ---- quantisers ----
struct QArgs {
    const float *x;        // the rows, or gate | up rows
    uint64_t ld;
    float mul;
    uint64_t rows, pitch;
    uint32_t cols, words;
    uint8_t *codes, *scales;
};

template <bool VEC> __device__ __forceinline__ void load8(const float *p, float *v) {
    if (VEC) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = p[i];
    }
}

__device__ __forceinline__ double swiglu64(double g, double u, double mul) { return g / (1.0 + exp(-g)) * u * mul; }

// The scale and the codes of a block in 64 bits.
template <bool NVF> __device__ __noinline__ uint32_t exact8(const double *v, uint32_t &sb) {
    double a = 0.0;
    bool bad = false;
    for (int i = 0; i < 8; i++) a = fmax(a, fabs(v[i])), bad |= !isfinite((float)v[i]);
    if (bad) a = __longlong_as_double(0x7ff8000000000000ll);
    unsigned long long u = (unsigned long long)__double_as_longlong(a);
    u = max(u, __shfl_xor_sync(0xffffffffu, u, 1));
    if (!NVF) u = max(u, __shfl_xor_sync(0xffffffffu, u, 2));
    a = __longlong_as_double((long long)u);
    double unit;
    if (a != a) {
        sb = NVF ? 0x7fu : 255u;
        return 0u;
    }
    if (NVF) {
        // nearest e4m3 number: steps of 2^-9 below 2^-6, of an eighth of the binade above
        const double want = a / 6.0;
        const int e = want > 0.0 ? max(ilogb(want), -6) : -6;
        const double s = fmin(rint(ldexp(want, 3 - e)) * ldexp(1.0, e - 3), 448.0);
        sb = e4m3_nearest((float)s);       // s is one of its values
        unit = s;
        if (sb == 0u) return 0u;
    } else {
        const int e = a > 0.0 ? ilogb(a) - 2 : -127;
        sb = (uint32_t)(min(max(e, -127), 127) + 127);
        unit = ldexp(1.0, (int)sb - 127);
    }
    uint32_t c = 0;
    for (int i = 0; i < 8; i++) {
        const double t = fabs(v[i]) / unit;
        const uint32_t m = (t > 0.25) + (t >= 0.75) + (t > 1.25) + (t >= 1.75) + (t > 2.5) + (t >= 3.5) + (t > 5.0);
        c |= (m | (v[i] < 0.0 ? 8u : 0u)) << (4 * i);
    }
    return c;
}

// A warp takes 256 values of a row at a time, eight a lane: a block is two or four lanes.  The eight warps of a CTA take the same
// columns of eight rows that follow one another; U such pieces of a row are loaded before the first is quantised (short runs: two of
// 8192 x 2048 14.6 us, 5.3 TB/s; one 16.4, four 16.0; with SwiGLU 22528 x 512 two 19.4 to 20.0 us, 5.0 to 5.1 TB/s, one 20.3; two over
// 0.3 s 15.0 and 20.5).  Bound by those loads and, with SwiGLU, by issue slots.
template <bool NVF, bool WF, bool SWIGLU, bool VEC> __global__ void __launch_bounds__(256) quantize_k(const QArgs a) {
    constexpr int U = 2;
    q4b_pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint64_t row = (uint64_t)blockIdx.x * 8u + warp;
    if (row >= a.rows) return;
    const float *const src = a.x + row * a.ld;
    uint8_t *const codes = a.codes + row * (a.cols >> 1);
    auto store = [&](uint32_t c0, uint32_t q, uint32_t sb) {
        const uint32_t c = c0 + lane * 8u;
        const bool live = c < a.cols;       // cols is a multiple of 32: a block is whole or not there
        if (live) *reinterpret_cast<uint32_t *>(codes + (c >> 1)) = q;
        // four blocks' bytes to a word: 8 lanes (NVFP4) or 16
        uint32_t w = live ? sb << (8u * (NVF ? (lane >> 1) & 3u : (lane >> 2) & 3u)) : 0u;
        w |= __shfl_xor_sync(0xffffffffu, w, NVF ? 2 : 4);
        w |= __shfl_xor_sync(0xffffffffu, w, NVF ? 4 : 8);
        if ((lane & (NVF ? 7u : 15u)) == 0u)
            *reinterpret_cast<uint32_t *>(a.scales + word_at<WF>(row, (c0 >> (NVF ? 6 : 7)) + lane / (NVF ? 8u : 16u), a.words, a.pitch)) = w;
    };
    const uint32_t step = gridDim.y * 256u;
    const float low = fabsf(a.mul) > 0x1p50f ? INFINITY : 1e-20f;
    for (uint32_t c0 = blockIdx.y * 256u; c0 < a.cols; c0 += U * step) {
        float v[U][8], u[U][8];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const uint32_t c = c0 + k * step + lane * 8u;
#pragma unroll
            for (int i = 0; i < 8; i++) v[k][i] = 0.f, u[k][i] = 0.f;
            if (c < a.cols) load8<VEC>(src + c, v[k]);
            if (SWIGLU && c < a.cols) load8<VEC>(src + a.cols + c, u[k]);
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            if (k && c0 + k * step >= a.cols) break;
            if (!SWIGLU) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[k][i] *= a.mul;
                const uint32_t sb = scale_byte<NVF>(block_max<NVF>(max8(v[k])));
                store(c0 + k * step, codes8<NVF>(v[k], sb), sb);
                continue;
            }
            // fp32 is off by at most 2 steps of 2^-23 for the exponential, half a one for the sum, 2 for the quotient (its divisor is
            // below 2^126), half a one each for two products and for the unit's, 1 for its inverse: below 2^-20.  Where that leaves
            // the scale or a code in doubt, or fp32's range is left, the warp computes in 64 bits.  A product g u or a quotient that has
            // lost bits (below 2^-126) is below 2^-76 after a mul of up to 2^50, and then a zero in a block whose largest is 1e-20 or more
            // (a code's lowest border is a 32nd of it at least); a block with less is in doubt, unless a factor of each of its products is 0.
            constexpr float LO = 1.f - 0x1p-20f, HI = 1.f + 0x1p-20f;
            float t[8];
            bool doubt = false;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float g = v[k][i];
                t[i] = __fdividef(g * u[k][i], 1.f + expf(-g)) * a.mul;
                doubt |= g < -80.f;
            }
            const float top = block_max<NVF>(max8(t));
            uint32_t sb = scale_byte<NVF>(top * LO);
            doubt |= scale_byte<NVF>(top * HI) != sb || !(top <= 1e38f) || top < low;
            const float inv = inverse<NVF>(sb);
            float lo[8], hi[8];
#pragma unroll
            for (int i = 0; i < 8; i++) lo[i] = t[i] * (inv * LO), hi[i] = t[i] * (inv * HI);
            uint32_t q = encode8(lo);
            doubt |= q != encode8(hi) && inv != 0.f;
            if (inv == 0.f) q = 0u;
            if (__any_sync(0xffffffffu, doubt)) {
                bool zeros = top == 0.f;
                for (int i = 0; i < 8; i++) zeros &= v[k][i] == 0.f || u[k][i] == 0.f;
                if (__any_sync(0xffffffffu, doubt && !zeros)) {
                    double w[8];
                    for (int i = 0; i < 8; i++) w[i] = swiglu64(v[k][i], u[k][i], a.mul);
                    q = exact8<NVF>(w, sb);
                }
            }
            store(c0 + k * step, q, sb);
        }
    }
}

// A quantised matrix as the values that it stands for: a warp 256 values of a row at a time, eight a lane, which are a sector (VEC) of the
// result.  Bound by its writes.
template <bool NVF, bool WF, bool VEC> __global__ void __launch_bounds__(256) values_k(const uint8_t *codes, const uint8_t *scales, uint64_t rows, uint64_t pitch,
                                                                                      uint32_t cols, uint32_t words, float *out, uint64_t ld) {
    constexpr int U = 4;
    q4b_pdl_wait();
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t row = (uint64_t)blockIdx.x * 8u + (threadIdx.x >> 5);
    if (row >= rows) return;
    const uint32_t step = gridDim.y * 256u;
    for (uint32_t c0 = blockIdx.y * 256u + lane * 8u; c0 < cols; c0 += U * step) {
        uint32_t q[U], sb[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const uint32_t c = c0 + k * step, b = c >> (NVF ? 4 : 5);
            if (c >= cols) break;
            q[k] = *reinterpret_cast<const uint32_t *>(codes + row * (cols >> 1) + (c >> 1));
            sb[k] = scales[word_at<WF>(row, b >> 2, words, pitch) + (b & 3u)];
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            const uint32_t c = c0 + k * step;
            if (c >= cols) break;
            const float s = scale_value<NVF>(sb[k]) * 0.5f;
            const uint32_t m[2] = {prmt(MAG_LO, MAG_HI, q[k] & 0x7777u), prmt(MAG_LO, MAG_HI, (q[k] >> 16) & 0x7777u)};
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float f = (float)((m[i >> 2] >> (8 * (i & 3))) & 0xffu) * s;
                v[i] = (q[k] >> (4 * i)) & 8u ? -f : f;
            }
            float *o = out + row * ld + c;
            if (VEC)
                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
                             "f"(v[5]), "f"(v[6]), "f"(v[7])
                             : "memory");
            else
#pragma unroll
                for (int i = 0; i < 8; i++) o[i] = v[i];
        }
    }
}

// Matrices in the form of a checkpoint to the weights order: a thread takes 16 bytes of codes (32 values), and the one that has a
// word's first block its scales.  scales == NULL: ggml blocks of 17 bytes, the scale and then codes j (low half) and j + 16 (high half)
// in byte j.  The tensor cores' e4m3 scales have no sign: a negative one gives its sign to the block's codes, so that a value is the same
// to every reader of the buffer.
template <bool NVF> __global__ void __launch_bounds__(256) put_k(const uint8_t *codes, const uint8_t *scales, uint32_t rows, uint32_t cols, uint32_t words,
                                                                 uint8_t *w, uint64_t stride, uint64_t scale_off, bool vec) {
    q4b_pdl_wait();
    constexpr uint32_t PER = NVF ? 2u : 4u;          // pieces of 32 values to a word of scales
    const uint32_t pieces = words * PER, nb = cols / (NVF ? 16u : 32u);
    const uint64_t n = (uint64_t)rows * pieces, step = (uint64_t)gridDim.x * blockDim.x;
    const uint64_t r0 = (uint64_t)blockIdx.y * rows;
    uint8_t *const to = w + blockIdx.y * stride;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
        const uint32_t row = (uint32_t)(i / pieces), p = (uint32_t)(i - (uint64_t)row * pieces);
        const uint64_t r = r0 + row;
        if (p % PER == 0u) {
            uint32_t sw = 0;
            for (uint32_t j = 0; j < 4u; j++) {
                const uint32_t b = p / PER * 4u + j;
                if (b < nb) sw |= (uint32_t)(scales ? scales[r * nb + b] : codes[(r * nb + b) * 17u]) << (8u * j);
            }
            *reinterpret_cast<uint32_t *>(to + scale_off + word_at<true>(row, p / PER, words, 0)) = NVF ? sw & 0x7f7f7f7fu : sw;
        }
        if (p * 32u >= cols) continue;
        uint32_t q[4] = {0, 0, 0, 0};
        if (scales && vec) {
            const uint4 v = *reinterpret_cast<const uint4 *>(codes + r * (cols >> 1) + p * 16u);
            q[0] = v.x, q[1] = v.y, q[2] = v.z, q[3] = v.w;
        } else if (scales) {
            for (uint32_t k = 0; k < 16u; k++) q[k >> 2] |= (uint32_t)codes[r * (cols >> 1) + p * 16u + k] << (8u * (k & 3u));
        } else {
            const uint8_t *s = codes + (r * nb + p) * 17u + 1u;
            for (uint32_t k = 0; k < 8u; k++) {       // values 2 k, 2 k + 1 and 16 further
                const uint32_t a = s[2u * k], b = s[2u * k + 1u];
                q[k >> 2] |= ((a & 15u) | ((b & 15u) << 4)) << (8u * (k & 3u));
                q[2u + (k >> 2)] |= ((a >> 4) | (b & 0xf0u)) << (8u * (k & 3u));
            }
        }
        if (NVF) {           // (p's two blocks; each is there, cols being a multiple of 32)
            if (scales[r * nb + 2u * p] & 0x80u) q[0] ^= 0x88888888u, q[1] ^= 0x88888888u;
            if (scales[r * nb + 2u * p + 1u] & 0x80u) q[2] ^= 0x88888888u, q[3] ^= 0x88888888u;
        }
        *reinterpret_cast<uint4 *>(to + (uint64_t)row * (cols >> 1) + p * 16u) = make_uint4(q[0], q[1], q[2], q[3]);
    }
}

// ---- the product on the CUDA cores ----
struct MArgs {
    const uint8_t *w;                    // codes of the first matrix; its scales w_off bytes behind
    uint64_t w_off, stride;
    uint32_t w_rows, cols, words;
    const uint8_t *x, *xs;               // codes and scales of the activations
    uint64_t x_rows, x_pitch;
    const int32_t *rows, *bounds;        // row p of the result is row rows[p] (or p) of x; expert e has rows [bounds[e], bounds[e + 1])
    uint32_t n_expert;
    uint64_t total;
    float scale;
    const float *each;
    float *dst;
    uint64_t ld;
    uint32_t *err;
};

// sum_i c_i d_i of eight codes each, times four, added to pos - neg: with the signs of one side given to the other, the
// magnitudes of the positive products and those of the negative ones are each a byte permute of a code word (a selector with
// bit 3 set replicates the byte's sign bit, which is 0).
__device__ __forceinline__ void dot8(uint32_t w, uint32_t sign, uint32_t m0, uint32_t m1, int &pos, int &neg) {
    const uint32_t p = w ^ sign, n = p ^ 0x88888888u;
    pos = __dp4a((int)prmt(MAG_LO, MAG_HI, p), (int)m0, pos);
    pos = __dp4a((int)prmt(MAG_LO, MAG_HI, p >> 16), (int)m1, pos);
    neg = __dp4a((int)prmt(MAG_LO, MAG_HI, n), (int)m0, neg);
    neg = __dp4a((int)prmt(MAG_LO, MAG_HI, n >> 16), (int)m1, neg);
}
// A block's integer (four times the sum of code products) times its two scales
template <bool NVF> __device__ __forceinline__ float scaled(int d, uint32_t sw, uint32_t sx) {
    if (NVF) return (float)d * (e4m3_value(sw) * e4m3_value(sx) * 0.25f);    // eight bits: exact
    // 2^(sw + sx - 256) as two factors, each an fp32 number whatever the bytes
    const int e = max((int)(sw + sx) - 256, -252), h = e >> 1;
    const float f = (float)d * __uint_as_float((uint32_t)(h + 127) << 23) * __uint_as_float((uint32_t)(e - h + 127) << 23);
    return sw == 255u || sx == 255u ? __uint_as_float(0x7fc00000u) : f;
}

// One row of the result a CTA row (blockIdx.y), a warp four weight rows 32 apart (their scale words are 16 bytes).  A lane takes 32
// values at a time, whose activations it decodes once for the four rows.  Bound by the latency of the weights' reads: a CTA asks for
// its weights (into the L2) before it waits for the kernel ahead, which quantises the activations, and a lane has the loads of
// 2048 columns under way at a time.
template <bool NVF> __global__ void __launch_bounds__(256) few_k(const MArgs a) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t set = blockIdx.x * 8u + warp;                       // rows of tile set / 32, set % 32 + 32 j
    const uint32_t r0 = (set >> 5) * 128u + (set & 31u);
    if (!a.bounds && r0 < a.w_rows)
        for (uint32_t j = 0; j < 4u && r0 + 32u * j < a.w_rows; j++)
            for (uint32_t c = lane * 256u; c < a.cols; c += 8192u) q4b_l2_prefetch(a.w + (uint64_t)(r0 + 32u * j) * (a.cols >> 1) + (c >> 1));
    q4b_pdl_wait();
    if (r0 >= a.w_rows) return;
    for (uint64_t p = blockIdx.y; p < a.total; p += gridDim.y) {
        uint32_t e = 0;
        if (a.bounds) {      // the expert that has row p: the last whose first row is not behind it
            if ((int64_t)p < a.bounds[0] || (int64_t)p >= a.bounds[a.n_expert]) continue;
            uint32_t lo = 0, hi = a.n_expert;
            while (hi - lo > 1u) {
                const uint32_t m = (lo + hi) >> 1;
                if (a.bounds[m] <= (int64_t)p) lo = m; else hi = m;
            }
            e = lo;
        }
        const uint64_t xr = a.rows ? (uint64_t)(uint32_t)a.rows[p] : p;
        const bool there = xr < a.x_rows;       // a row that is not there gives zeros
        const uint8_t *w = a.w + e * a.stride;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t c0 = lane * 32u; c0 < a.cols; c0 += 2048u) {
            uint4 x[2], q[2][4], ws[2];
            uint32_t xs[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t c = c0 + 1024u * h, wd = c >> (NVF ? 6 : 7);
                x[h] = make_uint4(0, 0, 0, 0), xs[h] = 0;
                if (c >= a.cols) continue;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (r0 + 32u * j < a.w_rows) q[h][j] = *reinterpret_cast<const uint4 *>(w + (uint64_t)(r0 + 32u * j) * (a.cols >> 1) + (c >> 1));
                ws[h] = *reinterpret_cast<const uint4 *>(w + a.w_off + word_at<true>(r0, wd, a.words, 0));
                if (there) {
                    x[h] = *reinterpret_cast<const uint4 *>(a.x + xr * (a.cols >> 1) + (c >> 1));
                    xs[h] = *reinterpret_cast<const uint32_t *>(a.xs + word_at<false>(xr, wd, a.words, a.x_pitch));
                }
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t c = c0 + 1024u * h;
                if (c >= a.cols) break;
                const uint32_t sh = NVF ? (c >> 1) & 16u : (c >> 2) & 24u;       // the first of the lane's scales in its word
                const uint32_t xw[4] = {x[h].x, x[h].y, x[h].z, x[h].w}, wsw[4] = {ws[h].x, ws[h].y, ws[h].z, ws[h].w}, xsw = xs[h] >> sh;
                uint32_t m[8];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    m[2 * i] = prmt(MAG_LO, MAG_HI, xw[i] & 0x7777u), m[2 * i + 1] = prmt(MAG_LO, MAG_HI, (xw[i] >> 16) & 0x7777u);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (r0 + 32u * j >= a.w_rows) break;
                    const uint32_t qw[4] = {q[h][j].x, q[h][j].y, q[h][j].z, q[h][j].w}, s = wsw[j] >> sh;
                    int pos = 0, neg = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        dot8(qw[i], xw[i] & 0x88888888u, m[2 * i], m[2 * i + 1], pos, neg);
                        if (NVF && i == 1) {
                            acc[j] += scaled<true>(pos - neg, s & 0xffu, xsw & 0xffu);
                            pos = neg = 0;
                        }
                    }
                    acc[j] += scaled<NVF>(pos - neg, NVF ? (s >> 8) & 0xffu : s & 0xffu, NVF ? (xsw >> 8) & 0xffu : xsw & 0xffu);
                }
            }
        }
        const float f = a.each ? a.scale * a.each[e] : a.scale;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float y = q4b_warp_sum(acc[j]);
            const uint32_t r = r0 + 32u * j;
            if (lane == 0 && r < a.w_rows) a.dst[p * a.ld + r] = there ? y * f : 0.f;
        }
    }
}

// ---- host side ----
// The library's device for the duration of a call.
struct OnDevice {
    int was = -1;
    OnDevice() {
        int d;
        if (cudaGetDevice(&d) == cudaSuccess && d != g_q4b.device && cudaSetDevice(g_q4b.device) == cudaSuccess) was = d;
    }
    ~OnDevice() {
        if (was >= 0) cudaSetDevice(was);
    }
};
bool shape(uint32_t type, uint64_t rows, uint64_t cols) {
    return (type == MX || type == NV) && rows && rows <= 0x7fffffffull && cols && cols % 32u == 0 && cols <= 65536u;
}
bool aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1u)) == 0; }

template <bool SWIGLU> bool quantize(uint32_t type, uint32_t form, const float *x, uint64_t ld, float mul, uint64_t rows, uint64_t cols, void *q) {
    QArgs a;
    a.x = x;
    a.ld = ld;
    a.mul = mul;
    a.rows = rows;
    a.pitch = row_pitch(rows);
    a.cols = (uint32_t)cols;
    a.words = n_words(type == NV, a.cols);
    a.codes = (uint8_t *)q;
    a.scales = a.codes + code_bytes(rows, a.cols);
    OnDevice dev;
    // a row's pieces of 256 values to one warp while there are rows enough for all SMs
    const uint32_t groups = (uint32_t)((rows + 7u) / 8u), pieces = (a.cols + 255u) / 256u;
    const uint32_t want = (8u * (uint32_t)g_q4b.n_sm + groups - 1u) / groups;
    const dim3 grid(groups, pieces < want ? pieces : want);
    auto go = [&](auto k) { q4b_launch(k, grid, dim3(256), 0, g_q4b.stream, a); };
    const bool vec = aligned(x, 16) && ld % 4u == 0;
    auto pick = [&](auto nv, auto wf) {
        constexpr bool N = decltype(nv)::value, W = decltype(wf)::value;
        vec ? go(quantize_k<N, W, SWIGLU, true>) : go(quantize_k<N, W, SWIGLU, false>);
    };
    using yes = std::true_type;
    using no = std::false_type;
    using weights = std::bool_constant<!SWIGLU>;
    if (form == ROWS) type == NV ? pick(yes(), no()) : pick(no(), no());
    else type == NV ? pick(yes(), weights()) : pick(no(), weights());
    g_q4b_launches++;
    return q4b_launch_ok("fp4 quantize");
}

bool tc_product(bool nv, const MArgs &a);      // q4b_fp4_tc.cu
static bool g_tc_ready = false;
static std::atomic<uint64_t> g_ran[3];         // products enqueued: CUDA cores, tensor cores by single CTAs, by pairs

// Few rows on the CUDA cores while they are at most two CTAs an SM, counted as often as one has 2048 columns, else on the tensor cores.
// us with the quantiser ahead, MXFP4, the first line's weights from HBM, the others' from the L2 (CUDA cores / tensor cores):
//   4096 x 2048   1 row 5.9 / 6.1, 2 rows 6.1 / 6.1, 3 rows 8.7 / 6.2
//   1024 x 1024   1 row 3.8 / 5.0, 8 rows 4.4 / 5.2, 12 rows 6.1 / 5.2, 18 rows 6.8 / 5.3
//   512 x 2048    1 row 4.6 / 5.8, 18 rows 6.1 / 6.1, 19 rows 8.3 / 6.1
//   8192 x 128    1 row 4.3 / 4.4, 8 rows 19.3 / 4.6
//   128 x 4096    8 rows 7.3 / 7.7, 37 rows 8.6 / 8.0
//   256 x 256     32 rows 4.4 / 4.5, 128 rows 11.0 / 5.3
//   64 x 128      32 rows 3.8 / 4.4, 128 rows 5.7 / 5.1, 1184 rows 31.6 / 5.3
// The two add a row up in different orders: its last bits change with the rows beside it where their number crosses the line.
bool product(uint32_t type, MArgs &a) {
    OnDevice dev;
    const uint64_t ctas = a.total * ((a.w_rows + 127u) / 128u * 4u);
    if (g_tc_ready && ctas * (a.cols < 2048u ? 2048u : a.cols) > 2u * (uint64_t)g_q4b.n_sm * 2048u) return tc_product(type == NV, a);
    const dim3 grid((a.w_rows + 127u) / 128u * 4u, (unsigned)(a.total < 65535u ? a.total : 65535u));
    if (type == NV) q4b_launch(few_k<true>, grid, dim3(256), 0, g_q4b.stream, a);
    else q4b_launch(few_k<false>, grid, dim3(256), 0, g_q4b.stream, a);
    g_q4b_launches++;
    g_ran[0]++;
    return q4b_launch_ok("fp4 product");
}

}  // namespace fp4

extern "C" uint64_t q4_cuda_fp4_bytes(uint32_t type, uint32_t form, uint64_t rows, uint64_t cols) {
    return fp4::shape(type, rows, cols) && form <= fp4::WEIGHTS ? fp4::bytes(type == fp4::NV, form, rows, (uint32_t)cols) : 0u;
}

extern "C" bool q4_cuda_fp4_put(uint32_t type, const uint8_t *d_codes, const uint8_t *d_scales, uint64_t rows, uint64_t cols, uint64_t n_mat,
                                void *d_w, uint64_t stride) {
    using namespace fp4;
    if (!g_q4b.ok || !shape(type, rows, cols) || !d_codes || !d_w || !n_mat || n_mat > 65535u || !aligned(d_w, 16) || stride % 16u ||
        (n_mat > 1u && stride < bytes(type == NV, WEIGHTS, rows, (uint32_t)cols)) || (type == NV && !d_scales))
        return false;
    OnDevice dev;
    const uint32_t words = n_words(type == NV, (uint32_t)cols);
    const uint64_t n = rows * words * (type == NV ? 2u : 4u), want = (n + 255u) / 256u, most = ((uint64_t)g_q4b.n_sm * 16u + n_mat - 1u) / n_mat;
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)n_mat);
    const uint64_t off = code_bytes(rows, (uint32_t)cols);
    const bool vec = aligned(d_codes, 16);
    auto go = [&](auto k) {
        q4b_launch(k, grid, dim3(256), 0, g_q4b.stream, d_codes, d_scales, (uint32_t)rows, (uint32_t)cols, words, (uint8_t *)d_w, stride, off, vec);
    };
    type == NV ? go(put_k<true>) : go(put_k<false>);
    g_q4b_launches++;
    return q4b_launch_ok("fp4 put");
}

extern "C" bool q4_cuda_fp4_quantize(uint32_t type, uint32_t form, const float *d_x, uint64_t ld_x, float mul, uint64_t rows, uint64_t cols, void *d_q) {
    using namespace fp4;
    if (!g_q4b.ok || !shape(type, rows, cols) || form > WEIGHTS || !d_x || !d_q || ld_x < cols || !aligned(d_x, 4) || !aligned(d_q, 16)) return false;
    return quantize<false>(type, form, d_x, ld_x, mul, rows, cols, d_q);
}

extern "C" bool q4_cuda_fp4_swiglu_quantize(uint32_t type, const float *d_gu, uint64_t ld_gu, float mul, uint64_t rows, uint64_t n_ff, void *d_hq) {
    using namespace fp4;
    if (!g_q4b.ok || !shape(type, rows, n_ff) || !d_gu || !d_hq || ld_gu < 2u * n_ff || !aligned(d_gu, 4) || !aligned(d_hq, 16)) return false;
    return quantize<true>(type, ROWS, d_gu, ld_gu, mul, rows, n_ff, d_hq);
}

extern "C" bool q4_cuda_fp4_values(uint32_t type, uint32_t form, const void *d_q, uint64_t rows, uint64_t cols, float *d_out, uint64_t ld_out) {
    using namespace fp4;
    if (!g_q4b.ok || !shape(type, rows, cols) || form > WEIGHTS || !d_q || !d_out || ld_out < cols || !aligned(d_q, 16) || !aligned(d_out, 4)) return false;
    OnDevice dev;
    const uint8_t *codes = (const uint8_t *)d_q, *scales = codes + code_bytes(rows, (uint32_t)cols);
    const uint32_t c = (uint32_t)cols, words = n_words(type == NV, c), groups = (uint32_t)((rows + 7u) / 8u), pieces = (c + 255u) / 256u;
    const uint32_t want = (8u * (uint32_t)g_q4b.n_sm + groups - 1u) / groups;
    const dim3 grid(groups, pieces < want ? pieces : want);
    auto go = [&](auto k) { q4b_launch(k, grid, dim3(256), 0, g_q4b.stream, codes, scales, rows, row_pitch(rows), c, words, d_out, ld_out); };
    const bool vec = aligned(d_out, 32) && ld_out % 8u == 0;
    auto pick = [&](auto nv, auto wf) {
        constexpr bool N = decltype(nv)::value, W = decltype(wf)::value;
        vec ? go(values_k<N, W, true>) : go(values_k<N, W, false>);
    };
    using yes = std::true_type;
    using no = std::false_type;
    if (form == ROWS) type == NV ? pick(yes(), no()) : pick(no(), no());
    else type == NV ? pick(yes(), yes()) : pick(no(), yes());
    g_q4b_launches++;
    return q4b_launch_ok("fp4 values");
}

extern "C" bool q4_cuda_fp4_mul(uint32_t type, const void *d_w, uint64_t w_rows, uint64_t w_cols, const void *d_xq, uint64_t rows, float scale,
                                float *d_y, uint64_t ld_y) {
    using namespace fp4;
    if (!g_q4b.ok || !shape(type, w_rows, w_cols) || !shape(type, rows, w_cols) || !d_w || !d_xq || !d_y || ld_y < w_rows || !aligned(d_w, 16) ||
        !aligned(d_xq, 16) || !aligned(d_y, 4))
        return false;
    MArgs a = {};
    a.w = (const uint8_t *)d_w;
    a.cols = (uint32_t)w_cols;
    a.w_rows = (uint32_t)w_rows;
    a.words = n_words(type == NV, a.cols);
    a.w_off = code_bytes(w_rows, a.cols);
    a.x = (const uint8_t *)d_xq;
    a.xs = a.x + code_bytes(rows, a.cols);
    a.x_rows = a.total = rows;
    a.x_pitch = row_pitch(rows);
    a.n_expert = 1;
    a.scale = scale;
    a.dst = d_y;
    a.ld = ld_y;
    a.err = g_q4b.err_d;
    return product(type, a);
}

extern "C" bool q4_cuda_fp4_mul_id(uint32_t type, const void *d_w, uint64_t w_rows, uint64_t w_cols, uint64_t expert_stride_bytes, uint32_t n_expert,
                                   const void *d_xq, uint64_t xq_rows, const int32_t *d_rows, const int32_t *d_bounds, uint64_t total_rows, float scale,
                                   const float *d_expert_scale, float *d_dst, uint64_t ld_dst) {
    using namespace fp4;
    if (!g_q4b.ok || !shape(type, w_rows, w_cols) || !shape(type, xq_rows, w_cols) || !d_w || !d_xq || !d_bounds || !d_dst || ld_dst < w_rows ||
        !n_expert || n_expert > 1024u || expert_stride_bytes % 16u ||
        (n_expert > 1u && expert_stride_bytes < bytes(type == NV, WEIGHTS, w_rows, (uint32_t)w_cols)) || total_rows > 0x7fffffffull ||
        (!d_rows && total_rows > xq_rows) || !aligned(d_w, 16) || !aligned(d_xq, 16) || !aligned(d_dst, 4))
        return false;
    if (!total_rows) return true;
    MArgs a = {};
    a.w = (const uint8_t *)d_w;
    a.stride = expert_stride_bytes;
    a.cols = (uint32_t)w_cols;
    a.w_rows = (uint32_t)w_rows;
    a.words = n_words(type == NV, a.cols);
    a.w_off = code_bytes(w_rows, a.cols);
    a.x = (const uint8_t *)d_xq;
    a.xs = a.x + code_bytes(xq_rows, a.cols);
    a.x_rows = xq_rows;
    a.x_pitch = row_pitch(xq_rows);
    a.rows = d_rows;
    a.bounds = d_bounds;
    a.n_expert = n_expert;
    a.total = total_rows;
    a.scale = scale;
    a.each = d_expert_scale;
    a.dst = d_dst;
    a.ld = ld_dst;
    a.err = g_q4b.err_d;
    return product(type, a);
}

extern "C" void q4_cuda_fp4_products(uint64_t count[3]) {
    for (int i = 0; count && i < 3; i++) count[i] = fp4::g_ran[i].load();
}
