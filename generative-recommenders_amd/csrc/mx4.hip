// Tables and layers in 4 bits: blocks of 32 values of a row share a power-of-two scale (e8m0 byte), values are e2m1.
//
// quantize / dequantize: one pass, bound by HBM.  A lane owns 8 columns, four lanes a block of 32.  4,000,001 x 64: fp32 to
// 4 bits 230 us (5.05 TB/s), to bf16 131 us (4.95 TB/s); a copy of 1 GiB reaches 5.1 TB/s.  Widths that are no multiple of 8 are
// read and written element by element: x 60 fp32 to 4 bits 245 us (4.5 TB/s), back 577 (1.9; bf16 237 and 310).
//
// linear: out[m, n] = sum_k x[m, k] W[n, k] for few rows of x, bound by the bytes of W (and by out where it is wide).  A
// lane loads one block of W (16 bytes, 32 codes); v_cvt_scalef32_pk_bf16_fp4 turns two codes and the scale into two bf16
// values exactly, and the bf16 MFMA (16 x 16 x 32) multiplies them by x with fp32 sums.  The scaled 4 x 8 bit MFMA would
// take the codes as they are, but it sums with fewer bits: 5e-5 relative error on random operands, against 1e-7 here.
// x enters as exact bf16: bfloat16 and mx8 values are, fp32 values are cut into three bf16 terms (8 + 8 + 8 bits); only what
// lies below bf16's last bit, 2^-133, is lost.
// The MFMA adds over k in any order, so the k of step i (0..3) and lane group j (0..3) is 32 j + 8 i + e (e = 0..7): the
// i-th dword of the lane's own block.
#include "hmx_common.h"

#include <algorithm>

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The factor of a scale byte as fp32 (2^-127 is a denormal number, 255 stands for NaN).
__device__ __forceinline__ float scale_value(uint32_t b) {
    const uint32_t bits = b << 23;
    return __uint_as_float(b == 0 ? 0x400000u : b == 255 ? 0x7fc00000u : bits);
}

// Least e with amax <= 6 * 2^e, -126 <= e <= 127 (0 for a block of zeros); 128 marks a block that is not finite.
__device__ __forceinline__ int mx4_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    if (u >= 0x7f800000u) return 128;
    if (u == 0) return 0;
    const int e = (int)(u >> 23) - 127 - 2 + ((u & 0x7fffffu) > 0x400000u);     // 6 = 1.5 * 2^2
    return max(e, -126);
}

// ------------------------------------------------------------------------------- quantize
// FAST: rows of a multiple of 8 columns, 16-byte aligned.  `oc` = octets of a row (a multiple of 4: whole blocks).
template <typename T, bool FAST>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* __restrict__ x, int64_t ld, int64_t total, uint32_t oc,
                                                           uint32_t d, uint32_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales) {
    for (int64_t base = (int64_t)blockIdx.x * 256; base < total; base += (int64_t)gridDim.x * 256) {
        const int64_t row0 = base / oc;
        const uint32_t local = (uint32_t)(base - row0 * oc) + threadIdx.x;
        const int64_t row = row0 + local / oc;
        const uint32_t q = local % oc, c = 8 * q;
        const bool ok = base + threadIdx.x < total;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
        if (ok) {
            const T* p = x + row * ld + c;
            if constexpr (FAST) {
                if (c < d) {
                    if constexpr (sizeof(T) == 4) {
                        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
                    } else {
                        const f32x8 a = __builtin_convertvector(*reinterpret_cast<const bf16x8*>(p), f32x8);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = a[e];
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < d) v[e] = (float)p[e];
            }
        }
        float amax = 0.f;
        bool nan = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            amax = fmaxf(amax, fabsf(v[e]));
            nan |= v[e] != v[e];
        }
        if (nan) amax = __uint_as_float(0x7f800000u);                  // fmaxf drops NaN
        amax = fmaxf(amax, __shfl_xor(amax, 1));
        amax = fmaxf(amax, __shfl_xor(amax, 2));
        const int ex = mx4_exponent(amax);
        if (!ok) continue;
        uint32_t word = 0;
        if (ex != 128) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], -ex);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], 1.f, 0);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], 1.f, 1);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], 1.f, 2);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], 1.f, 3);
        }
        const int64_t at = base + threadIdx.x;                          // = row * oc + q
        codes[at] = word;
        if ((q & 3) == 0) scales[at / 4] = (uint8_t)(ex + 127);
    }
}

// Eight codes of one block as fp32 (exact).
__device__ __forceinline__ void decode8(uint32_t word, float scale, float (&v)[8]) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2);
    const bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
    v[0] = (float)a[0], v[1] = (float)a[1], v[2] = (float)b[0], v[3] = (float)b[1];
    v[4] = (float)c[0], v[5] = (float)c[1], v[6] = (float)e[0], v[7] = (float)e[1];
}
__device__ __forceinline__ void decode8(u32x2 word, float scale, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)word[h], false);
        const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)word[h], true);
        v[4 * h] = a[0] * scale, v[4 * h + 1] = a[1] * scale, v[4 * h + 2] = b[0] * scale, v[4 * h + 3] = b[1] * scale;
    }
}

template <typename WORD, typename OUT, bool FAST>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const WORD* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            int64_t total, uint32_t oc, uint32_t d, OUT* __restrict__ out) {
    for (int64_t base = (int64_t)blockIdx.x * 256; base < total; base += (int64_t)gridDim.x * 256) {
        const int64_t at = base + threadIdx.x;
        if (at >= total) continue;
        const int64_t row0 = base / oc;
        const uint32_t local = (uint32_t)(base - row0 * oc) + threadIdx.x;
        const int64_t row = row0 + local / oc;
        const uint32_t c = 8 * (local % oc);
        if (c >= d) continue;
        float v[8];
        decode8(codes[at], scale_value(scales[at / 4]), v);
        OUT* p = out + row * d + c;
        if constexpr (FAST) {
            if constexpr (sizeof(OUT) == 4) {
                *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                const f32x8 a = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
                *reinterpret_cast<bf16x8*>(p) = __builtin_convertvector(a, bf16x8);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < d) p[e] = (OUT)v[e];
        }
    }
}

// ------------------------------------------------------------------------------- linear
enum { kXF32 = 0, kXBf16 = 1, kXMx8 = 2 };

struct LinearArgs {
    const void* x;
    int64_t ldx;
    const uint8_t* xs;
    int M;
    const u32x4* codes;       // (N, nblk) blocks of 32 codes
    const uint8_t* scales;    // (N, nblk)
    int64_t N;
    int K, nblk;
    void* out;
};

template <int XK>
constexpr int planes() { return XK == kXF32 ? 3 : 1; }

template <int PL>
struct XTerms {
    bf16x8 p[PL];
};

// v = h + m + l exactly: each term is the next 8 bits of the significand (cut, not rounded: no carry, and the largest finite
// value stays finite).  An infinity or a NaN stays in the first term alone.  The others may be zero where v is not, and zero
// times an infinite value of W (scale bytes 253 and 254) is NaN: what they would add to the first term's infinity, which has
// their sign, is left out (add_term, finite).
__device__ __forceinline__ XTerms<3> cut3(const float (&v)[8]) {
    uint32_t u[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        uint32_t b = __float_as_uint(v[e]);
        const bool fin = (b & 0x7f800000u) != 0x7f800000u;
        if (!fin && (b & 0x7fffffu)) b |= 0x400000u;                 // a NaN whose payload would be cut away
        u[0][e] = b & 0xffff0000u;
        const float r1 = fin ? v[e] - __uint_as_float(u[0][e]) : 0.f;
        u[1][e] = __float_as_uint(r1) & 0xffff0000u;
        u[2][e] = __float_as_uint(r1 - __uint_as_float(u[1][e]));
    }
    XTerms<3> t;
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (u[q][2 * e] >> 16) | (u[q][2 * e + 1] & 0xffff0000u);
        t.p[q] = __builtin_bit_cast(bf16x8, w);
    }
    return t;
}

// The sum of the products with the first term, and that with a later one: NaN where that met an infinity (or where the first's is).
__device__ __forceinline__ float add_term(float first, float later) { return later == later ? first + later : first; }
// W for the later terms of an accumulator that the first term shares: the largest number in place of an infinity.
__device__ __forceinline__ bf16x8 finite(bf16x8 v) {
    u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & 0x7fffu) == 0x7f80u) w[i] -= 1u;
        if ((w[i] & 0x7fff0000u) == 0x7f800000u) w[i] -= 0x10000u;
    }
    return __builtin_bit_cast(bf16x8, w);
}

// x[m, k .. k + 7] as exact bf16 terms; columns past K and rows past M read as zero.
template <int XK>
__device__ __forceinline__ XTerms<planes<XK>()> load_x8(const LinearArgs& a, int m, int k) {
    XTerms<planes<XK>()> t;
    const bool row = m < a.M;
    if constexpr (XK == kXBf16) {
        const __bf16* p = (const __bf16*)a.x + m * a.ldx + k;
#pragma unroll
        for (int e = 0; e < 8; ++e) t.p[0][e] = row && k + e < a.K ? p[e] : (__bf16)0.f;
    } else if constexpr (XK == kXMx8) {
        f32x8 v;
        if (row && k < a.K) {                                           // K = 32 * nblk
            const u32x2 w = *reinterpret_cast<const u32x2*>((const uint8_t*)a.x + (int64_t)m * a.K + k);
            float f[8];
            decode8(w, scale_value(a.xs[(int64_t)m * a.nblk + k / 32]), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = f[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
        }
        t.p[0] = __builtin_convertvector(v, bf16x8);
    } else {
        const float* p = (const float*)a.x + m * a.ldx + k;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = row && k + e < a.K ? p[e] : 0.f;
        t = cut3(v);
    }
    return t;
}

__device__ __forceinline__ bf16x8 decode_bf16(uint32_t word, float scale) {
    u32x4 w;
    w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1));
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3));
    return __builtin_bit_cast(bf16x8, w);
}

// Eight mx8 codes (two words) and their scale: what convertvector makes of the values, bit for bit.
__device__ __forceinline__ bf16x8 decode_bf16(uint32_t lo, uint32_t hi, float scale) {
    u32x4 w;
    w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return __builtin_bit_cast(bf16x8, w);
}

__device__ __forceinline__ bf16x8 zero_if(bool z, bf16x8 v) {
    u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = z ? 0u : w[i];
    return __builtin_bit_cast(bf16x8, w);
}

template <typename OUT>
__device__ __forceinline__ void store_out(OUT* p, float v) { *p = (OUT)v; }

// v[t] of lane group j becomes v[j] of lane group t (groups of 16 lanes).
__device__ __forceinline__ void transpose_groups(float (&v)[4]) {
    typedef uint32_t pair __attribute__((ext_vector_type(2)));
    uint32_t u[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) u[t] = __float_as_uint(v[t]);
    const pair a = __builtin_amdgcn_permlane32_swap(u[0], u[2], false, false), b = __builtin_amdgcn_permlane32_swap(u[1], u[3], false, false);
    const pair c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    v[0] = __uint_as_float(c[0]), v[1] = __uint_as_float(c[1]), v[2] = __uint_as_float(d[0]), v[3] = __uint_as_float(d[1]);
}

// K <= 128 (scores of a table of embeddings): x stays in registers, waves walk the table 64 rows at a time.
// Bound by HBM: 1 row x 4,000,001 x 64 27.8 us (152 MB, 5.5 TB/s), 16 rows x 1,000,003 x 60 22.2 us (98 MB, 64 of them written).
// Several fp32 rows (three terms each, one MFMA a term and row group) are bound by those and by their registers: 4 rows x
// 4,000,001 x 64 78 us (2.6 TB/s), 16 rows 108 (3.6; bf16 101), 67 rows, five passes over the table, 465 (bf16 450).
// With one or two blocks a row (R = 4 or 2), the lane groups of one load hold R groups of 16 rows, so that a load still is
// 1 KB of consecutive codes; the MFMA would add the groups up, so x is zero in the lane groups of the other row groups:
//   REP (planes * M <= 4): rows 4 j + i of the x operand hold term / row i for lane group j's own row group, so that lane
//        (j, c) ends with all its sums for table row 16 j + c of the 64, and a wave stores 64 consecutive scores;
//   else: one MFMA per row group, x masked to that group's lanes.
template <int XK, int R, bool REP, typename OUT>
__global__ __launch_bounds__(256) void linear_short_kernel(LinearArgs a) {
    constexpr int PL = planes<XK>(), LOADS = 4 / R;
    const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
    const int b = R == 1 ? j : R == 2 ? (j & 1) : 0;                    // the block of 32 this lane owns
    const int h = R == 1 ? 0 : R == 2 ? (j >> 1) : j;                   // the row group it loads from
    const int mbase = blockIdx.y * 16;
    bf16x8 xr[4][REP ? 1 : PL];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (REP) {
            const int jr = c >> 2, ir = c & 3;
            const bool mine = R == 1 || (R == 2 ? (j >> 1) == (jr & 1) : j == jr);
            const XTerms<PL> t = load_x8<XK>(a, mine ? (PL == 3 ? 0 : ir) : a.M, 32 * b + 8 * i);
            if constexpr (PL == 3) {
                xr[i][0] = zero_if(ir != 0, t.p[0]);
                xr[i][0] = ir == 1 ? t.p[1] : xr[i][0];
                xr[i][0] = ir == 2 ? t.p[2] : xr[i][0];
            } else {
                xr[i][0] = t.p[0];
            }
        } else {
            const XTerms<PL> t = load_x8<XK>(a, mbase + c, 32 * b + 8 * i);
#pragma unroll
            for (int q = 0; q < PL; ++q) xr[i][q] = t.p[q];
        }
    }
    OUT* out = (OUT*)a.out;
    const int64_t tiles = (a.N + 63) / 64, step = (int64_t)gridDim.x * 4;
    const bool block_ok = b < a.nblk;
    u32x4 w[LOADS], wn[LOADS];
    uint32_t sc[LOADS], scn[LOADS];
    auto fetch = [&](int64_t tile, u32x4(&wd)[LOADS], uint32_t(&sd)[LOADS]) {
#pragma unroll
        for (int t = 0; t < LOADS; ++t) {
            int64_t n = tile * 64 + t * (16 * R) + 16 * h + c;
            n = n < a.N ? n : a.N - 1;
            const int64_t at = n * a.nblk + (block_ok ? b : 0);
            wd[t] = a.codes[at];
            sd[t] = a.scales[at];
        }
    };
    int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile < tiles) fetch(tile, w, sc);
    for (; tile < tiles; tile += step) {
        if (tile + step < tiles) fetch(tile + step, wn, scn);
        f32x4 acc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < LOADS; ++t) {
            const float s = block_ok ? scale_value(sc[t]) : 1.f;
            // rows that share an MFMA must not meet each other's infinities (6 * 2^126 and up) and NaN: zero times those
            // is NaN, so then W is masked to one row group at a time as well
            const bool odd = (R > 1 || PL > 1) && __any(block_ok && sc[t] >= 253);
            if constexpr (REP) {
                if (R > 1 && odd) {
                    f32x4 kept = {0.f, 0.f, 0.f, 0.f};
                    for (int g = 0; g < R; ++g) {
                        f32x4 one = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            one = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                xr[i][0], zero_if(h != g, decode_bf16(block_ok ? w[t][i] : 0u, s)), one, 0, 0, 0);
                        const bool mine = (R == 2 ? (j & 1) : j) == g;
#pragma unroll
                        for (int i = 0; i < 4; ++i) kept[i] = mine ? one[i] : kept[i];
                    }
                    acc[t] = kept;
                    continue;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bf16x8 wv = decode_bf16(block_ok ? w[t][i] : 0u, s);
                if constexpr (REP) {
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xr[i][0], wv, acc[t], 0, 0, 0);
                } else {
#pragma unroll
                    for (int g = 0; g < R; ++g) {
                        const bf16x8 wg = R > 1 && odd ? zero_if(h != g, wv) : wv;
                        const bf16x8 wl = PL > 1 && odd ? finite(wg) : wg;
#pragma unroll
                        for (int q = 0; q < PL; ++q)
                            acc[t * R + g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(zero_if(R > 1 && h != g, xr[i][q]), q ? wl : wg,
                                                                                     acc[t * R + g], 0, 0, 0);
                    }
                }
            }
        }
        if constexpr (REP) {
            const int t = R == 1 ? j : R == 2 ? (j >> 1) : 0;
            f32x4 v = acc[0];
#pragma unroll
            for (int q = 1; q < LOADS; ++q) {
                const bool mine = t == q;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = mine ? acc[q][i] : v[i];
            }
            const int64_t n = tile * 64 + lane;                         // load t, row group of lane group j, table row c
            if (n < a.N) {
                if constexpr (PL == 3) {
                    store_out(out + n, add_term(add_term(v[0], v[1]), v[2]));
                } else {
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        if (m < a.M) store_out(out + m * a.N + n, v[m]);
                }
            }
        } else {
            // lane group j holds rows 4 j + i of each 16 table rows: exchanged, so that a store is 64 consecutive scores
            const int64_t n = tile * 64 + lane;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4] = {acc[0][i], acc[1][i], acc[2][i], acc[3][i]};
                transpose_groups(v);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int m = mbase + 4 * g + i;
                    if (n < a.N && m < a.M) store_out(out + m * a.N + n, v[g]);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < LOADS; ++t) w[t] = wn[t], sc[t] = scn[t];
    }
}

// Longer rows, more than 8 of them, go in two launches.  The first lays x out as the second one's lanes take it: per tile of 16 operand rows and
// 128 columns, step i and lane, the eight bf16 values of one MFMA operand.  An fp32 row is three operand rows (its terms; five
// rows of x to a tile), any other one.  Read as it lies, x cost more than W: rows of a power of two of bytes lie in one
// memory channel and one set of the cache, and every block decodes all of x (32 x 8192 x 8192 mx8: 22 us, this way 14 and 3).  What
// bounds the second: every block reads all of x from L2 (as bfloat16 134 MB there: with x at one address it took 6 us less,
// with W at one address 5; as mx8 half of that), and what a launch's waves need to start.
template <int XK>
__global__ __launch_bounds__(256) void linear_pack_kernel(LinearArgs a, int chunks, int64_t total, u32x4* __restrict__ packed) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= total) return;
    const int lane = (int)(t & 63), i = (int)(t >> 6) & 3, r = lane & 15;
    const int64_t unit = t >> 8;
    const int chunk = (int)(unit % chunks), tile = (int)(unit / chunks);
    const int m = XK == kXF32 ? tile * 5 + r / 3 : tile * 16 + r;
    if ((XK == kXF32 && r == 15) || m >= a.M) return;                // lanes that the second launch leaves out
    const XTerms<planes<XK>()> x = load_x8<XK>(a, m, 256 * (chunk >> 1) + 64 * (lane >> 4) + 32 * (chunk & 1) + 8 * i);
    bf16x8 v = x.p[0];
    if constexpr (XK == kXF32) v = r % 3 == 1 ? x.p[1] : r % 3 == 2 ? x.p[2] : v;
    packed[t] = __builtin_bit_cast(u32x4, v);
}

// mx8 rows stay in 8 bits, half of what bf16 would have the second launch read: per tile and chunk, half h of a lane's block
// and lane, 16 codes, and behind all of these the scale byte of each lane.
__global__ __launch_bounds__(256) void linear_pack_mx8_kernel(LinearArgs a, int chunks, int64_t total, u32x4* __restrict__ packed) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;          // (unit, half, lane)
    if (t >= total) return;
    const int lane = (int)(t & 63), h = (int)(t >> 6) & 1;
    const int64_t unit = t >> 7;
    const int chunk = (int)(unit % chunks), m = (int)(unit / chunks) * 16 + (lane & 15);
    if (m >= a.M) return;                                               // lanes that the second launch leaves out
    const int b = 8 * (chunk >> 1) + 2 * (lane >> 4) + (chunk & 1);
    const int64_t block = (int64_t)m * a.nblk + b;
    packed[t] = b < a.nblk ? ((const u32x4*)a.x)[2 * block + h] : u32x4{0, 0, 0, 0};
    if (h == 0) reinterpret_cast<uint8_t*>(packed + total)[unit * 64 + lane] = b < a.nblk ? a.xs[block] : 127;
}

// What lanes past the end of a row load in place of codes and scales.
__device__ const u32x4 kZeros = {};

// The second: W waves a block, KW of them share 16 RT rows of the table and split its K (256 columns in turn, two chunks of
// 128 of which a lane has two neighbouring blocks: a wave reads whole 128-byte lines); their sums meet in LDS and are added in
// wave order.  The next chunk is in flight while one is multiplied.  TERMS: operand rows of a row of x; PACKED: x comes from the
// first launch.
template <int XK, bool PACKED, int W, int MT, int RT, typename OUT>
__global__ __launch_bounds__(64 * W) void linear_long_kernel(LinearArgs a, const u32x4* __restrict__ packed,
                                                             const uint8_t* __restrict__ packed_scales, int KW) {
    constexpr int TERMS = planes<XK>(), XV = XK == kXMx8 ? 2 : 4;    // vectors of x to a lane's block
    constexpr int NE = RT * MT * 4, ROWS = TERMS == 3 ? 5 : 16;      // rows of x to a tile
    __shared__ float red[W][NE][64];
    const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4, wave = threadIdx.x >> 6;
    const int kw = wave % KW, group = wave / KW;
    const int64_t n0 = ((int64_t)blockIdx.x * (W / KW) + group) * (16 * RT);
    const int chunks = 2 * ((a.nblk + 7) / 8);
    f32x4 acc[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[r][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    int64_t row_at[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) row_at[r] = (n0 + 16 * r + c < a.N ? n0 + 16 * r + c : a.N - 1) * a.nblk;
    bool used[MT];                                                   // operand rows that there are; the others are zero
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int left = a.M - (int)(blockIdx.y * MT + m) * ROWS;
        used[m] = c < TERMS * (left < ROWS ? left : ROWS);
    }
    // blocks begin at different columns: rows of a power of two of bytes lie in the same memory channel column by column, and
    // blocks in step would all wait for it
    const int pairs = chunks / 2, mine = 2 * ((pairs - kw + KW - 1) / KW), turn = (int)(blockIdx.x * 37u % (unsigned)pairs);
    struct Chunk {
        u32x4 w[RT], x[MT][XV];
        uint8_t xs[MT];
    };
    uint32_t sc[RT];                                                 // both chunks' scales, the second's in the upper byte
    const int64_t all = a.N * a.nblk;
    auto pair_of = [&](int n) {
        const int pair = kw + KW * (n >> 1) + turn;
        return pair < pairs ? pair : pair - pairs;
    };
    auto fetch = [&](int n, Chunk& t) {                              // the n-th chunk of this wave
        const int chunk = 2 * pair_of(n) + (n & 1), b = 4 * (chunk & ~1) + 2 * j + (chunk & 1);
        const bool past = b >= a.nblk;
#pragma unroll
        for (int r = 0; r < RT; ++r) t.w[r] = *(past ? &kZeros : a.codes + row_at[r] + b);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int64_t unit = (int64_t)(blockIdx.y * MT + m) * chunks + chunk;
            const int row = (int)(blockIdx.y * MT + m) * 16 + c;     // not PACKED: of x itself
            const u32x4* p = PACKED ? packed + unit * (64 * XV) + lane
                                    : (const u32x4*)a.x + (XK == kXMx8 ? (int64_t)row * a.nblk * XV : row * (a.ldx / 8)) + (int64_t)b * XV;
#pragma unroll
            for (int i = 0; i < XV; ++i) {
                t.x[m][i] = u32x4{0, 0, 0, 0};
                if (used[m] && !past) t.x[m][i] = p[(PACKED ? 64 : 1) * i];
            }
            t.xs[m] = 127;
            if (XK == kXMx8 && used[m] && !past) t.xs[m] = PACKED ? packed_scales[unit * 64 + lane] : a.xs[(int64_t)row * a.nblk + b];
        }
    };
    auto fetch_scales = [&](int n, uint32_t (&sd)[RT]) {             // of the pair that the n-th chunk begins
        const int b = 8 * pair_of(n) + 2 * j;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int64_t at = row_at[r] + b;
            uint16_t two = 0;
            if (at + 2 <= all) __builtin_memcpy(&two, a.scales + at, 2);
            else if (b < a.nblk) two = a.scales[at];
            sd[r] = b + 1 < a.nblk ? two : b < a.nblk ? two & 255u : 0u;
        }
    };
    auto multiply = [&](const Chunk& t, int half) {
        float s[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r] = scale_value((sc[r] >> (8 * half)) & 255u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x8 xv[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if constexpr (XK == kXMx8) xv[m] = decode_bf16(t.x[m][i / 2][2 * (i & 1)], t.x[m][i / 2][2 * (i & 1) + 1], scale_value(t.xs[m]));
                else xv[m] = __builtin_bit_cast(bf16x8, t.x[m][i]);
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const bf16x8 wv = decode_bf16(t.w[r][i], s[r]);
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[r][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv[m], wv, acc[r][m], 0, 0, 0);
            }
        }
    };
    if (n0 < a.N && mine > 0) {
        Chunk even, odd;
        uint32_t next[RT];
        fetch(0, even);
        fetch_scales(0, sc);
#pragma unroll 1
        for (int n = 0; n < mine; n += 2) {
            fetch(n + 1, odd);
            multiply(even, 0);
            if (n + 2 < mine) {
                fetch(n + 2, even);
                fetch_scales(n + 2, next);
            }
            multiply(odd, 1);
#pragma unroll
            for (int r = 0; r < RT; ++r) sc[r] = next[r];
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[wave][(r * MT + m) * 4 + i][lane] = acc[r][m][i];
    __syncthreads();
    OUT* out = (OUT*)a.out;
    for (int e = kw * 64 + lane; e < RT * MT * ROWS * 16; e += KW * 64) {
        const int col = e & 15, q = (e >> 4) % ROWS, rm = (e >> 4) / ROWS;
        float v = 0.f;
#pragma unroll
        for (int p = 0; p < TERMS; ++p) {                            // the first term's sum, then the others'
            const int row = TERMS * q + p;
            float sum = 0.f;
            for (int k = 0; k < KW; ++k) sum += red[group * KW + k][rm * 4 + (row & 3)][(row >> 2) * 16 + col];
            v = p ? add_term(v, sum) : sum;
        }
        const int m = ((int)blockIdx.y * MT + rm % MT) * ROWS + q;
        const int64_t n = n0 + 16 * (rm / MT) + col;
        if (n < a.N && m < a.M) store_out(out + m * a.N + n, v);
    }
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int kWavesLong = 8;
constexpr int kDirect = 8;

// Tiles of 16 operand rows that M rows of x make for linear_long_kernel.
int operand_tiles(int x_kind, int64_t M) { return (int)hmx_ceil_div(M, x_kind == kXF32 ? 5 : 16); }

template <int XK, typename OUT>
void launch_linear(const LinearArgs& a, u32x4* packed, hipStream_t st) {
    if (a.nblk <= 4) {
        const bool rep = XK == kXF32 ? a.M == 1 : a.M <= 4;
        const int64_t want = hmx_ceil_div(hmx_ceil_div(a.N, 64), 4);
        const unsigned my = (unsigned)hmx_ceil_div(a.M, 16);
        // few enough blocks that one round holds them (a wave's start, x from memory into registers, costs 3 us), and where the
        // output is wide fewer still: its write streams disturb each other.  Measured with 512 / 1024 / 2048 blocks: 1 x
        // 4,000,001 x 64 fp32 38 / 33 / 37 us, 16 x 1,000,003 x 60 bf16 26 / 30 / 37 us.
        const int64_t most = rep ? 1024 : std::max<int64_t>(1, 512 / my);
        const dim3 grid((unsigned)std::min<int64_t>(want, most), rep ? 1 : my);
#define SHORT(R, REP) hipLaunchKernelGGL((linear_short_kernel<XK, R, REP, OUT>), grid, dim3(256), 0, st, a)
        if (a.nblk == 1) { if (rep) SHORT(4, true); else SHORT(4, false); }
        else if (a.nblk == 2) { if (rep) SHORT(2, true); else SHORT(2, false); }
        else { if (rep) SHORT(1, true); else SHORT(1, false); }
#undef SHORT
        return;
    }
    const int chunks = 2 * (int)hmx_ceil_div(a.nblk, 8), tiles = operand_tiles(XK, a.M);
    int kw = kWavesLong;
    while (kw > 1 && chunks < 4 * kw) kw /= 2;
#define LONG(PACKED, MT, RT)                                                                                              \
    hipLaunchKernelGGL((linear_long_kernel<XK, PACKED, kWavesLong, MT, RT, OUT>),                                          \
                       dim3((unsigned)hmx_ceil_div(a.N, 16 * RT * (kWavesLong / kw)), (unsigned)hmx_ceil_div(tiles, MT)), \
                       dim3(64 * kWavesLong), 0, st, a, packed, packed_scales, kw)
    // two tiles of x a wave share what decoding W costs, two of W what loading x does; one of W where two would leave compute
    // units without a block (32 x 4096 x 4096 mx8: 8.5 us against 10.0; 32 x 8192 x 8192, which has enough: 17.9 against 16.0)
    const bool wide = hmx_ceil_div(a.N, 32 * (kWavesLong / kw)) >= 256;
    const int64_t total = (int64_t)tiles * chunks * (XK == kXMx8 ? 128 : 256);
    const uint8_t* packed_scales = reinterpret_cast<const uint8_t*>(packed + total);
    // few rows are read as they lie (fp32 has to be cut, a bf16 row has to have whole blocks): one launch, and the rows share
    // few enough cache lines.  As they lie / packed: 1 x 8192 x 8192 bf16 10.7 / 13.3 us, 8 rows 13.4 / 13.8, 16 rows 18.6 / 14.5;
    // 1 x 1000 x 5024 4.4 / 6.8; 8 x 8192 x 8192 mx8 12.1 / 13.1, 16 rows 14.3 / 13.3
    if constexpr (XK != kXF32) {
        if (a.M <= kDirect && (XK == kXMx8 || ((a.M == 1 || a.ldx % 8 == 0) && a.K % 32 == 0 && aligned(a.x, 16)))) {
            if (wide) LONG(false, 1, 2); else LONG(false, 1, 1);
            return;
        }
    }
    const dim3 pack_grid((unsigned)hmx_ceil_div(total, 256));
    if constexpr (XK == kXMx8) hipLaunchKernelGGL(linear_pack_mx8_kernel, pack_grid, dim3(256), 0, st, a, chunks, total, packed);
    else hipLaunchKernelGGL(linear_pack_kernel<XK>, pack_grid, dim3(256), 0, st, a, chunks, total, packed);
    if (tiles == 1) { if (wide) LONG(true, 1, 2); else LONG(true, 1, 1); }
    else { if (wide) LONG(true, 2, 2); else LONG(true, 2, 1); }
#undef LONG
}

// Octets of a row, or 0 when the sizes do not fit the kernels' 32-bit column arithmetic.
uint32_t octets(int64_t d) { return d >= 1 && d <= (1 << 26) ? (uint32_t)(hmx_ceil_div(d, 32) * 4) : 0; }

}  // namespace

// ================================================================================ C ABI
extern "C" int hmx_mx4_quantize(const void* table, int64_t ld, int64_t n, int64_t d, int bf16, void* codes, void* scales,
                                void* stream) {
    HMX_ENTER();
    const uint32_t oc = octets(d);
    if (n < 0 || ld < 0 || oc == 0) return HMX_EINVAL;
    if (n == 0) return HMX_OK;
    if (!table || !codes || !scales || !aligned(codes, 16)) return HMX_EINVAL;
    const int64_t total = n * oc;
    const dim3 grid((unsigned)std::min<int64_t>(hmx_ceil_div(total, 256), 1 << 20));
    const bool fast = d % 8 == 0 && (ld * (bf16 ? 2 : 4)) % 16 == 0 && aligned(table, 16);
    const hipStream_t st = (hipStream_t)stream;
#define QUANT(T, FAST)                                                                                               \
    hipLaunchKernelGGL((mx4_quantize_kernel<T, FAST>), grid, dim3(256), 0, st, (const T*)table, ld, total, oc, (uint32_t)d, \
                       (uint32_t*)codes, (uint8_t*)scales)
    if (bf16) { if (fast) QUANT(__bf16, true); else QUANT(__bf16, false); }
    else { if (fast) QUANT(float, true); else QUANT(float, false); }
#undef QUANT
    HMX_CHECK_LAUNCH();
    return HMX_OK;
}

extern "C" int hmx_mx_dequantize(const void* codes, const void* scales, int64_t n, int64_t d, int bits, int bf16, void* out,
                                 void* stream) {
    HMX_ENTER();
    const uint32_t oc = octets(d);
    if (n < 0 || oc == 0 || (bits != 4 && bits != 8)) return HMX_EINVAL;
    if (n == 0) return HMX_OK;
    if (!codes || !scales || !out || !aligned(codes, 16)) return HMX_EINVAL;
    const int64_t total = n * oc;
    const dim3 grid((unsigned)std::min<int64_t>(hmx_ceil_div(total, 256), 1 << 20));
    const bool fast = d % 8 == 0 && aligned(out, 16);
    const hipStream_t st = (hipStream_t)stream;
#define DEQUANT(W, OUT, FAST)                                                                                          \
    hipLaunchKernelGGL((mx_dequantize_kernel<W, OUT, FAST>), grid, dim3(256), 0, st, (const W*)codes, (const uint8_t*)scales, \
                       total, oc, (uint32_t)d, (OUT*)out)
    if (bits == 4) {
        if (bf16) { if (fast) DEQUANT(uint32_t, __bf16, true); else DEQUANT(uint32_t, __bf16, false); }
        else { if (fast) DEQUANT(uint32_t, float, true); else DEQUANT(uint32_t, float, false); }
    } else {
        if (bf16) { if (fast) DEQUANT(u32x2, __bf16, true); else DEQUANT(u32x2, __bf16, false); }
        else { if (fast) DEQUANT(u32x2, float, true); else DEQUANT(u32x2, float, false); }
    }
#undef DEQUANT
    HMX_CHECK_LAUNCH();
    return HMX_OK;
}

extern "C" size_t hmx_linear_mx4_workspace_bytes(int x_kind, int64_t M, int64_t K) {
    if (M <= 0 || K <= 128) return 0;
    const int64_t tiles = hmx_ceil_div(operand_tiles(x_kind, M), 2) * 2;      // read in twos
    return (size_t)(tiles * hmx_ceil_div(K, 256) * 2) * 4096;
}

extern "C" int hmx_linear_mx4(const void* x, int64_t ldx, const void* x_scales, int x_kind, int64_t M, const void* codes,
                              const void* scales, int64_t N, int64_t K, int out_bf16, void* out, void* workspace,
                              size_t workspace_bytes, void* stream) {
    HMX_ENTER();
    if (M < 0 || N < 0 || K < 1 || K > (1 << 26) || ldx < 0 || x_kind < 0 || x_kind > 2) return HMX_EINVAL;
    if (M == 0 || N == 0) return HMX_OK;
    if (!x || !codes || !scales || !out || !aligned(codes, 16) || (x_kind == kXMx8) != (x_scales != nullptr)) return HMX_EINVAL;
    // the grid's limits: 65535 blocks in y, 2^32 threads in x
    if (M > 65535 * 16 || hmx_ceil_div(N, 32) > (1 << 22)) return HMX_EINVAL;
    if (K > 128) {
        const int64_t tiles = operand_tiles(x_kind, M), chunks = 2 * hmx_ceil_div(K, 256);
        if (hmx_ceil_div(tiles, 2) > 65535 || tiles * chunks * (x_kind == kXMx8 ? 128 : 256) > (int64_t)UINT32_MAX - 256) return HMX_EINVAL;
    }
    if (x_kind == kXMx8 && (K % 32 || !aligned(x, 16))) return HMX_EINVAL;
    const LinearArgs a = {x, ldx, (const uint8_t*)x_scales, (int)M, (const u32x4*)codes, (const uint8_t*)scales, N, (int)K,
                          (int)hmx_ceil_div(K, 32), out};
    const size_t need = hmx_linear_mx4_workspace_bytes(x_kind, M, K);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return HMX_EWORKSPACE;
    const hipStream_t st = (hipStream_t)stream;
#define LINEAR(XK)                                                          \
    if (out_bf16) launch_linear<XK, __bf16>(a, (u32x4*)workspace, st);      \
    else launch_linear<XK, float>(a, (u32x4*)workspace, st)
    if (x_kind == kXF32) { LINEAR(kXF32); }
    else if (x_kind == kXBf16) { LINEAR(kXBf16); }
    else { LINEAR(kXMx8); }
#undef LINEAR
    HMX_CHECK_LAUNCH();
    return HMX_OK;
}
