// Residual add + RMS norm: s = rnd(x + r), y = s * (mean(s^2) + eps)^(-1/2) * w, its gradient, and the form whose output
// is stored in 8 bits (e4m3 with one power-of-two scale per 32 columns).
//
// All three are bound by HBM: forward reads x, r and writes s, y once (the row stays in registers between the sum of
// squares and the scaling), backward reads s, dy, ds and writes dx once.  LPR lanes share a row; a lane owns NV vectors
// of VEC consecutive columns (16 bytes when the rows allow it, single columns otherwise), so LPR * NV * VEC >= d.
// Sums are fp32 in a fixed order (lane, then a butterfly over the lanes, then over the waves): no atomics.
// Measured, us (a copy of 1 GiB: 5.1 TB/s): 102,400 x 64 fp32 forward 22.6 (4.7 TB/s), backward 19.2 + 4.2 for the column sums
// (its operands partly from cache); 16,384 x 4096 bf16 forward 92 (5.8 TB/s), backward 112 + 6 (4.8 TB/s, 17 MB of partials
// included: 4 blocks a compute unit keep them few); 8191 x 1000 fp32 into 8 bits 22.9 (4.7 TB/s); 1024 x 64: 3.3 and 5.7,
// 1 x 4096 into 8 bits 4.3: the launch.
// Rows whose width is no multiple of the vector go column by column: 8191 x 1001 bf16 forward 23.5, into 8 bits 35.7 (1000 columns:
// 12.5, 16.1).  Wide rows spill registers: backward past 16,384 columns (102 fp32, 103 bf16; 1024 x 32,768 278 and 254 us, 1.9 and
// 1.1 TB/s; forward, which does not, 111 and 60), and the single-column 8-bit form past 8192 (713 fp32, 2696 bf16: 1024 x 20,001
// 882 and 2560 us, against 104 and 62 at 20,000 columns).
#include "hmx_common.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxD = 32768;
// Up to this many rows the backward pass is one launch, whose blocks for dscale read s and dy again.  One launch / two, us, fp32:
// 256 x 64 4.5 / 5.1, 1024 x 64 4.8 / 5.8, 2048 x 64 6.7 / 5.6, 4096 x 64 16.3 / 5.8; 1024 x 1024 9.6 / 12.3, 2048 x 1024 15.2 / 14.1;
// 256 x 8192 13.5 / 12.2, 1024 x 8192 47.9 / 41.6, 2048 x 8192 89 / 65.  The border is where a step of few kernels gains the most: there
// the host's time counts, and a launch and a buffer less with it.
constexpr int64_t kFewRows = 2048;
constexpr int kBwdBlocks = 1024;      // rows of weight-gradient partials at most (4 blocks per CU)

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
    static __device__ __forceinline__ float round(float v) { return v; }
};
template <>
struct Elem<__bf16> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float load(const __bf16* p) { return (float)*p; }
    static __device__ __forceinline__ void store(__bf16* p, float v) { *p = (__bf16)v; }
    static __device__ __forceinline__ float round(float v) { return (float)(__bf16)v; }
};

// VEC consecutive elements at p (16-byte aligned when VEC > 1) as fp32 and back (one rounding per element).
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = Elem<T>::load(p);
    } else if constexpr (sizeof(T) == 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i];
    } else {
        const f32x8 a = __builtin_convertvector(*reinterpret_cast<const bf16x8*>(p), f32x8);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = a[i];
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        Elem<T>::store(p, v[0]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
        const f32x8 a = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
        *reinterpret_cast<bf16x8*>(p) = __builtin_convertvector(a, bf16x8);
    }
}
// fp32 weights: 16-byte aligned when VEC > 1
template <int VEC>
__device__ __forceinline__ void load_weight(const float* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = *p;
    } else {
#pragma unroll
        for (int q = 0; q < VEC / 4; ++q) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p + 4 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * q + i] = a[i];
        }
    }
}

// Sum over the LPR lanes that share a row, in every one of them.  LPR > 64: the block is one row; `red` holds one float
// per wave and may be reused after the next call's first barrier.
template <int LPR, typename S>
__device__ __forceinline__ S row_sum(S v, S* red) {
#pragma unroll
    for (int off = (LPR < 64 ? LPR : 64) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
    if constexpr (LPR > 64) {
        __syncthreads();                                   // the previous row's sums have been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < LPR / 64; ++i) v += red[i];
    }
    return v;
}

// fp64 to fp32 so that a later rounding to fewer bits comes out as if it were the only one: cut, and the last bit set where
// anything was cut off.  fp32 stays as it is.
__device__ __forceinline__ float round_to_odd(float v) { return v; }
__device__ __forceinline__ float round_to_odd(double v) {
    const float f = (float)v;
    uint32_t u = __float_as_uint(f);
    if ((double)f == v || f != f) return f;
    if (fabs((double)f) > fabs(v)) --u;                                // rounded away from zero (to infinity: the largest number)
    return __uint_as_float(u | 1);
}

// Least e with amax <= 448 * 2^e, -126 <= e <= 127 (0 for a block of zeros); 128 marks a block that is not finite.
__device__ __forceinline__ int mx8_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    if (u >= 0x7f800000u) return 128;
    if (u == 0) return 0;
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);     // 448 = 1.75 * 2^8
    return max(e, -126);
}

template <typename T, int VEC, int LPR, int NV, bool MX8>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void add_rmsnorm_fwd_kernel(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ r, int64_t ldr, const float* __restrict__ w, int64_t T_rows,
    int d, double eps, T* __restrict__ s, T* __restrict__ y, float* __restrict__ rstd, uint8_t* __restrict__ codes,
    uint8_t* __restrict__ scales, int dp) {
    constexpr int kRows = (LPR > 256 ? LPR : 256) / LPR;
    __shared__ typename std::conditional<MX8, double, float>::type red[LPR > 64 ? LPR / 64 : 1];
    const int l = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < T_rows; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = row0 + slot;
        const bool ok = row < T_rows;
        float sv[NV][VEC];
        // the 8-bit form rounds coarsely, and an error of y next to a rounding border becomes a whole step of it: statistics
        // and y are fp64 there (a tenth of the time that the row's bytes take)
        using Sum = typename std::conditional<MX8, double, float>::type;
        Sum ss = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + LPR * i) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sv[i][e] = 0.f;
            if (ok && c < d) {
                load_vec<T, VEC>(x + row * ldx + c, sv[i]);
                if (r) {
                    float rv[VEC];
                    load_vec<T, VEC>(r + row * ldr + c, rv);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) sv[i][e] = Elem<T>::round(sv[i][e] + rv[e]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) ss = fma((Sum)sv[i][e], (Sum)sv[i][e], ss);
        ss = row_sum<LPR>(ss, red);
        const Sum inv = (Sum)1 / sqrt(ss / (Sum)d + (Sum)eps);
        if (ok && rstd && l == 0) rstd[row] = inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + LPR * i) * VEC;
            float yv[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) yv[e] = 0.f;
            if (ok && c < d) {
                float wv[VEC];
                load_weight<VEC>(w + c, wv);
                if (s) store_vec<T, VEC>(s + row * d + c, sv[i]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) yv[e] = round_to_odd((Sum)sv[i][e] * inv * (Sum)wv[e]);
                if constexpr (!MX8) store_vec<T, VEC>(y + row * d + c, yv);
            }
            if constexpr (MX8) {
                // a block of 32 columns lies in 32 / VEC neighbouring lanes; lanes past d hold zeros
                float amax = 0.f;
                bool nan = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    amax = fmaxf(amax, fabsf(yv[e]));
                    nan |= yv[e] != yv[e];
                }
                if (nan) amax = __uint_as_float(0x7f800000u);          // fmaxf drops NaN
#pragma unroll
                for (int off = 16 / VEC; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
                const int ex = mx8_exponent(amax);
                if (ok && c < dp) {
                    const int64_t at = row * dp + c;
                    if ((c & 31) == 0) scales[row * (dp / 32) + c / 32] = (uint8_t)(ex + 127);
                    const int shift = ex == 128 ? 0 : -ex;
                    if constexpr (VEC == 1) {
                        const float v = ex == 128 ? 0.f : ldexpf(yv[0], shift);
                        codes[at] = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 255);
                    } else {
                        uint32_t word[VEC / 4];
#pragma unroll
                        for (int q = 0; q < VEC / 4; ++q) {
                            float v[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = ex == 128 ? 0.f : ldexpf(yv[4 * q + e], shift);
                            int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
                            p = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], p, true);
                            word[q] = (uint32_t)p;
                        }
                        if constexpr (VEC == 4)
                            *reinterpret_cast<uint32_t*>(codes + at) = word[0];
                        else
                            *reinterpret_cast<uint2*>(codes + at) = make_uint2(word[0], word[1]);
                    }
                }
            }
        }
    }
}

// g = dy * w;  dx = ds + rstd * (g - s rstd^2 mean(g s));  dw[c] = sum over rows dy s rstd.
// Blocks below row_blocks take rows.  dw: long inputs, each of them leaves a row of partials in dw_part (summed by a second
// launch); few rows (dw), one more block for each 16 columns reads them all once more, out of cache: a call of that size
// costs what its launches and buffers cost the host.
template <typename T, int VEC, int LPR, int NV>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void add_rmsnorm_bwd_kernel(
    const T* __restrict__ s, const float* __restrict__ w, const float* __restrict__ rstd, const T* __restrict__ dy,
    const T* __restrict__ ds, int64_t T_rows, int d, T* __restrict__ dx, float* __restrict__ dw_part, float* __restrict__ dw_all,
    int row_blocks) {
    constexpr int kThreads = LPR > 256 ? LPR : 256, kRows = kThreads / LPR;
    __shared__ float red[LPR > 64 ? LPR / 64 : 1];
    __shared__ float dws[kThreads * (kRows > 1 ? VEC : 1)];
    const int l = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    if ((int)blockIdx.x >= row_blocks) {
        const int c = ((int)blockIdx.x - row_blocks) * 16 + (int)(threadIdx.x & 15);
        float a = 0.f;
        if (c < d) {
#pragma unroll 8
            for (int64_t row = threadIdx.x >> 4; row < T_rows; row += kThreads / 16)
                a = fmaf(Elem<T>::load(dy + row * d + c), Elem<T>::load(s + row * d + c) * rstd[row], a);
        }
        dws[threadIdx.x] = a;
        __syncthreads();
        if (threadIdx.x < 16 && c < d) {
            a = 0.f;
            for (int q = 0; q < kThreads / 16; ++q) a += dws[q * 16 + threadIdx.x];
            dw_all[c] = a;
        }
        return;
    }
    float dw[NV][VEC], wv[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (l + LPR * i) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[i][e] = wv[i][e] = 0.f;
        if (c < d) load_weight<VEC>(w + c, wv[i]);
    }
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < T_rows; row0 += (int64_t)row_blocks * kRows) {
        const int64_t row = row0 + slot;
        const bool ok = row < T_rows;
        float sv[NV][VEC], gv[NV][VEC];
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + LPR * i) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sv[i][e] = gv[i][e] = 0.f;
            if (ok && c < d) {
                load_vec<T, VEC>(s + row * d + c, sv[i]);
                load_vec<T, VEC>(dy + row * d + c, gv[i]);
            }
        }
        const float inv = ok ? rstd[row] : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                dw[i][e] = fmaf(gv[i][e], sv[i][e] * inv, dw[i][e]);
                gv[i][e] *= wv[i][e];
                dot = fmaf(gv[i][e], sv[i][e], dot);
            }
        dot = row_sum<LPR>(dot, red);
        const float k = dot / (float)d * inv * inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + LPR * i) * VEC;
            if (ok && c < d) {
                float o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] = inv * (gv[i][e] - sv[i][e] * k);
                if (ds) {
                    float a[VEC];
                    load_vec<T, VEC>(ds + row * d + c, a);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) o[e] += a[e];
                }
                store_vec<T, VEC>(dx + row * d + c, o);
            }
        }
    }
    if (!dw_part) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (l + LPR * i) * VEC;
        if constexpr (kRows > 1) {                         // the block's row slots, added in slot order
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VEC; ++e) dws[threadIdx.x * VEC + e] = dw[i][e];
            __syncthreads();
            if (slot == 0 && c < d) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    float a = 0.f;
                    for (int q = 0; q < kRows; ++q) a += dws[(q * LPR + l) * VEC + e];
                    dw_part[(int64_t)blockIdx.x * d + c + e] = a;
                }
            }
        } else if (c < d) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) dw_part[(int64_t)blockIdx.x * d + c + e] = dw[i][e];
        }
    }
}

// Blocks of the backward pass, each with a row of weight-gradient partials (none: no rows).
int64_t bwd_blocks(int64_t T, int64_t d) {
    return std::min<int64_t>(std::min<int64_t>(T, hmx_ceil_div(T * std::min<int64_t>(d, 1024), 1024)), kBwdBlocks);
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

struct FwdArgs {
    const void *x, *r;
    int64_t ldx, ldr;
    const float* w;
    int64_t T;
    int d;
    double eps;
    void *s, *y;
    float* rstd;
    uint8_t *codes, *scales;
    int dp;
};

template <typename T, int VEC, int LPR, int NV, bool MX8>
void launch_fwd(const FwdArgs& a, hipStream_t st) {
    constexpr int kThreads = LPR > 256 ? LPR : 256, kRows = kThreads / LPR;
    const int grid = (int)std::min<int64_t>(hmx_ceil_div(a.T, kRows), 1 << 20);
    hipLaunchKernelGGL((add_rmsnorm_fwd_kernel<T, VEC, LPR, NV, MX8>), dim3(grid), dim3(kThreads), 0, st, (const T*)a.x, a.ldx,
                       (const T*)a.r, a.ldr, a.w, a.T, a.d, a.eps, (T*)a.s, (T*)a.y, a.rstd, a.codes, a.scales, a.dp);
}

// The row's vectors over the fewest lanes that keep NV <= 2 (<= 4 on a wave: a wave needs no barrier), so that a lane has
// independent loads in flight; wider rows take the block, then NV up to what kMaxD needs.
#define HMX_NORM_WIDTHS(CALL)                                      \
    if (nvec <= 16) { CALL(16, 1); }                               \
    else if (nvec <= 32) { CALL(16, 2); }                          \
    else if (nvec <= 64) { CALL(64, 1); }                          \
    else if (nvec <= 128) { CALL(64, 2); }                         \
    else if (nvec <= 256) { CALL(64, 4); }                         \
    else if (nvec <= 512) { CALL(256, 2); }                        \
    else if (nvec <= 1024) { CALL(256, 4); }                       \
    else if (nvec <= 2048) { CALL(1024, 2); }                      \
    else if (nvec <= 4096) { CALL(1024, 4); }                      \
    else if (nvec <= 8192) { CALL(1024, 8); }                      \
    else { CALL(1024, 32); }

template <typename T, bool MX8>
int dispatch_fwd(const FwdArgs& a, hipStream_t st) {
    constexpr int V = Elem<T>::kVec;
    const int width = MX8 ? a.dp : a.d;
    const bool vec = a.d % V == 0 && a.ldx % V == 0 && a.ldr % V == 0 && aligned(a.x, 16) && (!a.r || aligned(a.r, 16)) &&
                     aligned(a.w, 16) && aligned(a.s, 16) && aligned(a.y, 16) && aligned(a.codes, 8);
    if (vec) {
        const int nvec = width / V;
#define CALL(LPR, NV)                                                              \
    if constexpr (LPR * NV <= kMaxD / V) launch_fwd<T, V, LPR, NV, MX8>(a, st)
        HMX_NORM_WIDTHS(CALL)
#undef CALL
    } else if constexpr (MX8) {
        // single columns: a block of 32 needs 32 neighbouring lanes
        const int nvec = width;
#define CALL(LPR, NV) launch_fwd<T, 1, (LPR < 64 ? 64 : LPR), NV, MX8>(a, st)
        HMX_NORM_WIDTHS(CALL)
#undef CALL
    } else {
        const int nvec = width;
#define CALL(LPR, NV) launch_fwd<T, 1, LPR, NV, MX8>(a, st)
        HMX_NORM_WIDTHS(CALL)
#undef CALL
    }
    HMX_CHECK_LAUNCH();
    return HMX_OK;
}

struct BwdArgs {
    const void *s, *dy, *ds;
    const float *w, *rstd;
    int64_t T;
    int d;
    void* dx;
    float *part, *dw;
};

template <typename T, int VEC, int LPR, int NV>
void launch_bwd(const BwdArgs& a, hipStream_t st) {
    constexpr int kThreads = LPR > 256 ? LPR : 256;
    const int rows = (int)bwd_blocks(a.T, a.d), more = a.dw ? (int)hmx_ceil_div(a.d, 16) : 0;
    hipLaunchKernelGGL((add_rmsnorm_bwd_kernel<T, VEC, LPR, NV>), dim3(rows + more), dim3(kThreads), 0, st, (const T*)a.s, a.w, a.rstd,
                       (const T*)a.dy, (const T*)a.ds, a.T, a.d, (T*)a.dx, a.part, a.dw, rows);
}

template <typename T>
int dispatch_bwd(const BwdArgs& a, hipStream_t st) {
    constexpr int V = Elem<T>::kVec;
    const bool vec = a.d % V == 0 && aligned(a.s, 16) && aligned(a.dy, 16) && (!a.ds || aligned(a.ds, 16)) &&
                     aligned(a.w, 16) && aligned(a.dx, 16);
    if (vec) {
        const int nvec = a.d / V;
#define CALL(LPR, NV)                                                              \
    if constexpr (LPR * NV <= kMaxD / V) launch_bwd<T, V, LPR, NV>(a, st)
        HMX_NORM_WIDTHS(CALL)
#undef CALL
    } else {
        const int nvec = a.d;
#define CALL(LPR, NV) launch_bwd<T, 1, LPR, NV>(a, st)
        HMX_NORM_WIDTHS(CALL)
#undef CALL
    }
    HMX_CHECK_LAUNCH();
    return HMX_OK;
}

bool bad_rows(int64_t T, int64_t d) { return T < 0 || d <= 0 || d > kMaxD; }

}  // namespace

// ================================================================================ C ABI
extern "C" int hmx_add_rmsnorm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* scale, int64_t T,
                                   int64_t d, double eps, int bf16, void* s, void* y, float* rstd, void* stream) {
    HMX_ENTER();
    if (bad_rows(T, d) || !(eps >= 0.0)) return HMX_EINVAL;
    if (T == 0) return HMX_OK;
    if (!x || !scale || !y || (residual && !s) || ldx < 0 || ldr < 0) return HMX_EINVAL;
    const FwdArgs a = {x, residual, ldx, residual ? ldr : 0, scale, T, (int)d, eps, s, y, rstd, nullptr, nullptr, 0};
    return bf16 ? dispatch_fwd<__bf16, false>(a, (hipStream_t)stream) : dispatch_fwd<float, false>(a, (hipStream_t)stream);
}

extern "C" int hmx_add_rmsnorm_mx8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* scale, int64_t T,
                                   int64_t d, double eps, int bf16, void* s, void* codes, void* scales, void* stream) {
    HMX_ENTER();
    if (bad_rows(T, d) || !(eps >= 0.0)) return HMX_EINVAL;
    if (T == 0) return HMX_OK;
    if (!x || !scale || !codes || !scales || (residual && !s) || ldx < 0 || ldr < 0) return HMX_EINVAL;
    const FwdArgs a = {x, residual, ldx, residual ? ldr : 0, scale, T, (int)d, eps, s, nullptr, nullptr, (uint8_t*)codes,
                       (uint8_t*)scales, (int)hmx_ceil_div(d, 32) * 32};
    return bf16 ? dispatch_fwd<__bf16, true>(a, (hipStream_t)stream) : dispatch_fwd<float, true>(a, (hipStream_t)stream);
}

extern "C" size_t hmx_add_rmsnorm_bwd_workspace_bytes(int64_t T, int64_t d) {
    if (T <= kFewRows || d <= 0) return 0;
    const int64_t blocks = bwd_blocks(T, d);
    return hmx_align_up((size_t)blocks * d * sizeof(float), 256) + hmx_colsum_workspace_bytes(blocks, d);
}

extern "C" int hmx_add_rmsnorm_bwd(const void* s, const float* scale, const float* rstd, const void* dy, const void* ds, int64_t T,
                                   int64_t d, int bf16, void* dx, float* dscale, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    HMX_ENTER();
    if (bad_rows(T, d)) return HMX_EINVAL;
    if (T > 0 && (!s || !scale || !rstd || !dy || !dx)) return HMX_EINVAL;
    const size_t need = hmx_add_rmsnorm_bwd_workspace_bytes(T, d);
    if (dscale && need > 0 && (!workspace || workspace_bytes < need)) return HMX_EWORKSPACE;
    const hipStream_t st = (hipStream_t)stream;
    if (T == 0) return dscale ? hmx_colsum_f32(nullptr, 0, d, d, dscale, nullptr, 0, stream) : HMX_OK;       // zeros
    HmxCarver carve(workspace);
    const int64_t blocks = bwd_blocks(T, d);
    float* part = dscale && need > 0 ? carve.take<float>((size_t)(blocks * d)) : nullptr;
    const BwdArgs a = {s, dy, ds, scale, rstd, T, (int)d, dx, part, part ? nullptr : dscale};
    const int rc = bf16 ? dispatch_bwd<__bf16>(a, st) : dispatch_bwd<float>(a, st);
    if (rc != HMX_OK || !part) return rc;
    const size_t left = hmx_colsum_workspace_bytes(blocks, d);
    return hmx_colsum_f32(part, blocks, d, d, dscale, left ? carve.take<char>(left) : nullptr, left, stream);
}
