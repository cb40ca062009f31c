// Sampling from rows of scores with temperature, top-k, top-p and min-p, from given uniform numbers.
//
// w_i = exp((l_i - max l) / T).  Kept are the top_k first by (l descending, i ascending); of these the shortest prefix of
// that order whose mass is at least top_p of theirs; of these the ones with w_i >= min_p.  A draw is the first kept i in
// INDEX order whose running sum of w passes u * (kept mass): no sort of the row is needed, only the border of the kept set.
//
// Weights are fp64 (z exactly as far as fp64 goes, exp by table and polynomial, 1e-15) turned into integers w * 2^s, with s
// the largest scale at which the row's mass is sure to fit 62 bits (51 at most): integer sums do not depend on their order,
// so LDS and global atomics and any number of waves give the same set and the same draw on every run.  (How a row is worked on,
// by its length and the number of rows, sets the bound on its mass and so the scale: one rounding of a weight.)
//
// What bounds it: at four cycles a wave an instruction per element costs 0.9 us for 33.5 M elements on the whole card, so the
// few instructions that every element meets come first, the 25 of a weight where they can be spared:
//   bfloat16: one look counts the 16-bit values (8192 counters for 2^-22 <= |l| < 2^10, a list for the rest), which gives
//     every border exactly: a value and how many of its elements are kept.
//   fp32, top_k: the k-th largest of the maxima of groups of elements is a value that at least k elements reach; what
//     reaches it is gathered into a list, and the list does the rest (top_p and min_p on top of top_k included).
//   fp32, top_p: masses of 4096 bins of equal width in l.  What lies so far below the maximum that V of it weigh less than
//     half of 1 - top_p is summed without a bin.
//   Then one look at the row sums, tile by tile of 1024 elements or more, the weights above the border, counts the elements
//   at the border value (or gathers the border bin's few), and the draws go by the tiles' running sums.
//   Where a list overflows (equal scores, scores that differ in their last bits): counts or masses of equal ranges of the
//   ordered 32-bit key, three looks at most, until a range is one key.
// One block does a row on its own; few long rows are cut into segments for the looks at all elements, with one block a row
// between them.
// Measured, us: 256 x 131,072 bf16 44.6 in one launch: start and cleared counters 2.9, the count of values 12, the border from 8192
// counters 10, the tiles 14.7, the draws 5.1 (67 MB once at 5.1 TB/s: 13); 4 x 4,000,001 fp32, top_k 1000 and 16 draws 44: maxima
// 12, plan 6, gather 13, list and draws 13; 1 x 50,000 fp32, top_k 50: 12.
#include "hmx_common.h"

#include <algorithm>

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 4096;                // bins, tiles and list entries: four per thread
constexpr int kPer = kBins / kThreads;
constexpr int kTile = 1024;                // elements of a tile at least: one step of a wave
constexpr int kSmall = 2048;               // rows up to this length go into the list whole
constexpr int kMaxSplit = 64;              // blocks a row is cut over at most (64 groups of each have their maximum)
constexpr uint32_t kLowestKey = 0x00800000u;        // the key after that of -infinity
constexpr float kMaxFloat = 3.402823466e38f;
constexpr float kRange = 32.f;             // bins reach down to exp(-32) of the largest weight
constexpr uint32_t kFirstMag = (127 - 22) << 7;     // bfloat16 magnitudes with a counter: 2^-22 up to 2^10
constexpr int kValues = 2 * 4096, kPerValue = kValues / kThreads;

typedef unsigned long long u64;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

struct SampleArgs {
    const void* logits;
    int64_t ld;
    uint32_t V;
    const void* u;
    int u64bit, draws;
    const float *temperature, *top_p, *min_p;       // per row, or null: the numbers below
    const int32_t* top_k;
    double t, p, mp;
    int64_t k;
    int64_t* ids;
    float* probs;
    uint32_t tile;                                   // elements of a tile, a multiple of kTile
};

// ------------------------------------------------------------------------------- elements
__device__ __forceinline__ uint32_t key_of(float l) {               // ascending in l; -0 counts as +0
    const uint32_t u = __float_as_uint(l + 0.f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ bool candidate(float l) { return l > -__builtin_inff(); }      // neither -infinity nor NaN

// Four consecutive elements as they lie in memory (rows start anywhere: the loads need only the type's own alignment), and
// their values.  Kept apart so that a load can be in flight while earlier elements are used.
template <typename T>
struct Raw;
template <>
struct Raw<float> {
    f32x4 v;
    __device__ __forceinline__ void load(const float* p) { __builtin_memcpy(&v, p, 16); }
    __device__ __forceinline__ float get(int e) const { return v[e]; }
    __device__ __forceinline__ void drop(int e) { v[e] = __builtin_nanf(""); }
};
template <>
struct Raw<__bf16> {
    uint2 v;
    __device__ __forceinline__ void load(const __bf16* p) { __builtin_memcpy(&v, p, 8); }
    __device__ __forceinline__ float get(int e) const {
        const uint32_t w = e < 2 ? v.x : v.y;
        return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
    __device__ __forceinline__ void drop(int e) { (e < 2 ? v.x : v.y) |= e & 1 ? 0x7fff0000u : 0x7fffu; }
};

// f(Raw of four elements, index of the first) for the elements of [lo, hi), hi >= 4, by `threads` threads (all of them take
// part in every step; elements outside are NaN), DEPTH steps' loads in flight.  The loop is unrolled over these, since a load's
// register must not be moved while it is awaited, and every step has its load, also past the end (of the last four): the
// compiler counts the loads to wait for, and one that may be missing makes it wait for all.
template <int DEPTH, typename T, typename F>
__device__ __forceinline__ void each_raw(const T* row, uint32_t lo, uint32_t hi, int thread, int threads, F f) {
    const uint32_t stride = threads * 4, steps = (hi - lo + stride - 1) / stride, last = hi - 4;
    uint32_t i = lo + thread * 4;
    Raw<T> ahead[DEPTH];
#pragma unroll
    for (int q = 0; q < DEPTH; ++q) ahead[q].load(row + std::min(i + q * stride, last));
#pragma unroll 1
    for (uint32_t n = 0; n < steps; n += DEPTH) {
#pragma unroll
        for (int q = 0; q < DEPTH; ++q) {
            if (n + q >= steps) break;
            Raw<T> x = ahead[q];
            ahead[q].load(row + std::min(i + DEPTH * stride, last));
            uint32_t first = i;
            if (n + q + 1 == steps) {               // past the end: the row's last four, without what came before
                first = std::min(i, last);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (first + e < i) x.drop(e);
            }
            f(x, first);
            i += stride;
        }
    }
}

// f(four values, index of the first)
template <int DEPTH, typename T, typename F>
__device__ __forceinline__ void each_element(const T* row, uint32_t lo, uint32_t hi, int thread, int threads, F f) {
    each_raw<DEPTH>(row, lo, hi, thread, threads, [&](const Raw<T>& x, uint32_t first) {
        const float l[4] = {x.get(0), x.get(1), x.get(2), x.get(3)};
        f(l, first);
    });
}

// ------------------------------------------------------------------------------- weights
// What a row's weights and bins are computed with.
struct Row {
    uint32_t top;                   // key of the maximum
    float lmax_f, bin_scale;        // the maximum (at most the largest finite number), bins per unit of l
    int scale;                      // units are 2^-scale
    double lmax;                    // the maximum (1e300 for infinity: all that is finite is nothing beside it)
    double inv_t, step;             // step: 128 / (T ln 2)
    double log_min_p;               // -infinity: off
    double cut;                     // steps at which a weight is a quarter of a unit
    double p;                       // 1: off
    int64_t k;                      // 0: off
};

// Ascending as l falls, kBins: all that lies lower (and -infinity).  NaN: any of them.
__device__ __forceinline__ int bin_of(const Row& r, float l) {
    return (int)__builtin_amdgcn_fmed3f((r.lmax_f - l) * r.bin_scale, 0.f, (float)kBins);
}
__device__ __forceinline__ double log_weight(const Row& r, float l) { return ((double)l - r.lmax) * r.inv_t; }

// exp((l - max) / T) in units of 2^-scale (2^51 at most; 1/4 where it is less), and that rounded to an integer; 0 for
// -infinity and NaN.  With n + x = 128 z / ln 2, |x| <= 1/2 and n = 128 q + i: 2^q * 2^(i / 128) * e^(x ln2 / 128), the last by
// four terms after 1 (what they leave off: 1e-15), the second from the table.  Adding 1.5 * 2^52 rounds to n and leaves its
// bits; 2^q goes into the exponent, which stays in range because of the cut.
__device__ __forceinline__ double weight_units(const Row& r, float l, const double* tab) {
    const double y = fmin(fmax(((double)l - r.lmax) * r.step, r.cut), 0.0);      // fmax drops NaN
    const double shifted = y + 6755399441055744.0;
    const int n = (int)(uint32_t)__double_as_longlong(shifted);
    const double x = y - (shifted - 6755399441055744.0);
    double e = fma(x, 3.583032305400251e-11, 2.646642144433097e-08);                 // (ln2 / 128)^k / k!
    e = fma(x, e, 1.4662262387640425e-05);
    e = fma(x, e, 0.0054152123481245725);
    e = fma(x, e, 1.0);
    const double m = tab[n & 127] * e;
    return __longlong_as_double(__double_as_longlong(m) + ((long long)((n >> 7) + r.scale) << 52));
}
__device__ __forceinline__ u64 weight(const Row& r, float l, const double* tab) {
    return __double_as_longlong(weight_units(r, l, tab) + 4503599627370496.0) & 0xfffffffffffffull;
}
__device__ __forceinline__ bool passes(const Row& r, float l) { return log_weight(r, l) >= r.log_min_p; }

__device__ __forceinline__ u64 share_of(double p, u64 total) {
    const u64 t = (u64)ceil((p > 0.0 ? p : 0.0) * (double)total);
    return t < 1 ? 1 : t > total ? total : t;
}

__device__ __forceinline__ Row settings(const SampleArgs& a, int64_t b) {
    double t = a.temperature ? (double)a.temperature[b] : a.t;
    const double p = a.top_p ? (double)a.top_p[b] : a.p, mp = a.min_p ? (double)a.min_p[b] : a.mp;
    Row r;
    r.k = a.top_k ? a.top_k[b] : a.k;
    if (!(t > 0.0) || t == __builtin_inf()) t = 1.0, r.k = 1;
    // two fp32 scores lie 2^-149 apart at least and 2^129 at most: below 1e-60 all but the ones equal to the maximum weigh
    // nothing, above 1e60 all finite ones weigh the same to the last bit.  Within, 128 / (T ln 2) is finite (times 0, for the
    // maximum itself, infinity would be NaN) and an infinite maximum's 1e300 still leaves the others nothing.
    t = fmin(fmax(t, 1e-60), 1e60);
    if (r.k < 0 || r.k >= a.V) r.k = 0;
    r.p = p < 1.0 ? p : 1.0;
    r.inv_t = 1.0 / t;
    r.log_min_p = -__builtin_inf();
    if (mp > 0.0) r.log_min_p = log(mp < 1.0 ? mp : 1.0);
    r.step = 184.6649652337873 * r.inv_t;                            // 128 / ln 2
    r.top = 0;
    r.lmax_f = r.bin_scale = 0.f;
    r.lmax = r.cut = 0.0;
    r.scale = 0;
    return r;
}

// The maximum, and the scale: the row's mass, at most `most` times the largest weight, has to fit 62 bits.
__device__ __forceinline__ void set_scale(Row& r, float lmax, float most) {
    const bool finite = lmax <= kMaxFloat;
    r.top = key_of(lmax);
    r.lmax_f = finite ? lmax : kMaxFloat;
    r.lmax = finite ? (double)lmax : 1e300;
    const int ex = (int)((__float_as_uint(most) >> 23) & 255) - 126;  // most < 2^ex
    r.scale = min(51, 62 - ex);
    r.cut = -128.0 * (double)(r.scale + 2);
}
// exp((l - top) / T) in fp32, for bounds of a row's mass, with `by` = rough_by(r).  Halves, since finite scores may lie further
// apart than the largest number; an infinite top leaves the others some weight where T is near it too: more is no harm.
__device__ __forceinline__ float rough_by(const Row& r) { return fminf((float)(2.8853900817779268 * r.inv_t), kMaxFloat); }      // 2 / ln 2
__device__ __forceinline__ float rough_weight(float l, float top, float by) {
    return l == top ? 1.f : __builtin_amdgcn_exp2f(fmaxf(0.5f * l - 0.5f * top, -kMaxFloat) * by);
}
__device__ __forceinline__ void set_bins(Row& r, float range) {
    r.bin_scale = fminf((float)((double)kBins * r.inv_t) / range, kMaxFloat);
}
// For top_p: V elements below the bins' range weigh less than half of what top_p leaves out of a mass of at least `least`.
__device__ __forceinline__ float range_for(const Row& r, uint32_t V, float least) {
    const float out = (float)(1.0 - r.p) * least * 0.75f;
    const float down = 0.6931472f * __builtin_amdgcn_logf(2.f * (float)V / out);
    return out > 0.f && down < kRange ? fmaxf(down, 0.125f) : kRange;
}
// Whether the k-th largest of `groups` maxima leads to a list: groups * ln(groups / (groups - k)) elements reach it where the
// groups are alike, 1650 of 1024 groups, 2750 of 4096 at most.
__host__ __device__ inline bool by_maxima(int64_t k, int groups) { return k > 0 && 5 * k <= 4 * groups && k <= 2000; }

// ------------------------------------------------------------------------------- block sums
// v of the lane that the DPP control names; 0 where there is none, or where the row mask leaves the lane out.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp64(u64 v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, ROWS == 0xf);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, ROWS == 0xf);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 row_incl(u64 v) {                     // inclusive sums in rows of 16 lanes
    v += dpp64<0x111, 0xf>(v);                                       // shift right by 1, 2, 4, 8 in a row
    v += dpp64<0x112, 0xf>(v);
    v += dpp64<0x114, 0xf>(v);
    v += dpp64<0x118, 0xf>(v);
    return v;
}
__device__ __forceinline__ u64 wave_incl(u64 v) {                    // all lanes active
    v = row_incl(v);
    v += dpp64<0x142, 0xa>(v);                                       // lane 15 of rows 0 and 2 to rows 1 and 3
    v += dpp64<0x143, 0xc>(v);                                       // lane 31 to rows 2 and 3
    return v;
}
__device__ __forceinline__ u64 lane64(u64 v, int lane) {
    return ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

// How far a row has come (Mode names what the next look at its elements has to do).
enum Mode : int { kDone, kGather, kBinning, kTiles, kAlone };
struct State {
    Row r;
    int mode;
    uint32_t klo, khi;              // gather: from klo on; tiles: weights above khi, klo to khi apart
    int ties;                       // tiles: 1 = klo == khi and `need` of that key's elements are kept, 0 = the list has them
    u64 need;                       // elements of the border key, or units of the border bin's mass
};

constexpr int kLine = 96;            // fours in a wave's queue: a full load of 64 and as many as may come too many
struct Line {
    f32x4 four[kLine];
    uint32_t t[kLine];
};
struct Shared {
    double tab[128];
    union {
        u64 bins[kBins];
        uint32_t count[kValues];
        u64 tile[kBins];
    };
    union {
        u64 list[kBins];
        float group[kBins];
    };
    uint32_t ties[kBins];
    Line queue[kWaves];
    State st;
    u64 wsum[kWaves], wsums[4][kWaves];
    float wmax[kWaves];
    u64 above;
    uint32_t bin, n_list, at;
};

template <typename SH>
__device__ __forceinline__ void make_table(SH& sh) {
    // 2^(i / 128) from the powers that i's bits stand for: a few roundings, and little code
    const double root[7] = {1.0054299011128027, 1.0108892860517005, 1.0218971486541166, 1.0442737824274138,
                            1.0905077326652577, 1.189207115002721, 1.4142135623730951};
    double v = 1.0;
#pragma unroll
    for (int q = 0; q < 7; ++q) v *= (threadIdx.x >> q) & 1 ? root[q] : 1.0;
    if (threadIdx.x < 128) sh.tab[threadIdx.x] = v;
}

// Inclusive sums over the block in thread order; *total gets the sum of all.
__device__ __forceinline__ u64 block_incl(u64 v, Shared& sh, u64* total) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_incl(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.wsum[wave] = v;
    __syncthreads();
    const u64 sums = row_incl(sh.wsum[threadIdx.x & 15]);            // kWaves = 16: one row of lanes
    *total = lane64(sums, 15);
    return v + (wave ? lane64(sums, wave - 1) : 0);
}
// The block's sums of N values, in every thread.
template <int N>
__device__ __forceinline__ void block_sums(u64 (&v)[N], Shared& sh) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < N; ++q) {
        v[q] = wave_incl(v[q]);
        if ((threadIdx.x & 63) == 63) sh.wsums[q][wave] = v[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = lane64(row_incl(sh.wsums[q][threadIdx.x & 15]), 15);
}
__device__ __forceinline__ float block_max(float v, Shared& sh) {
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wmax[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.wmax[threadIdx.x & 15];
    for (int d = 1; d < 16; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ float block_sum(float v, Shared& sh) {
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wmax[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.wmax[threadIdx.x & 15];
    for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// The place among N values a thread (in thread order) at which their running sum reaches `target` (> 0): sh.bin (N * kThreads
// where they do not), sh.above before it.  `extra` comes before the second half of the values.  SHARE: the target is a share of
// the sum.
template <bool SHARE = false, int N>
__device__ __forceinline__ void find_place(const u64 (&v)[N], u64 target, u64 extra, Shared& sh, double share = 1.0) {
    u64 all, sum = 0;
#pragma unroll
    for (int q = 0; q < N; ++q) sum += v[q];
    u64 upto = block_incl(sum, sh, &all) - sum + (threadIdx.x >= kThreads / 2 ? extra : 0);
    if (SHARE) target = share_of(share, all);
    if (threadIdx.x == 0) sh.bin = N * kThreads, sh.above = all + extra;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < N; ++q) {
        if (upto < target && target <= upto + v[q]) sh.bin = N * threadIdx.x + q, sh.above = upto;
        upto += v[q];
    }
    __syncthreads();
}

// ------------------------------------------------------------------------------- the list
__device__ __forceinline__ u64 entry(uint32_t key, uint32_t i) { return ((u64)key << 32) | (uint32_t)~i; }
__device__ __forceinline__ float entry_value(u64 x) { return value_of((uint32_t)(x >> 32)); }

// Sorts n entries that differ; DESC: the largest first.  Up to 256: each goes to the place that the count of those before it
// names.  More: bitonic; steps of up to 64 stay in a wave's own 128 entries and need no barrier of the block.
template <bool DESC>
__device__ __forceinline__ void sort_list(uint32_t n, u64* list) {
    __syncthreads();
    if (n <= 256) {
        const u64 x = threadIdx.x < n ? list[threadIdx.x] : 0;
        uint32_t place = 0;
        if ((threadIdx.x & ~63u) < n)
            for (uint32_t i = 0; i < n; ++i) place += DESC ? list[i] > x : list[i] < x;
        __syncthreads();
        if (threadIdx.x < n) list[place] = x;
        __syncthreads();
        return;
    }
    uint32_t m = 512;
    while (m < n) m <<= 1;
    for (uint32_t i = n + threadIdx.x; i < m; i += kThreads) list[i] = DESC ? 0 : ~0ull;
    __syncthreads();
#pragma unroll 1
    for (uint32_t size = 2; size <= m; size <<= 1) {
#pragma unroll 1
        for (uint32_t stride = size / 2; stride > 0; stride >>= 1) {
            for (uint32_t t = threadIdx.x; t < m / 2; t += kThreads) {
                const uint32_t i = 2 * t - (t & (stride - 1)), j = i + stride;
                const u64 x = list[i], y = list[j];
                const bool up = ((i & size) != 0) == DESC;
                if (x != y && (x > y) == up) list[i] = y, list[j] = x;
            }
            // a wave's pairs at strides up to 64 are its own: the block meets where the next stride or size needs it
            if (stride > 64 || (stride == 1 && size >= 128)) __syncthreads();
            else {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
    }
    __syncthreads();
}

// sort_list<true> for keys from klo to khi, by way of 4096 ranges of keys (in sh.count): a range's entries go to its place,
// and each to the one that its range's larger entries leave it.  Where many share a range, the bitonic way does it.
__device__ __forceinline__ void sort_by_ranges(uint32_t n, uint32_t klo, uint32_t khi, Shared& sh) {
    if (n <= 256) return sort_list<true>(n, sh.list);
    const int bits = klo == khi ? 0 : 32 - __clz(khi - klo), shift = bits > 12 ? bits - 12 : 0;
    __syncthreads();
    for (int q = 0; q < kPer; ++q) sh.count[q * kThreads + threadIdx.x] = 0;
    __syncthreads();
    u64 x[kPer];
    uint32_t rank[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        const uint32_t i = q * kThreads + threadIdx.x;
        x[q] = i < n ? sh.list[i] : 0;
        if (i < n) rank[q] = atomicAdd(&sh.count[(khi - (uint32_t)(x[q] >> 32)) >> shift], 1u);
    }
    __syncthreads();
    uint32_t c[kPer], most = 0;
    u64 sum = 0, all;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        c[q] = sh.count[kPer * threadIdx.x + q];
        most = std::max(most, c[q]);
        sum += c[q];
    }
    if (__syncthreads_or(most > 64)) return sort_list<true>(n, sh.list);
    uint32_t at = (uint32_t)(block_incl(sum, sh, &all) - sum);
#pragma unroll
    for (int q = 0; q < kPer; ++q) sh.count[kPer * threadIdx.x + q] = at, at += c[q];
    __syncthreads();
    uint32_t first[kPer], end[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        if (q * kThreads + threadIdx.x >= n) continue;
        const uint32_t range = (khi - (uint32_t)(x[q] >> 32)) >> shift;
        first[q] = sh.count[range];
        end[q] = range + 1 < kBins ? sh.count[range + 1] : n;
        sh.list[first[q] + rank[q]] = x[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        if (q * kThreads + threadIdx.x >= n) continue;
        rank[q] = first[q];
        for (uint32_t i = first[q]; i < end[q]; ++i) rank[q] += sh.list[i] > x[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q)
        if (q * kThreads + threadIdx.x < n) sh.list[rank[q]] = x[q];
    __syncthreads();
}

// The place in the list's first n entries (sorted) at which their running mass reaches `target`, or (SHARE) top_p of theirs.
template <bool SHARE>
__device__ __forceinline__ uint32_t place_of_mass(const Row& r, uint32_t n, u64 target, Shared& sh) {
    u64 v[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        const uint32_t i = kPer * threadIdx.x + q;
        v[q] = i < n ? weight(r, entry_value(sh.list[i]), sh.tab) : 0;
    }
    find_place<SHARE>(v, target, 0, sh, r.p);
    return n ? std::min(sh.bin, n - 1) : 0;
}

__device__ __forceinline__ u64 draw_target(const SampleArgs& a, int64_t at, u64 total) {
    const double u = a.u64bit ? ((const double*)a.u)[at] : (double)((const float*)a.u)[at];
    const double t = u > 0.0 ? u * (double)total : 0.0;             // NaN counts as 0
    return t < (double)total ? std::min<u64>((u64)t, total - 1) : total - 1;
}
__device__ __forceinline__ void put_draw(const SampleArgs& a, const Row& r, int64_t at, uint32_t i, float l, u64 total, const double* tab) {
    a.ids[at] = i;
    a.probs[at] = (float)(weight_units(r, l, tab) / (double)total);
}
__device__ __forceinline__ void draw_nothing(const SampleArgs& a, int64_t b) {
    for (int q = threadIdx.x; q < a.draws; q += kThreads) a.ids[b * a.draws + q] = -1, a.probs[b * a.draws + q] = 0.f;
}

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The draw of a tile whose kept elements are few, by the wave, from the list's first n entries: false where they are more than
// 64.  `before`: the weights of earlier tiles.
__device__ __forceinline__ bool draw_from_entries(const SampleArgs& a, const Row& r, uint32_t n, uint32_t from, uint32_t end, u64 before,
                                                  u64 want, int64_t at, u64 total, u64* hits, const Shared& sh) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t m = 0;
    wave_sync();
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {
        const u64 x = sh.list[std::min(i0 + lane, n - 1)];
        const uint32_t i = ~(uint32_t)x;
        const bool in = i0 + lane < n && i >= from && i < end;
        const u64 all = __ballot(in);
        if (!all) continue;
        const uint32_t place = m + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
        if (in && place < 64) hits[place] = x;
        m += __popcll(all);
    }
    wave_sync();
    if (m > 64) return false;
    const u64 x = hits[lane];
    const uint32_t own = ~(uint32_t)x;
    const float l = entry_value(x);
    const u64 w = lane < m && passes(r, l) ? weight(r, l, sh.tab) : 0;
    u64 sum = before;                                                // of the elements before the lane's own
    for (uint32_t q = 0; q < m; ++q) {
        const uint32_t other = __builtin_amdgcn_readlane((int)own, q);
        const u64 one = lane64(w, q);
        sum += other < own ? one : 0;
    }
    const bool hit = w != 0 && sum <= want && want < sum + w;
    if (hit) put_draw(a, r, at, own, l, total, sh.tab);
    return __any(hit);
}

// The draws by the tiles' sums (sh.tile): the kept elements are the entries from `last` on that pass min_p; where `listed` is
// not 0, they are among the list's first `listed` entries.  One wave a draw finds the tile by running sums, then the element:
// among the list's entries where a tile has few of them (no read of the row: 7 -> 3 us), or with 1024 elements' loads at once.
template <typename T>
__device__ __forceinline__ void draw_by_tiles(const SampleArgs& a, const T* row, const Row& r, u64 last, uint32_t listed, int64_t b, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t tiles = (a.V + a.tile - 1) / a.tile;
    u64 w[kPer], sum = 0, total;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        const uint32_t t = kPer * threadIdx.x + q;
        w[q] = t < tiles ? sh.tile[t] : 0;
        sum += w[q];
    }
    u64 upto = block_incl(sum, sh, &total) - sum;
#pragma unroll
    for (int q = 0; q < kPer; ++q) upto += w[q], sh.tile[kPer * threadIdx.x + q] = upto;
    __syncthreads();
    for (int q = wave; q < a.draws; q += kWaves) {
        const u64 want = draw_target(a, b * a.draws + q, total);
        // the first tile whose running sum is above `want`: among each 64th, then among 64 (past the last tile all are above)
        const uint32_t part = __ffsll((long long)__ballot(sh.tile[64 * lane + 63] > want)) - 1;
        const uint32_t lo = 64 * part + __ffsll((long long)__ballot(sh.tile[64 * part + lane] > want)) - 1;
        u64 before = lo ? sh.tile[lo - 1] : 0;
        const uint32_t end = std::min(a.V, (lo + 1) * a.tile);
        bool found = listed && listed <= 16 * tiles &&
                     draw_from_entries(a, r, listed, lo * a.tile, end, before, want, b * a.draws + q, total,
                                       reinterpret_cast<u64*>(sh.queue[wave].four), sh);
#pragma unroll 1
        for (uint32_t i0 = lo * a.tile; i0 < end && !found; i0 += kTile) {
            float l[4][4];
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) l[g][e] = (float)row[std::min(i0 + 256 * g + 4 * lane + e, a.V - 1)];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (found) continue;
                u64 x[4], four = 0;
                bool kept[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t i = i0 + 256 * g + 4 * lane + e;
                    kept[e] = i < end && candidate(l[g][e]) && entry(key_of(l[g][e]), i) >= last && passes(r, l[g][e]);
                }
                if (!__any(kept[0] || kept[1] || kept[2] || kept[3])) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u64 one = weight(r, l[g][e], sh.tab);
                    x[e] = kept[e] ? one : 0;
                    four += x[e];
                }
                const u64 sums = before + wave_incl(four);
                const u64 hit = __ballot(sums > want);
                before = lane64(sums, 63);
                if (hit) {
                    found = true;
                    if (lane == __ffsll((long long)hit) - 1) {
                        u64 at = sums - four;
                        float l0 = l[g][0];
                        uint32_t e0 = 0;
                        bool past = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            at += x[e];
                            if (!past) l0 = l[g][e], e0 = e;
                            past |= at > want;
                        }
                        put_draw(a, r, b * a.draws + q, i0 + 256 * g + 4 * lane + e0, l0, total, sh.tab);
                    }
                }
            }
        }
    }
}

// Adds the weights of the list's first n entries that pass min_p to their tiles.
__device__ __forceinline__ void list_to_tiles(const SampleArgs& a, const Row& r, uint32_t n, Shared& sh) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const u64 x = sh.list[i];
        const float l = entry_value(x);
        if (passes(r, l)) atomicAdd(&sh.tile[~(uint32_t)x / a.tile], weight(r, l, sh.tab));
    }
}

// The draws of a row whose first top_k elements (all, where that is off) are among the list's n entries, which are the
// row's elements from klo on.
template <typename T>
__device__ __forceinline__ void draw_from_list(const SampleArgs& a, const T* row, const Row& r, int64_t b, uint32_t n, uint32_t klo, Shared& sh) {
    uint32_t keep = n;
    u64 last = (u64)klo << 32;
    if ((r.k > 0 && r.k < n) || r.p < 1.0) {
        sort_by_ranges(n, klo, r.top, sh);
        if (r.k > 0 && r.k < n) keep = (uint32_t)r.k;
        if (r.p < 1.0) keep = place_of_mass<true>(r, keep, 0, sh) + 1;
        last = sh.list[keep - 1];
    }
    __syncthreads();
    for (int q = 0; q < kPer; ++q) sh.tile[q * kThreads + threadIdx.x] = 0;
    __syncthreads();
    list_to_tiles(a, r, keep, sh);
    draw_by_tiles(a, row, r, last, keep, b, sh);
}

// ------------------------------------------------------------------------------- looks at the elements
// Adds one to *n and puts x at that place of the list, if it has one.
__device__ __forceinline__ void append(u64 x, u64* list, uint32_t* n) {
    const uint32_t at = atomicAdd(n, 1u);
    if (at < kBins) list[at] = x;
}

template <typename T>
__device__ __forceinline__ float look_max(const T* row, uint32_t lo, uint32_t hi) {
    float top = -__builtin_inff();
    each_element<4>(row, lo, hi, threadIdx.x, kThreads, [&](const float(&l)[4], uint32_t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, l[e]);          // fmaxf drops NaN
    });
    return top;
}

// Elements from klo on, into the list.
template <typename T>
__device__ __forceinline__ void look_gather(const T* row, uint32_t lo, uint32_t hi, uint32_t klo, u64* list, uint32_t* n) {
    const float from = value_of(klo);                                // a candidate: NaN and -infinity fail the comparison
    each_element<4>(row, lo, hi, threadIdx.x, kThreads, [&](const float(&l)[4], uint32_t i) {
        if (fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= from) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (l[e] >= from) append(entry(key_of(l[e]), i + e), list, n);
        }
    });
}

// Masses by bins of l in sh.bins, which the caller has cleared; returns the thread's sum of all its weights.
template <typename T, typename SH>
__device__ __forceinline__ u64 look_bins(const T* row, uint32_t lo, uint32_t hi, const Row& r, SH& sh) {
    u64 sum = 0;
    each_element<2>(row, lo, hi, threadIdx.x, kThreads, [&](const float(&l)[4], uint32_t) {
        u64 w[4];
        int bin[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {                                // all four without a branch: their steps overlap
            w[e] = weight(r, l[e], sh.tab);                          // zero for what is no candidate
            bin[e] = bin_of(r, l[e]);
            sum += w[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (bin[e] < kBins) atomicAdd(&sh.bins[bin[e]], w[e]);
    });
    return sum;
}

// Counts (MASS: masses) of the keys klo to khi by ranges of 2^shift below khi, in sh.bins.
template <typename T, bool MASS>
__device__ __forceinline__ void look_ranges(const T* row, uint32_t V, const Row& r, uint32_t klo, uint32_t khi, int shift, Shared& sh) {
    for (int q = 0; q < kPer; ++q) sh.bins[q * kThreads + threadIdx.x] = 0;
    __syncthreads();
    each_element<2>(row, 0, V, threadIdx.x, kThreads, [&](const float(&l)[4], uint32_t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t key = key_of(l[e]);
            if (candidate(l[e]) && key >= klo && key <= khi)
                atomicAdd(&sh.bins[(khi - key) >> shift], MASS ? weight(r, l[e], sh.tab) : 1);
        }
    });
    __syncthreads();
}

// bfloat16 values with a counter have a place in descending order; the value of a place.
__device__ __forceinline__ float value_of_place(uint32_t place) {
    const uint32_t d = place < 4096 ? 4095 - place : place - 4096;
    return __uint_as_float(((d + kFirstMag) << 16) | (place < 4096 ? 0u : 0x80000000u));
}
// Counts by value in sh.count, which the caller has cleared; candidates without a counter go to the list.  The counters lie
// by magnitude, the negative ones behind; two elements are worked on in a register.
__device__ __forceinline__ uint32_t place_of_counter(uint32_t c) { return c < 4096 ? 4095 - c : c; }       // in descending order
template <typename SH>
__device__ __forceinline__ void look_values(const __bf16* row, uint32_t lo, uint32_t hi, SH& sh) {
    char* const count = reinterpret_cast<char*>(sh.count);
    each_raw<4>(row, lo, hi, threadIdx.x, kThreads, [&](const Raw<__bf16>& x, uint32_t i) {
        uint32_t d[2], at[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t w = h ? x.v.y : x.v.x;
            const u16x2 m = __builtin_bit_cast(u16x2, w & 0x7fff7fffu) - (unsigned short)kFirstMag;
            d[h] = __builtin_bit_cast(uint32_t, m);
            at[h] = (d[h] << 2) | ((w >> 1) & 0x40004000u);          // bytes; no carry where both have a counter
        }
        if (!((d[0] | d[1]) & 0xf000f000u)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                atomicAdd(reinterpret_cast<uint32_t*>(count + (at[h] & 0xffffu)), 1u);
                atomicAdd(reinterpret_cast<uint32_t*>(count + (at[h] >> 16)), 1u);
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float l = x.get(e);
            const uint32_t one = e & 1 ? d[e / 2] >> 16 : d[e / 2] & 0xffffu;
            if (one < 4096) atomicAdd(&sh.count[one | (l < 0 ? 4096 : 0)], 1u);
            else if (candidate(l)) append(entry(key_of(l), i + e), sh.list, &sh.n_list);
        }
    });
}

// Tile by tile of [t0, t1), each wave its share: adds the weights above khi to tile[t - t0], which the caller has cleared, and
// of the elements from klo to khi the count to ties[t] (TIES) or the entries to the list.  Values are compared, not keys, four
// at once.  Where few are kept, a wave lines up the fours that hold one and takes their weights 64 fours at a time: a weight
// is some 40 instructions, and few of a step's 64 fours hold one.
template <bool TIES, typename T>
__device__ __forceinline__ void look_tiles(const SampleArgs& a, const T* row, const State& st, uint32_t t0, uint32_t t1, const double* tab,
                                           Line* queue, u64* tile, uint32_t* ties, u64* list, uint32_t* n_list) {
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);      // one value: the loops below are the wave's
    const Row r = st.r;
    const float above = st.khi < kLowestKey ? -__builtin_inff() : value_of(st.khi);
    const float from = st.klo <= st.khi ? value_of(st.klo) : __builtin_inff();      // with no border: nothing from `from` to `above`
    Line& line = queue[wave];
    const uint32_t per = (t1 - t0 + kWaves - 1) / kWaves, per_tile = a.tile / 256;
    uint32_t t = t0 + wave * per, left = per_tile;                   // steps left of tile t
    if (t >= t1) return;
    const uint32_t hi = std::min(a.V, std::min(t + per, t1) * a.tile);
    u64 w = 0;
    uint32_t n = 0, queued = 0;
    auto take = [&](uint32_t m) {                                    // the first m (at most 64) fours of the line
        wave_sync();
        const f32x4 x = line.four[lane];
        const uint32_t at = line.t[lane] - t0;
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) bits |= x[e] > above ? 1 << e : 0;
        if (lane >= m) bits = 0;
#pragma unroll 1
        while (__any(bits != 0)) {                                   // mostly once or twice
            if (bits) {
                const float l = bits & 1 ? x[0] : bits & 2 ? x[1] : bits & 4 ? x[2] : x[3];
                atomicAdd(&tile[at], weight(r, l, tab));
                bits &= bits - 1;
            }
        }
        wave_sync();
    };
    auto store = [&] {                                               // the end of tile t
        if (__any(w != 0)) {
            const u64 all = wave_incl(w);
            if (lane == 63) atomicAdd(&tile[t - t0], all);
        }
        if (TIES && lane == 0) ties[t] = n;
        w = 0, n = 0, ++t, left = per_tile;
    };
    each_element<4>(row, t * a.tile, hi, lane, 64, [&](const float(&l)[4], uint32_t i) {
        const float top = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3]));          // fmaxf drops NaN
        const bool some = top > above;
        const u64 kept = __ballot(some);
        if (__any(top >= from)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool border = l[e] >= from && !(l[e] > above);
                if (TIES) n += __popcll(__ballot(border));
                else if (border) append(entry(key_of(l[e]), i + e), list, n_list);
            }
        }
        const uint32_t more = __popcll(kept);
        if (more > kLine - 64) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w += weight(r, l[e] > above ? l[e] : -__builtin_inff(), tab);
        } else if (more) {
            const uint32_t at = queued + __builtin_amdgcn_mbcnt_hi((uint32_t)(kept >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)kept, 0));
            if (some) line.four[at] = {l[0], l[1], l[2], l[3]}, line.t[at] = t;
            queued += more;
            if (queued >= 64) {
                take(64);
                const f32x4 rest = line.four[64 + (lane & (kLine - 65))];
                const uint32_t rest_t = line.t[64 + (lane & (kLine - 65))];
                wave_sync();
                if (lane < kLine - 64) line.four[lane] = rest, line.t[lane] = rest_t;
                queued -= 64;
            }
        }
        if (--left == 0) store();
    });
    if (left < per_tile) store();                                    // the row's end
    if (queued) take(queued);
}

// ------------------------------------------------------------------------------- borders
// The keys of a bin: [first, last]; every wave searches for itself, 64 keys at a time.
__device__ __forceinline__ void keys_of_bin(const Row& r, int bin, uint32_t* first, uint32_t* last) {
    uint32_t end[2];
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {                                    // the largest key with bin_of >= bin + s
        uint32_t lo = kLowestKey - 1, hi = r.top + 1;                // holds at lo, not at hi
        if (bin + s <= 0) lo = hi - 1;
        if (bin + s > kBins) hi = lo + 1;
#pragma unroll 1
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo - 1) / 64 + 1;
            const u64 at = (u64)lo + (u64)step * ((threadIdx.x & 63) + 1);
            const bool yes = at < hi && bin_of(r, value_of((uint32_t)at)) >= bin + s;
            const int n = __popcll(__ballot(yes));
            const u64 next = (u64)lo + (u64)step * (n + 1);
            lo += step * n;
            hi = next < hi ? (uint32_t)next : hi;
        }
        end[s] = lo;
    }
    *last = end[0];
    *first = end[1] + 1;
}

// Where min_p cuts off the border itself, it is the border: all that passes lies above, nothing apart.
__device__ __forceinline__ void fold_min_p(State& st) {
    if (!(st.r.log_min_p > -__builtin_inf())) return;
    uint32_t lo = kLowestKey - 1, hi = st.r.top;                     // the largest key that does not pass; the maximum does
#pragma unroll 1
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo - 1) / 64 + 1;
        const u64 at = (u64)lo + (u64)step * ((threadIdx.x & 63) + 1);
        const int n = __popcll(__ballot(at < hi && !passes(st.r, value_of((uint32_t)at))));
        const u64 next = (u64)lo + (u64)step * (n + 1);
        lo += step * n;
        hi = next < hi ? (uint32_t)next : hi;
    }
    if (lo >= st.khi) st.klo = lo + 1, st.khi = lo, st.ties = 1, st.need = 0;
}

// A key that k elements reach, and few more: the least of the groups' maxima in the bin of the k-th largest of them (0: below
// the bins).
__device__ __forceinline__ uint32_t key_by_maxima(const Row& r, int groups, Shared& sh) {
    for (int q = 0; q < kPer; ++q) sh.count[q * kThreads + threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.at = ~0u;
    __syncthreads();
    auto bin = [&](int g) {
        const float m = sh.group[g];
        return candidate(m) ? bin_of(r, m) : kBins;
    };
    for (int g = threadIdx.x; g < groups; g += kThreads) {
        const int at = bin(g);
        if (at < kBins) atomicAdd(&sh.count[at], 1u);
    }
    __syncthreads();
    u64 v[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) v[q] = sh.count[kPer * threadIdx.x + q];
    find_place(v, (u64)r.k, 0, sh);
    if (sh.bin >= kBins) return 0;
    for (int g = threadIdx.x; g < groups; g += kThreads)
        if (bin(g) == (int)sh.bin) atomicMin(&sh.at, key_of(sh.group[g]));
    __syncthreads();
    return sh.at;
}

// Narrows the keys klo to khi, which hold the border, to its own key; *need becomes the number of that key's elements that
// are kept.  MASS: it comes in as units of mass.
template <typename T, bool MASS>
__device__ __forceinline__ void narrow(const SampleArgs& a, const T* row, const Row& r, uint32_t klo, uint32_t* khi, u64* need, Shared& sh) {
#pragma unroll 1
    do {
        const int bits = klo == *khi ? 0 : 32 - __clz(*khi - klo), shift = bits > 12 ? bits - 12 : 0;      // 2^12 = kBins ranges
        look_ranges<T, MASS>(row, a.V, r, klo, *khi, shift, sh);
        u64 v[kPer];
#pragma unroll
        for (int q = 0; q < kPer; ++q) v[q] = sh.bins[kPer * threadIdx.x + q];
        find_place(v, *need, 0, sh);
        *need -= sh.above;
        *khi -= std::min<uint32_t>(sh.bin, kBins - 1) << shift;
        const uint32_t width = (1u << shift) - 1;
        klo = *khi - klo > width ? *khi - width : klo;
        __syncthreads();
    } while (klo < *khi);
    if (MASS) {
        const u64 w = weight(r, value_of(*khi), sh.tab);
        *need = w ? (*need + w - 1) / w : 1;
    }
}

// sh.bins holds the masses by bins: the border of top_p of the mass `of` for look_tiles.
__device__ __forceinline__ void border_by_bins(State& st, u64 of, Shared& sh) {
    u64 v[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) v[q] = sh.bins[kPer * threadIdx.x + q];
    const u64 target = share_of(st.r.p, of);
    find_place(v, target, 0, sh);
    st.need = target - sh.above;
    keys_of_bin(st.r, sh.bin, &st.klo, &st.khi);
    st.ties = 0;
    st.mode = kTiles;
    __syncthreads();
}

// sh.count holds the counts by value, the list the n others: the border of top_k and top_p for look_tiles.
__device__ __forceinline__ void border_by_values(const SampleArgs& a, State& st, uint32_t n, Shared& sh) {
    uint32_t c[kPerValue];
    float top = -__builtin_inff(), l[kPerValue];
#pragma unroll
    for (int q = 0; q < kPerValue; ++q) {
        c[q] = sh.count[place_of_counter(kPerValue * threadIdx.x + q)];
        l[q] = value_of_place(kPerValue * threadIdx.x + q);
        top = c[q] ? fmaxf(top, l[q]) : top;
    }
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) top = fmaxf(top, entry_value(sh.list[i]));
    top = block_max(top, sh);
    Row& r = st.r;
    st.mode = kDone;
    st.klo = 1, st.khi = 0;                                          // none: every key lies above
    st.ties = 1;
    st.need = 0;
    if (!candidate(top)) return;
    st.mode = kTiles;
    const float by = rough_by(r);
    float mass = 0.f;
#pragma unroll
    for (int q = 0; q < kPerValue; ++q) mass += c[q] ? (float)c[q] * rough_weight(l[q], top, by) : 0.f;
    mass = block_sum(mass, sh);
    if (n) {                                                         // in the list's order, which changes: integers
        u64 listed[1] = {0};
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) listed[0] += (u64)(rough_weight(entry_value(sh.list[i]), top, by) * 0x1p40f);
        block_sums(listed, sh);
        mass += (float)listed[0] * 0x1p-40f;
    }
    set_scale(r, top, fminf(mass * 1.01f + 1.f, (float)a.V));
    if (r.k == 0 && !(r.p < 1.0)) return;
    // in descending order: the list above the counters' range, the positive values, the list between, the negative, the rest
    const float high = value_of_place(0), low = value_of_place(kValues - 1);
    u64 w[kPerValue];
#pragma unroll
    for (int q = 0; q < kPerValue; ++q) {                            // many waves have no value that occurs
        w[q] = 0;
        if (__any(c[q] != 0)) w[q] = c[q] ? weight(r, l[q], sh.tab) : 0;
    }
    u64 of = 0;
#pragma unroll 1
    for (int pass = r.k > 0 ? 0 : 1; pass < (r.p < 1.0 ? 2 : 1); ++pass) {           // by count, then by mass
        u64 v[kPerValue], zone[4] = {0, 0, 0, 0};                         // the list's three, and the counters
#pragma unroll
        for (int q = 0; q < kPerValue; ++q) v[q] = pass ? w[q] * c[q] : c[q], zone[3] += v[q];
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const float x = entry_value(sh.list[i]);
            const u64 one = pass ? weight(r, x, sh.tab) : 1;
            const int at = x > high ? 0 : x < low ? 2 : 1;
            zone[0] += at == 0 ? one : 0;
            zone[1] += at == 1 ? one : 0;
            zone[2] += at == 2 ? one : 0;
        }
        if (n) {
            block_sums(zone, sh);
        } else {
            u64 all[1] = {zone[3]};
            block_sums(all, sh);
            zone[3] = all[0];
        }
        const u64 total = zone[0] + zone[1] + zone[2] + zone[3];
        if (pass == 0 && (u64)r.k >= total) continue;
        const u64 target = pass ? share_of(r.p, of ? of : total) : (u64)r.k;
        uint32_t place = kValues;
        if (target > zone[0]) {
            find_place(v, target - zone[0], zone[1], sh);
            place = sh.bin;
        }
        if (place < kValues) {
            const u64 need = target - zone[0] - sh.above;
            const float x = value_of_place(place);
            const u64 one = weight(r, x, sh.tab);
            st.klo = st.khi = key_of(x);
            st.need = pass ? (need + one - 1) / one : need;          // a place found by mass has weight
            // the mass of the first k, for top_p: all above the place, and need of it
            if (pass == 0) {
                u64 above = 0;
#pragma unroll
                for (int q = 0; q < kPerValue; ++q) above += kPerValue * threadIdx.x + q < place ? w[q] * c[q] : 0;
                for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
                    const float y = entry_value(sh.list[i]);
                    above += y > x ? weight(r, y, sh.tab) : 0;
                }
                block_incl(above, sh, &of);
                of += need * one;
            }
        } else {                                                     // among the list's entries, one by one
            st.mode = kAlone;
            return;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------- the end of a row
// The tiles' sums and the border (ties or list entries) are in LDS: adds the border's kept elements to their tiles, and
// draws.  False: the list has overflown.
template <typename T>
__device__ __forceinline__ bool draw_from_tiles(const SampleArgs& a, const T* row, const State& st, int64_t b, Shared& sh) {
    const Row r = st.r;
    const uint32_t tiles = (a.V + a.tile - 1) / a.tile;
    u64 last = (u64)(st.khi + 1) << 32;                              // kept are the entries from it on
    __syncthreads();
    if (st.need) {
        if (st.ties) {
            u64 v[kPer];
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                const uint32_t t = kPer * threadIdx.x + q;
                v[q] = t < tiles ? sh.ties[t] : 0;
            }
            find_place(v, st.need, 0, sh);
            const uint32_t t = sh.bin, end = std::min(a.V, (t + 1) * a.tile);        // the tile of the last kept
            const uint32_t left = (uint32_t)(st.need - sh.above);
            const u64 one = weight(r, value_of(st.khi), sh.tab);
            for (uint32_t i = threadIdx.x; i <= t && i < tiles; i += kThreads) sh.tile[i] += one * (i < t ? sh.ties[i] : left);
            u64 carry = 0, all;
            for (uint32_t i0 = t * a.tile; i0 < end; i0 += kThreads) {
                const uint32_t i = i0 + threadIdx.x;
                const float x = i < end ? (float)row[i] : __builtin_nanf("");
                const bool tie = candidate(x) && key_of(x) == st.khi;
                const u64 upto = carry + block_incl(tie, sh, &all);
                if (tie && upto == left) sh.at = i;
                carry += all;
            }
            __syncthreads();
            last = entry(st.khi, sh.at);
        } else {
            const uint32_t n = sh.n_list;
            if (n > kBins) return false;
            sort_list<true>(n, sh.list);
            const uint32_t place = place_of_mass<false>(r, n, st.need, sh);
            list_to_tiles(a, r, place + 1, sh);
            last = sh.list[place];
            __syncthreads();
        }
    }
    draw_by_tiles(a, row, r, last, 0, b, sh);
    return true;
}

// ------------------------------------------------------------------------------- one block, one row
template <typename T>
__device__ __forceinline__ void look_tiles_alone(const SampleArgs& a, const T* row, const State& st, Shared& sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.n_list = 0;
    for (int q = 0; q < kPer; ++q) sh.tile[q * kThreads + threadIdx.x] = 0;
    __syncthreads();
    const uint32_t tiles = (a.V + a.tile - 1) / a.tile;
    if (st.ties) look_tiles<true>(a, row, st, 0, tiles, sh.tab, sh.queue, sh.tile, sh.ties, sh.list, &sh.n_list);
    else look_tiles<false>(a, row, st, 0, tiles, sh.tab, sh.queue, sh.tile, sh.ties, sh.list, &sh.n_list);
    __syncthreads();
}

// The row by looks for any type; what the lists of the quick ways cannot hold ends here too (quick false).
template <typename T>
__device__ __forceinline__ void row_by_bins(const SampleArgs& a, int64_t b, bool quick, Shared& sh) {
    const T* row = (const T*)a.logits + b * a.ld;
    State st;
    st.r = settings(a, b);
    Row& r = st.r;
    const float own = look_max(row, 0, a.V);
    const float top = block_max(own, sh);
    if (!candidate(top)) return draw_nothing(a, b);
    if (quick && by_maxima(r.k, kThreads)) {
        set_scale(r, top, (float)kBins);
        set_bins(r, kRange);
        if (threadIdx.x == 0) sh.n_list = 0;
        sh.group[threadIdx.x] = own;
        const uint32_t klo = key_by_maxima(r, kThreads, sh);
        if (klo) {
            look_gather(row, 0, a.V, klo, sh.list, &sh.n_list);
            __syncthreads();
            if (sh.n_list <= kBins) return draw_from_list(a, row, r, b, sh.n_list, klo, sh);
        }
    }
    // the maxima of the threads bound the mass from below and, as often as a thread has elements, from above
    const float least = 0.99f * block_sum(candidate(own) ? rough_weight(own, top, rough_by(r)) : 0.f, sh);
    set_scale(r, top, 1.03f * least * 4.f * (float)((a.V + 4 * kThreads - 1) / (4 * kThreads)));
    st.klo = 1, st.khi = 0;
    st.ties = 1;
    st.need = 0;
    u64 of = 0;
    if (r.k > 0) {
        uint32_t khi = r.top;
        u64 need = (u64)r.k;
        // at least k candidates?  narrow() may only look for a border that is there
        u64 n = 0, all;
        each_element<4>(row, 0, a.V, threadIdx.x, kThreads, [&](const float(&l)[4], uint32_t) {
            for (int e = 0; e < 4; ++e) n += candidate(l[e]);
        });
        block_incl(n, sh, &all);
        if (need < all) {
            narrow<T, false>(a, row, r, kLowestKey, &khi, &need, sh);
            st.klo = st.khi = khi;
            st.need = need;
            if (r.p < 1.0) {                                         // the mass of the first k
                u64 w = 0;
                each_element<4>(row, 0, a.V, threadIdx.x, kThreads, [&](const float(&l)[4], uint32_t) {
                    for (int e = 0; e < 4; ++e) {
                        const u64 one = weight(r, l[e], sh.tab);
                        w += candidate(l[e]) && key_of(l[e]) > khi ? one : 0;
                    }
                });
                block_incl(w, sh, &of);
                of += need * weight(r, value_of(khi), sh.tab);
            }
        }
    }
    if (r.p < 1.0) {
        set_bins(r, r.k == 0 ? range_for(r, a.V, least) : kRange);
        __syncthreads();
        for (int q = 0; q < kPer; ++q) sh.bins[q * kThreads + threadIdx.x] = 0;
        __syncthreads();
        u64 sum[1] = {look_bins(row, 0, a.V, r, sh)};
        block_sums(sum, sh);
        border_by_bins(st, of ? of : sum[0], sh);
        fold_min_p(st);
        look_tiles_alone(a, row, st, sh);
        if (draw_from_tiles(a, row, st, b, sh)) return;
        narrow<T, true>(a, row, r, st.klo, &st.khi, &st.need, sh);
        st.klo = st.khi;
        st.ties = 1;
    }
    fold_min_p(st);
    look_tiles_alone(a, row, st, sh);
    draw_from_tiles(a, row, st, b, sh);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int64_t b = blockIdx.x;
    make_table(sh);
    if (threadIdx.x == 0) sh.n_list = 0;
    for (int q = 0; q < kPerValue; ++q) sh.count[q * kThreads + threadIdx.x] = 0;
    __syncthreads();
    const T* row = (const T*)a.logits + b * a.ld;
    if (a.V <= kSmall) {                                             // the list, whatever the settings
        float top = -__builtin_inff();
        for (uint32_t i = threadIdx.x; i < a.V; i += kThreads) {
            const float l = (float)row[i];
            top = fmaxf(top, l);
            if (candidate(l)) append(entry(key_of(l), i), sh.list, &sh.n_list);
        }
        top = block_max(top, sh);
        if (!candidate(top)) return draw_nothing(a, b);
        Row r = settings(a, b);
        set_scale(r, top, (float)kSmall);
        return draw_from_list(a, row, r, b, sh.n_list, kLowestKey, sh);
    }
    if constexpr (sizeof(T) == 2) {
        look_values(row, 0, a.V, sh);
        __syncthreads();
        if (sh.n_list <= kBins) {
            State st;
            st.r = settings(a, b);
            border_by_values(a, st, sh.n_list, sh);
            if (st.mode == kDone) return draw_nothing(a, b);
            if (st.mode == kTiles) {
                fold_min_p(st);
                look_tiles_alone(a, row, st, sh);
                draw_from_tiles(a, row, st, b, sh);
                return;
            }
        }
        __syncthreads();
    }
    row_by_bins<T>(a, b, sizeof(T) == 4, sh);
}

// ------------------------------------------------------------------------------- many blocks, one row
// row_by_bins on one block is the slow way, six to eight reads of the row: fp32 with a top_k that the groups' maxima do not lead to a
// list (above 819 on one block, 51 for each block of a cut row, or 2000; or, the k-th of them more than 32 T below the maximum), lists
// that overflow, bfloat16 with more than 4096 scores that have no counter.  1 x 4,000,001 fp32 top_k 1000 29 us, 3000 1715, with
// top_p 3494; 256 x 131,072 fp32 top_k 800 53, 1000 126; 1 x 50,000 top_k 50 13, at T = 0.05 39; bf16 256 x 131,072 half of it zeros 112.
// Between the kernels a row's state lies in the workspace.  The looks run on gridDim.x segments of whole tiles a row, the
// steps between them on one block a row.
struct RowSpace {
    u64 bins[kBins];                // or the kValues counts of bfloat16 values
    u64 tile[kBins];
    u64 list[kBins];
    uint32_t ties[kBins];
    float group[kBins];
    u64 mass;
    State st;
    uint32_t n_list;
};

struct Segment {
    uint32_t t0, t1, lo, hi;        // tiles and elements
};
__device__ __forceinline__ Segment segment(const SampleArgs& a) {
    const uint32_t tiles = (a.V + a.tile - 1) / a.tile, per = (tiles + gridDim.x - 1) / gridDim.x;
    Segment s;
    s.t0 = std::min(blockIdx.x * per, tiles);
    s.t1 = std::min(s.t0 + per, tiles);
    s.lo = s.t0 * a.tile;
    s.hi = std::min(a.V, s.t1 * a.tile);
    return s;
}

// fp32: the maxima of the 64 groups of each segment; clears what later kernels add to.
template <typename T>
__global__ __launch_bounds__(kThreads, 8) void split_max_kernel(SampleArgs a, RowSpace* ws) {
    RowSpace& w = ws[blockIdx.y];
    const Segment s = segment(a);
    for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < kBins; i += gridDim.x * kThreads) w.bins[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) w.n_list = 0, w.mass = 0;
    float top = s.t0 < s.t1 ? look_max((const T*)a.logits + blockIdx.y * a.ld, s.lo, s.hi) : -__builtin_inff();
    for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    if ((threadIdx.x & 15) == 0) w.group[blockIdx.x * 64 + threadIdx.x / 16] = top;
}

__global__ __launch_bounds__(kThreads) void split_clear_kernel(RowSpace* ws) {
    RowSpace& w = ws[blockIdx.x];
    for (int i = threadIdx.x; i < kBins; i += kThreads) w.bins[i] = 0;
    if (threadIdx.x == 0) w.n_list = 0;
}

// Appends the block's list (which may have overflown) to the row's.
template <typename SH>
__device__ __forceinline__ void to_row_list(SH& sh, RowSpace& w) {
    __syncthreads();
    if (threadIdx.x == 0) sh.base = sh.n_list ? atomicAdd(&w.n_list, sh.n_list) : 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < sh.n_list && i < kBins; i += kThreads)
        if (sh.base < kBins && i < kBins - sh.base) w.list[sh.base + i] = sh.list[i];
}

// bfloat16: the counts of the values.
struct SharedValues {
    uint32_t count[kValues];
    u64 list[kBins];
    uint32_t n_list, base;
};
__global__ __launch_bounds__(kThreads, 8) void split_values_kernel(SampleArgs a, RowSpace* ws) {
    __shared__ SharedValues sh;
    RowSpace& w = ws[blockIdx.y];
    const Segment s = segment(a);
    for (int q = 0; q < kPerValue; ++q) sh.count[q * kThreads + threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    if (s.t0 < s.t1) look_values((const __bf16*)a.logits + blockIdx.y * a.ld, s.lo, s.hi, sh);
    __syncthreads();
    uint32_t* count = reinterpret_cast<uint32_t*>(w.bins);
    for (int q = 0; q < kPerValue; ++q) {
        const uint32_t c = sh.count[q * kThreads + threadIdx.x];
        if (c) atomicAdd(&count[q * kThreads + threadIdx.x], c);
    }
    to_row_list(sh, w);
}

// What the looks have to do, from the groups' maxima (fp32) or the counts (bfloat16).
template <typename T>
__global__ __launch_bounds__(kThreads) void split_plan_kernel(SampleArgs a, RowSpace* ws, int groups) {
    __shared__ Shared sh;
    const int64_t b = blockIdx.x;
    RowSpace& w = ws[b];
    make_table(sh);
    State st;
    st.r = settings(a, b);
    st.mode = kAlone;
    st.klo = 1, st.khi = 0;
    st.ties = 1;
    st.need = 0;
    Row& r = st.r;
    if constexpr (sizeof(T) == 2) {
        const uint32_t n = w.n_list;
        if (n <= kBins) {
            const uint32_t* count = reinterpret_cast<const uint32_t*>(w.bins);
            for (int q = 0; q < kPerValue; ++q) sh.count[q * kThreads + threadIdx.x] = count[q * kThreads + threadIdx.x];
            for (uint32_t i = threadIdx.x; i < n; i += kThreads) sh.list[i] = w.list[i];
            __syncthreads();
            border_by_values(a, st, n, sh);
        }
    } else {
        float top = -__builtin_inff();
        for (int g = threadIdx.x; g < groups; g += kThreads) {
            sh.group[g] = w.group[g];
            top = fmaxf(top, sh.group[g]);
        }
        top = block_max(top, sh);
        if (!candidate(top)) {
            st.mode = kDone;
        } else if (by_maxima(r.k, groups)) {
            set_scale(r, top, (float)kBins);
            set_bins(r, kRange);
            st.klo = key_by_maxima(r, groups, sh);
            st.mode = st.klo ? kGather : kAlone;
        } else if (r.k == 0) {
            const float by = rough_by(r);
            float least = 0.f;
            for (int g = threadIdx.x; g < groups; g += kThreads) {
                const float m = sh.group[g];
                least += candidate(m) ? rough_weight(m, top, by) : 0.f;
            }
            least = 0.99f * block_sum(least, sh);
            const uint32_t tiles = (a.V + a.tile - 1) / a.tile, per = (tiles + groups / 64 - 1) / (groups / 64);
            set_scale(r, top, 1.03f * least * (float)per * (float)(a.tile / 64 + 64));       // elements of a group at most
            if (r.p < 1.0) {
                set_bins(r, range_for(r, a.V, least));
                st.mode = kBinning;
            } else {
                st.mode = kTiles;
            }
        }
    }
    if (st.mode == kDone) draw_nothing(a, b);
    if (st.mode == kTiles) fold_min_p(st);
    if (threadIdx.x == 0) w.st = st;
}

struct SharedLook {
    double tab[128];
    union {
        u64 bins[kBins];
        u64 list[kBins];
    };
    Line queue[kWaves];
    u64 mass;
    uint32_t n_list, base;
};
// Two blocks a compute unit leave 64 registers: the fp32 form spills 45.  With / without that bound: 4 x 4,000,001 top_p 0.9 131 /
// 131 us, no border 47 / 45, 64 x 131,072 33.4 / 33.2, with top_p 66.5 / 60.4.
template <typename T>
__global__ __launch_bounds__(kThreads, 8) void split_look_kernel(SampleArgs a, RowSpace* ws) {
    __shared__ SharedLook sh;
    RowSpace& w = ws[blockIdx.y];
    const T* row = (const T*)a.logits + blockIdx.y * a.ld;
    const int mode = w.st.mode;
    if (mode == kDone || mode == kAlone) return;
    const Segment s = segment(a);
    if (s.t0 >= s.t1) return;
    make_table(sh);
    if (mode == kTiles) {
        for (uint32_t t = threadIdx.x; t < s.t1 - s.t0; t += kThreads) sh.bins[t] = 0;
        __syncthreads();
        if (w.st.ties) look_tiles<true>(a, row, w.st, s.t0, s.t1, sh.tab, sh.queue, sh.bins, w.ties, w.list, &w.n_list);
        else look_tiles<false>(a, row, w.st, s.t0, s.t1, sh.tab, sh.queue, sh.bins, w.ties, w.list, &w.n_list);
        __syncthreads();
        for (uint32_t t = threadIdx.x; t < s.t1 - s.t0; t += kThreads) w.tile[s.t0 + t] = sh.bins[t];
        return;
    }
    if (mode == kGather) {
        // by way of LDS: an atomic on one address of the memory costs some 20 ns, and all blocks of a row share it
        if (threadIdx.x == 0) sh.n_list = 0;
        __syncthreads();
        look_gather(row, s.lo, s.hi, w.st.klo, sh.list, &sh.n_list);
        to_row_list(sh, w);
        return;
    }
    for (int q = 0; q < kPer; ++q) sh.bins[q * kThreads + threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.mass = 0;
    __syncthreads();
    const u64 mine = wave_incl(look_bins(row, s.lo, s.hi, w.st.r, sh));
    if ((threadIdx.x & 63) == 63) atomicAdd(&sh.mass, mine);
    __syncthreads();
    for (int q = 0; q < kPer; ++q) {
        const u64 m = sh.bins[q * kThreads + threadIdx.x];
        if (m) atomicAdd(&w.bins[q * kThreads + threadIdx.x], m);
    }
    if (threadIdx.x == 0) atomicAdd(&w.mass, sh.mass);
}

// After a look: the draws, or (bins) the border and what the next look has to do.
template <typename T>
__global__ __launch_bounds__(kThreads) void split_border_kernel(SampleArgs a, RowSpace* ws) {
    __shared__ Shared sh;
    const int64_t b = blockIdx.x;
    RowSpace& w = ws[b];
    const T* row = (const T*)a.logits + b * a.ld;
    const int mode = w.st.mode;
    if (mode == kDone) return;
    make_table(sh);
    bool alone = mode == kAlone;
    if (mode == kGather) {
        const uint32_t n = w.n_list;
        if (n <= kBins) {
            for (uint32_t i = threadIdx.x; i < n; i += kThreads) sh.list[i] = w.list[i];
            __syncthreads();
            draw_from_list(a, row, w.st.r, b, n, w.st.klo, sh);
        } else {
            alone = true;
        }
    } else if (mode == kBinning) {
        for (int q = 0; q < kPer; ++q) sh.bins[q * kThreads + threadIdx.x] = w.bins[q * kThreads + threadIdx.x];
        __syncthreads();
        State st = w.st;
        border_by_bins(st, w.mass, sh);
        fold_min_p(st);
        __syncthreads();
        if (threadIdx.x == 0) w.st = st, w.n_list = 0;
        return;
    } else if (mode == kTiles) {
        const State st = w.st;
        for (int q = 0; q < kPer; ++q) {
            const int t = q * kThreads + threadIdx.x;
            sh.tile[t] = w.tile[t];
            if (st.ties) sh.ties[t] = w.ties[t];
        }
        const uint32_t n = st.ties ? 0 : w.n_list;
        if (threadIdx.x == 0) sh.n_list = n;
        for (uint32_t i = threadIdx.x; i < n && i < kBins; i += kThreads) sh.list[i] = w.list[i];
        __syncthreads();
        alone = !draw_from_tiles(a, row, st, b, sh);
    }
    __syncthreads();
    if (alone) row_by_bins<T>(a, b, false, sh);
    if (threadIdx.x == 0) w.st.mode = kDone;
}

// Blocks over which a row is cut; 1: not cut.  One block's time grows with the row, a cut row costs four to six launches, and
// from some 64 rows on the rows fill the card by themselves.  Measured, us, one block a row / cut (spread 3, T = 1):
//                         top_k 50 fp32   top_p 0.9 fp32   no border fp32   top_p 0.9 bf16
//    1 x    32,768         11 /  16         26 /  31         15 / 16          21 / 27
//    1 x   131,072         16 /  17         60 /  32         39 / 17          39 / 27
//    1 x 1,000,000         65 /  19        371 /  41        254 / 21         205 / 31
//   64 x   131,072         18 /  22         63 /  64         40 / 30          41 / 38
//  128 x   131,072         27 /  36         72 /  93         47 / 45          41 / 45
// Where every row leads to a list by a small top_k, one block looks at it but twice: 1 x 262,144 24 / 17, 32 x 262,144 25 / 21,
// 64 x 500,000 52 / 53.  Rows of a larger batch are not cut, however long: 4,000,001 fp32, top_p 0.9, 64 rows 929, 67 rows 2264.
int splits(int64_t B, int64_t V) {
    const int64_t c = std::min<int64_t>(std::min<int64_t>(512 / B, V / 4096), kMaxSplit);
    return V >= 1 << 16 && c >= 8 ? (int)c : 1;
}

// Whether every row's top_k is sure to lead to a list (no looks by bins), for `groups` groups of maxima.
bool listed(const SampleArgs& a, int groups) { return !a.top_k && a.k > 0 && a.k < a.V && by_maxima(a.k, groups); }

template <typename T>
void launch_split(const SampleArgs& a, int64_t B, int C, RowSpace* ws, hipStream_t st) {
    const dim3 wide((unsigned)C, (unsigned)B), one((unsigned)B), block(kThreads);
    if constexpr (sizeof(T) == 2) {
        hipLaunchKernelGGL(split_clear_kernel, one, block, 0, st, ws);
        hipLaunchKernelGGL(split_values_kernel, wide, block, 0, st, a, ws);
    } else {
        hipLaunchKernelGGL(split_max_kernel<T>, wide, block, 0, st, a, ws);
    }
    hipLaunchKernelGGL(split_plan_kernel<T>, one, block, 0, st, a, ws, 64 * C);
    hipLaunchKernelGGL(split_look_kernel<T>, wide, block, 0, st, a, ws);
    hipLaunchKernelGGL(split_border_kernel<T>, one, block, 0, st, a, ws);
    // rows that top_p may send over bins have one more look; none does whose top_k leads to a list
    if (sizeof(T) == 4 && !listed(a, 64 * C) && (a.top_p || a.p < 1.0)) {
        hipLaunchKernelGGL(split_look_kernel<T>, wide, block, 0, st, a, ws);
        hipLaunchKernelGGL(split_border_kernel<T>, one, block, 0, st, a, ws);
    }
}

}  // namespace

// ================================================================================ C ABI
extern "C" size_t hmx_sample_logits_workspace_bytes(int64_t B, int64_t V) {
    return B > 0 && V > 0 && splits(B, V) > 1 ? (size_t)B * sizeof(RowSpace) : 0;
}

extern "C" int hmx_sample_logits(const void* logits, int64_t ld, int64_t B, int64_t V, int bf16, const void* u, int u_f64,
                                 int64_t draws, const float* temperature, const int32_t* top_k, const float* top_p,
                                 const float* min_p, double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all,
                                 int64_t* ids, float* probs, void* workspace, size_t workspace_bytes, void* stream) {
    HMX_ENTER();
    if (B < 0 || V < 1 || V >= (int64_t)1 << 31 || draws < 0 || draws >= (int64_t)1 << 31 || ld < 0 || B >= (int64_t)1 << 22)
        return HMX_EINVAL;
    if (B == 0 || draws == 0) return HMX_OK;
    if (!logits || !u || !ids || !probs) return HMX_EINVAL;
    const int C = splits(B, V);
    if (workspace_bytes < hmx_sample_logits_workspace_bytes(B, V) ||
        (C > 1 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)))
        return HMX_EWORKSPACE;
    SampleArgs a = {logits, ld, (uint32_t)V, u, u_f64 != 0, (int)draws, temperature, top_p, min_p, top_k, temperature_all,
                    top_p_all, min_p_all, top_k_all, ids, probs, (uint32_t)(hmx_ceil_div(V, (int64_t)kBins * kTile) * kTile)};
    if (C > 1 && (bf16 || !listed(a, kThreads) || (V >= 1 << 18 && B <= 32))) {
        if (bf16) launch_split<__bf16>(a, B, C, (RowSpace*)workspace, (hipStream_t)stream);
        else launch_split<float>(a, B, C, (RowSpace*)workspace, (hipStream_t)stream);
    } else if (bf16) {
        hipLaunchKernelGGL(sample_row_kernel<__bf16>, dim3((unsigned)B), dim3(kThreads), 0, (hipStream_t)stream, a);
    } else {
        hipLaunchKernelGGL(sample_row_kernel<float>, dim3((unsigned)B), dim3(kThreads), 0, (hipStream_t)stream, a);
    }
    HMX_CHECK_LAUNCH();
    return HMX_OK;
}
