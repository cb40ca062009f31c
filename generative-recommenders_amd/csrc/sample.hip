// Sampling from rows of scores with temperature, top-k, top-p and min-p, from given uniform numbers.
//
// w_i = exp((l_i - max l) / T).  Kept are the top_k first by (l descending, i ascending); of these the shortest prefix of
// that order whose mass is at least top_p of theirs; of these the ones with w_i >= min_p.  A draw is the first kept i in
// INDEX order whose running sum of w passes u * (kept mass): no sort of the row is needed, only the border of the kept set.
//
// Weights are fp64 (z exactly as far as fp64 goes, exp by table and polynomial, 2e-16) turned into integers w * 2^s, with s
// the largest scale at which the row's mass fits 62 bits (51 at most): integer sums do not depend on their order, so LDS
// and global atomics, any split of a row and any number of waves give the same set and the same draw.
//
// How the border is found, with as few looks at the row as its settings allow:
//   top_k: the k-th largest of the maxima of groups of elements is a value that at least k elements reach; what reaches it
//     is gathered into a list, and the list does the rest (top_p and min_p on top of top_k included).
//   top_p: masses of 4096 bins of equal width in l.  What lies so far below the maximum that V of it weigh less than half of
//     1 - top_p is summed without a bin.  One more look sums the tiles of the row above the border's bin and gathers that
//     bin's few elements, which are sorted for the border itself; the draw goes by the sums of the tiles.
//   Where a list overflows (equal scores, scores that differ in their last bits): equal ranges of the ordered 32-bit key,
//     until a range fits the list or is one key, whose border is the index of its r-th element.
#include "hmx_common.h"

#include <algorithm>

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 4096;                // four per thread
constexpr int kPer = kBins / kThreads;
constexpr int kList = 4096;
constexpr int kSmall = 2048;               // rows up to this length go into the list whole
constexpr int kTiles = 4096;               // tiles of a row at most (their running sums stay in LDS), four per thread
constexpr uint32_t kLowestKey = 0x00800000u;        // the key after that of -infinity
constexpr float kRange = 32.f;             // bins reach down to exp(-32) of the largest weight

typedef unsigned long long u64;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

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
    uint32_t tile;                                   // elements of a tile, a multiple of 256
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

// Elements i .. i + 3 of a row (NaN past its end).  Rows start anywhere: the loads need only the type's own alignment.
template <typename T>
__device__ __forceinline__ void load4(const T* row, uint32_t i, uint32_t V, float (&v)[4]) {
    if (i + 4 <= V) {
        if constexpr (sizeof(T) == 4) {
            f32x4 a;
            __builtin_memcpy(&a, row + i, 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = a[e];
        } else {
            bf16x4 a;
            __builtin_memcpy(&a, row + i, 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)a[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i < V && i + e < V ? (float)row[i + e] : __builtin_nanf("");
    }
}

// f(value, index) for the elements of [lo, hi), `threads` threads in steps of four, four steps' loads ahead of their use.
template <typename T, typename F>
__device__ __forceinline__ void each_element(const T* row, uint32_t lo, uint32_t hi, int thread, int threads, F f) {
    constexpr int U = 4;
    for (uint32_t i0 = lo; i0 < hi; i0 += threads * 4 * U) {
        float v[U][4];
#pragma unroll
        for (int q = 0; q < U; ++q) load4(row, i0 + (q * threads + thread) * 4, hi, v[q]);
#pragma unroll
        for (int q = 0; q < U; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) f(v[q][e], i0 + (q * threads + thread) * 4 + e);
    }
}

// What a row's weights and bins are computed with.
struct Row {
    float lmax, bin_scale;          // bins per unit of l
    double inv_t, step;             // step: 128 / (T ln 2)
    double log_min_p;               // -infinity: off
    double cut;                     // weights of steps below it round to zero units
    int scale;                      // units are 2^-scale
    double p;                       // 1: off
    int64_t k;                      // 0: off
};

__device__ __forceinline__ int bin_of(const Row& r, float l) {      // ascending as l falls; kBins: all that lies lower
    const float t = l == r.lmax ? 0.f : (r.lmax - l) * r.bin_scale;
    return t < (float)kBins ? (int)t : kBins;
}
__device__ __forceinline__ double log_weight(const Row& r, float l) {
    return l == r.lmax ? 0.0 : ((double)l - (double)r.lmax) * r.inv_t;
}

// exp((l - max) / T) in units of 2^-scale, rounded to an integer (at most 2^51).  With n + x = 128 z / ln 2, |x| <= 1/2 and
// n = 128 q + i: 2^q * 2^(i / 128) * e^(x ln2 / 128), the last by four terms after 1 (what they leave off: 1e-15), the
// second from the table.  Adding 1.5 * 2^52 rounds to n and leaves its bits; 2^q goes into the exponent, which stays in
// range because smaller weights than half a unit end at the cut.
__device__ __forceinline__ u64 weight(const Row& r, float l, const double* tab) {
    const double y = l == r.lmax ? 0.0 : ((double)l - (double)r.lmax) * r.step;
    if (!(y > r.cut)) return 0;
    const double shifted = y + 6755399441055744.0;
    const int n = (int)(uint32_t)__double_as_longlong(shifted);
    const double x = y - (shifted - 6755399441055744.0);
    double e = fma(x, 3.583032305400251e-11, 2.646642144433097e-08);                 // (ln2 / 128)^k / k!
    e = fma(x, e, 1.4662262387640425e-05);
    e = fma(x, e, 0.0054152123481245725);
    e = fma(x, e, 1.0);
    const double m = tab[n & 127] * e;
    const double w = __longlong_as_double(__double_as_longlong(m) + ((long long)((n >> 7) + r.scale) << 52));
    return __double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
}

// The kept set so far: keys above `key`, and of those equal to it the indices up to `idx`.
struct Border {
    uint32_t key, idx;
};
__device__ __forceinline__ bool inside(const Border& b, uint32_t key, uint32_t i) {
    return key > b.key || (key == b.key && i <= b.idx);
}
__device__ __forceinline__ u64 kept_weight(const Row& r, const Border& in, float l, uint32_t i, const double* tab) {
    if (!candidate(l) || !inside(in, key_of(l), i)) return 0;
    return log_weight(r, l) >= r.log_min_p ? weight(r, l, tab) : 0;
}

// The largest candidate of a thread's share of [lo, hi) (-infinity: none).
template <typename T>
__device__ __forceinline__ float thread_max(const T* row, uint32_t lo, uint32_t hi, int thread, int threads) {
    float top = -__builtin_inff();
    each_element(row, lo, hi, thread, threads, [&](float l, uint32_t) { top = fmaxf(top, l); });       // fmaxf drops NaN
    return top;
}

// ------------------------------------------------------------------------------- block sums
__device__ __forceinline__ u64 shfl_up64(u64 v, int d) {
    const uint32_t lo = __shfl_up((uint32_t)v, d), hi = __shfl_up((uint32_t)(v >> 32), d);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 wave_incl(u64 v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

struct Shared {
    double tab[128];
    union {
        u64 mass[kBins];
        uint32_t count[kBins];
        u64 run[kList];
        u64 tile[kTiles];
    };
    union {
        u64 list[kList];
        uint32_t ties[kTiles];
        float group[kThreads];
    };
    u64 wsum[kWaves];
    float wmax[kWaves];
    u64 rest, above, target, total, in_bin;
    uint32_t bin, n_list, at;
};

__device__ __forceinline__ void make_table(Shared& sh) {
    if (threadIdx.x < 128) sh.tab[threadIdx.x] = exp2((double)threadIdx.x / 128.0);
}

// Inclusive sums over the block in thread order; *total gets the sum of all.
__device__ __forceinline__ u64 block_incl(u64 v, Shared& sh, u64* total) {
    const int wave = threadIdx.x >> 6;
    v = wave_incl(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.wsum[wave] = v;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        before += i < wave ? sh.wsum[i] : 0;
        all += sh.wsum[i];
    }
    *total = all;
    return v + before;
}

// ------------------------------------------------------------------------------- selection
enum Kind { kCount, kMass };

// Adds one element to the bins; what lies below them goes to the thread's own `rest`.
template <Kind KIND>
__device__ __forceinline__ void add_to_bin(const Row& r, float l, int b, u64* mass, uint32_t* count, const double* tab, u64& rest) {
    if constexpr (KIND == kMass) {
        const u64 w = weight(r, l, tab);
        if (b == kBins) rest += w;
        else atomicAdd(&mass[b], w);
    } else {
        if (b == kBins) ++rest;
        else atomicAdd(&count[b], 1u);
    }
}

// Counts or masses of the row's elements inside `in` by bin.  SUB false: bins of bin_of(), the rest apart; true: ranges of
// 2^shift keys below khi, elements from klo to khi only.
template <typename T, Kind KIND, bool SUB>
__device__ __forceinline__ void histogram(const SampleArgs& a, const T* row, const Row& r, const Border& in, uint32_t klo, uint32_t khi,
                          int shift, Shared& sh) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
        if (KIND == kMass) sh.mass[b] = 0;
        else sh.count[b] = 0;
    }
    if (threadIdx.x == 0) sh.rest = 0;
    __syncthreads();
    u64 rest = 0;
    each_element(row, 0, a.V, threadIdx.x, kThreads, [&](float l, uint32_t i) {
        if (!candidate(l)) return;
        const uint32_t key = key_of(l);
        if (!inside(in, key, i)) return;
        if (SUB && (key < klo || key > khi)) return;
        add_to_bin<KIND>(r, l, SUB ? (int)((khi - key) >> shift) : bin_of(r, l), sh.mass, sh.count, sh.tab, rest);
    });
    if (!SUB && rest) atomicAdd(&sh.rest, rest);
    __syncthreads();
}

// The first bin at which the running count (mass) reaches `target` (> 0): sh.bin (kBins where the bins do not reach it),
// sh.above, sh.in_bin, sh.target, and sh.total of all bins and the rest.  share >= 0: the target is that part of the total.
template <Kind KIND>
__device__ __forceinline__ void find_bin(u64 target, double share, Shared& sh) {
    u64 v[kPer], sum = 0;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        v[q] = KIND == kMass ? sh.mass[kPer * threadIdx.x + q] : (u64)sh.count[kPer * threadIdx.x + q];
        sum += v[q];
    }
    u64 all;
    u64 upto = block_incl(sum, sh, &all) - sum;
    const u64 total = all + sh.rest;
    if (share >= 0.0) {
        target = (u64)ceil(share * (double)total);
        target = target < 1 ? 1 : target > total ? total : target;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sh.bin = kBins;
        sh.above = all;
        sh.in_bin = sh.rest;
        sh.target = target;
        sh.total = total;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        if (upto < target && target <= upto + v[q]) sh.bin = kPer * threadIdx.x + q, sh.above = upto, sh.in_bin = v[q];
        upto += v[q];
    }
    __syncthreads();
}

// The largest key with bin_of >= b (kLowestKey - 1: none); every wave searches for itself, 64 keys at a time.
__device__ __forceinline__ uint32_t last_key_of_bin(const Row& r, int b) {
    uint32_t lo = kLowestKey - 1, hi = key_of(r.lmax) + 1;          // holds at lo, not at hi
    if (b <= 0) return hi - 1;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo - 1) / 64 + 1;
        const u64 at = (u64)lo + (u64)step * ((threadIdx.x & 63) + 1);
        const bool yes = at < hi && bin_of(r, value_of((uint32_t)at)) >= b;
        const int n = __popcll(__ballot(yes));
        const u64 top = (u64)lo + (u64)step * (n + 1);
        lo += step * n;
        hi = top < hi ? (uint32_t)top : hi;
    }
    return lo;
}
__device__ __forceinline__ uint32_t first_key_of_bin(const Row& r, int b) {      // the smallest key with bin_of <= b
    return b >= kBins ? kLowestKey : last_key_of_bin(r, b + 1) + 1;
}

__device__ __forceinline__ u64 entry(uint32_t key, uint32_t i) { return ((u64)key << 32) | (uint32_t)~i; }
__device__ __forceinline__ float entry_value(u64 x) { return value_of((uint32_t)(x >> 32)); }

// Sorts the list's first n entries; DESC: the largest first.  Bitonic: steps of up to 64 stay in a wave's own 128 entries
// and need no barrier of the block.
template <bool DESC>
__device__ __forceinline__ void sort_list(uint32_t n, u64* list) {
    uint32_t m = 2;
    while (m < n) m <<= 1;
    for (uint32_t i = n + threadIdx.x; i < m; i += kThreads) list[i] = DESC ? 0 : ~0ull;
    __syncthreads();
    auto step = [&](uint32_t size, uint32_t stride) {
        for (uint32_t t = threadIdx.x; t < m / 2; t += kThreads) {
            const uint32_t i = 2 * t - (t & (stride - 1)), j = i + stride;
            const u64 x = list[i], y = list[j];
            const bool up = ((i & size) != 0) == DESC;
            if (x != y && (x > y) == up) list[i] = y, list[j] = x;
        }
    };
    for (uint32_t size = 2; size <= m; size <<= 1) {
        uint32_t stride = size / 2;
        if (stride > 64) {
            __syncthreads();
            for (; stride > 64; stride >>= 1) {
                step(size, stride);
                __syncthreads();
            }
        }
        for (; stride > 0; stride >>= 1) {
            step(size, stride);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
    __syncthreads();
}

// Gathers the elements of `in` with klo <= key <= khi into the list.  False: there are more than fit.
template <typename T>
__device__ __forceinline__ bool gather(const SampleArgs& a, const T* row, const Border& in, uint32_t klo, uint32_t khi, Shared& sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    each_element(row, 0, a.V, threadIdx.x, kThreads, [&](float l, uint32_t i) {
        const uint32_t key = key_of(l);
        if (!candidate(l) || key < klo || key > khi || !inside(in, key, i)) return;
        const uint32_t at = atomicAdd(&sh.n_list, 1u);
        if (at < kList) sh.list[at] = entry(key, i);
    });
    __syncthreads();
    return sh.n_list <= kList;
}

// The place in the list's first n entries (sorted) at which their running mass reaches `target`.
__device__ __forceinline__ uint32_t place_of_mass(const Row& r, uint32_t n, u64 target, Shared& sh) {
    u64 carry = 0, all;
    __syncthreads();
    if (threadIdx.x == 0) sh.at = n - 1;
    for (uint32_t i0 = 0; i0 < n; i0 += kThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const u64 w = i < n ? weight(r, entry_value(sh.list[i]), sh.tab) : 0;
        const u64 upto = carry + block_incl(w, sh, &all);
        if (i < n && upto >= target && upto - w < target) sh.at = i;
        carry += all;
    }
    __syncthreads();
    return sh.at;
}

// The index of the rank-th element with this key, by counts of tiles (rank >= 1, and there are that many).
template <typename T>
__device__ __forceinline__ uint32_t index_of_rank(const SampleArgs& a, const T* row, const Border& in, uint32_t key, u64 rank, Shared& sh) {
    const uint32_t tiles = (a.V + a.tile - 1) / a.tile;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    for (uint32_t t = tiles + threadIdx.x; t < kTiles; t += kThreads) sh.ties[t] = 0;
    for (uint32_t t = wave; t < tiles; t += kWaves) {
        uint32_t n = 0;
        each_element(row, t * a.tile, std::min(a.V, (t + 1) * a.tile), lane, 64,
                     [&](float l, uint32_t i) { n += candidate(l) && key_of(l) == key && inside(in, key, i); });
        for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
        if (lane == 0) sh.ties[t] = n;
    }
    __syncthreads();
    u64 n[kPer], sum = 0, all;
#pragma unroll
    for (int q = 0; q < kPer; ++q) n[q] = sh.ties[kPer * threadIdx.x + q], sum += n[q];
    u64 upto = block_incl(sum, sh, &all) - sum;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        if (upto < rank && rank <= upto + n[q]) sh.bin = kPer * threadIdx.x + q, sh.above = upto;
        upto += n[q];
    }
    __syncthreads();
    if (wave == 0) {
        const uint32_t t = sh.bin, end = std::min(a.V, (t + 1) * a.tile);
        uint32_t left = (uint32_t)(rank - sh.above);
        for (uint32_t i0 = t * a.tile; i0 < end; i0 += 64) {
            const uint32_t i = i0 + lane;
            const float l = i < end ? (float)row[i] : __builtin_nanf("");
            const bool tie = candidate(l) && key_of(l) == key && inside(in, key, i);
            const u64 ties = __ballot(tie);
            const uint32_t here = __popcll(ties);
            if (here < left) {
                left -= here;
                continue;
            }
            if (tie && __popcll(ties & ((1ull << lane) - 1)) == left - 1) sh.at = i;
            break;
        }
    }
    __syncthreads();
    return sh.at;
}

// The border of the share / count `need` (> 0) of the elements with klo <= key <= khi inside `in`.
template <typename T, Kind KIND>
__device__ __forceinline__ Border border_in(const SampleArgs& a, const T* row, const Row& r, const Border& in, uint32_t klo, uint32_t khi, u64 need,
                            Shared& sh) {
    while (!gather(a, row, in, klo, khi, sh)) {
        if (klo == khi) {
            u64 rank = need;
            if (KIND == kMass) {
                const u64 w = weight(r, value_of(khi), sh.tab);
                rank = w ? (need + w - 1) / w : 1;
            }
            const u64 n = sh.n_list;
            return Border{khi, index_of_rank(a, row, in, khi, rank < n ? rank : n, sh)};
        }
        const int bits = 32 - __clz(khi - klo), shift = bits > 12 ? bits - 12 : 0;      // 2^12 = kBins ranges
        histogram<T, KIND, true>(a, row, r, in, klo, khi, shift, sh);
        find_bin<KIND>(need, -1.0, sh);
        need -= sh.above;
        khi -= sh.bin << shift;
        const uint32_t width = (1u << shift) - 1;
        klo = khi - klo > width ? khi - width : klo;
    }
    const uint32_t n = sh.n_list;
    sort_list<true>(n, sh.list);
    const u64 x = sh.list[KIND == kMass ? place_of_mass(r, n, need, sh) : (uint32_t)std::min<u64>(need, n) - 1];
    __syncthreads();
    return Border{(uint32_t)(x >> 32), ~(uint32_t)x};
}

__device__ __forceinline__ u64 share_of(double p, u64 total) {
    const u64 t = (u64)ceil((p > 0.0 ? p : 0.0) * (double)total);
    return t < 1 ? 1 : t > total ? total : t;
}

__device__ __forceinline__ u64 draw_target(const SampleArgs& a, int64_t at, u64 total) {
    const double u = a.u64bit ? ((const double*)a.u)[at] : (double)((const float*)a.u)[at];
    const double t = u > 0.0 ? u * (double)total : 0.0;             // NaN counts as 0
    return t < (double)total ? std::min<u64>((u64)t, total - 1) : total - 1;
}
__device__ __forceinline__ void put_draw(const SampleArgs& a, const Row& r, int64_t at, uint32_t i, float l, u64 total) {
    a.ids[at] = i;
    a.probs[at] = (float)(ldexp(exp(log_weight(r, l)), r.scale) / (double)total);
}

// The draws of a row whose first top_k elements (all, where that is off) are among the list's n entries.
__device__ __forceinline__ void draw_from_list(const SampleArgs& a, const Row& r, int64_t b, uint32_t n, Shared& sh) {
    uint32_t keep = n;
    if ((r.k > 0 && r.k < n) || r.p < 1.0) {
        sort_list<true>(n, sh.list);
        if (r.k > 0 && r.k < n) keep = (uint32_t)r.k;
    }
    u64 all;
    if (r.p < 1.0) {
        u64 total = 0;
        for (uint32_t i0 = 0; i0 < keep; i0 += kThreads) {
            const uint32_t i = i0 + threadIdx.x;
            block_incl(i < keep ? weight(r, entry_value(sh.list[i]), sh.tab) : 0, sh, &all);
            total += all;
        }
        keep = place_of_mass(r, keep, share_of(r.p, total), sh) + 1;
    }
    // the kept entries in index order, with their running sums (below min_p: weight zero)
    for (uint32_t i = threadIdx.x; i < keep; i += kThreads) {
        const u64 x = sh.list[i];
        sh.list[i] = ((u64)(~(uint32_t)x) << 32) | (uint32_t)(x >> 32);
    }
    sort_list<false>(keep, sh.list);
    u64 total = 0;
    for (uint32_t i0 = 0; i0 < keep; i0 += kThreads) {
        const uint32_t i = i0 + threadIdx.x;
        u64 w = 0;
        if (i < keep) {
            const float l = value_of((uint32_t)sh.list[i]);
            if (log_weight(r, l) >= r.log_min_p) w = weight(r, l, sh.tab);
        }
        const u64 upto = total + block_incl(w, sh, &all);
        if (i < keep) sh.run[i] = upto;
        total += all;
    }
    __syncthreads();
    for (int q = threadIdx.x; q < a.draws; q += kThreads) {
        const u64 want = draw_target(a, b * a.draws + q, total);
        uint32_t lo = 0, hi = keep - 1;                              // the first with a running sum above `want`
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (sh.run[mid] > want) hi = mid;
            else lo = mid + 1;
        }
        const u64 x = sh.list[lo];
        put_draw(a, r, b * a.draws + q, (uint32_t)(x >> 32), value_of((uint32_t)x), total);
    }
}

// The draws by the sums of the row's tiles in sh.tile (zero past the last): one wave a draw.
template <typename T>
__device__ __forceinline__ void draw_from_tiles(const SampleArgs& a, const T* row, const Row& r, const Border& in, int64_t b, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 w[kPer], sum = 0, total;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q) w[q] = sh.tile[kPer * threadIdx.x + q], sum += w[q];
    u64 upto = block_incl(sum, sh, &total) - sum;
#pragma unroll
    for (int q = 0; q < kPer; ++q) upto += w[q], sh.tile[kPer * threadIdx.x + q] = upto;
    __syncthreads();
    for (int q = wave; q < a.draws; q += kWaves) {
        const u64 want = draw_target(a, b * a.draws + q, total);
        uint32_t lo = 0, hi = kTiles - 1;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (sh.tile[mid] > want) hi = mid;
            else lo = mid + 1;
        }
        u64 before = lo ? sh.tile[lo - 1] : 0;
        const uint32_t end = std::min(a.V, (lo + 1) * a.tile);
        for (uint32_t i0 = lo * a.tile; i0 < end; i0 += 256) {
            float v[4];
            u64 x[4], four = 0;
            const uint32_t i = i0 + 4 * lane;
            load4(row, i, end, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = kept_weight(r, in, v[e], i + e, sh.tab), four += x[e];
            const u64 sums = before + wave_incl(four);
            const u64 hit = __ballot(sums > want);
            if (hit) {
                if (lane == __ffsll((long long)hit) - 1) {
                    u64 at = sums - four;
                    int e = 0;
                    for (; e < 3; ++e) {
                        at += x[e];
                        if (at > want) break;
                    }
                    float l = v[0];
#pragma unroll
                    for (int g = 1; g < 4; ++g) l = e == g ? v[g] : l;
                    put_draw(a, r, b * a.draws + q, i + e, l, total);
                }
                break;
            }
            before = ((u64)__shfl((uint32_t)(sums >> 32), 63) << 32) | __shfl((uint32_t)sums, 63);
        }
    }
}

__device__ __forceinline__ void draw_nothing(const SampleArgs& a, int64_t b) {
    for (int q = threadIdx.x; q < a.draws; q += kThreads) a.ids[b * a.draws + q] = -1, a.probs[b * a.draws + q] = 0.f;
}

// ------------------------------------------------------------------------------- a row's settings
__device__ __forceinline__ Row settings(const SampleArgs& a, int64_t b) {
    double t = a.temperature ? (double)a.temperature[b] : a.t;
    const double p = a.top_p ? (double)a.top_p[b] : a.p, mp = a.min_p ? (double)a.min_p[b] : a.mp;
    Row r;
    r.k = a.top_k ? a.top_k[b] : a.k;
    if (!(t > 0.0) || t > 3e38) t = 1.0, r.k = 1;
    if (r.k < 0 || r.k >= a.V) r.k = 0;
    r.p = p < 1.0 ? p : 1.0;
    r.inv_t = 1.0 / t;
    r.log_min_p = mp > 0.0 ? log(mp < 1.0 ? mp : 1.0) : -__builtin_inf();
    r.step = 184.6649652337873 * r.inv_t;                            // 128 / ln 2
    r.lmax = 0.f;
    r.scale = 0;
    r.cut = 0.0;
    r.bin_scale = (float)((double)kBins / (double)kRange * r.inv_t);
    return r;
}
// Whether the k-th largest of `groups` maxima leads to a list: groups * ln(groups / (groups - k)) <= 1.7 groups elements
// reach it where the groups are alike.
__device__ __forceinline__ bool by_maxima(const Row& r, int64_t groups) { return r.k > 0 && 5 * r.k <= 4 * groups; }

// The maximum, the scale (the row's mass, at most `most` times the largest weight, has to fit 62 bits), and for top_p the
// range of the bins: V elements below it weigh less than half of what top_p leaves out of a mass of at least `least`.
__device__ __forceinline__ void set_scale(const SampleArgs& a, Row& r, float lmax, float least, float most) {
    r.lmax = lmax;
    int ex;
    (void)frexpf(most, &ex);                                         // most < 2^ex
    r.scale = min(51, 62 - ex);
    r.cut = -128.0 * (double)(r.scale + 2);
    float range = kRange;
    if (r.k == 0 && r.p < 1.0) {
        const float out = (float)(1.0 - r.p) * least * 0.75f;
        const float down = logf(2.f * (float)a.V / out);
        range = out > 0.f && down < kRange ? fmaxf(down, 0.125f) : kRange;
    }
    r.bin_scale = (float)((double)kBins / (double)range * r.inv_t);
}

// ------------------------------------------------------------------------------- one block, one row
// Counts the maxima (threads' own groups) into bins and gathers what reaches the k-th largest.  False: more than the list
// holds, or the k-th largest lies below the bins.
__device__ __forceinline__ uint32_t key_by_maxima(const Row& r, const float* maxima, uint32_t groups, Shared& sh) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) sh.count[b] = 0;
    if (threadIdx.x == 0) sh.rest = 0;
    __syncthreads();
    for (uint32_t g = threadIdx.x; g < groups; g += kThreads) {
        const float m = maxima[g];
        const int b = candidate(m) ? bin_of(r, m) : kBins;
        if (b < kBins) atomicAdd(&sh.count[b], 1u);
    }
    __syncthreads();
    find_bin<kCount>((u64)r.k, -1.0, sh);
    return sh.bin < kBins ? first_key_of_bin(r, sh.bin) : 0;
}

// The sums over the row's tiles (sh.tile) of the weights inside `in`; BORDER: of those above khi alone, the ones from klo to
// khi go to the list, false when they do not fit.
template <typename T, bool BORDER>
__device__ __forceinline__ bool sum_tiles(const SampleArgs& a, const T* row, const Row& r, const Border& in, uint32_t klo,
                                          uint32_t khi, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t tiles = (a.V + a.tile - 1) / a.tile;
    __syncthreads();
    if (threadIdx.x == 0) sh.n_list = 0;
    for (uint32_t t = tiles + threadIdx.x; t < kTiles; t += kThreads) sh.tile[t] = 0;
    __syncthreads();
    for (uint32_t t = wave; t < tiles; t += kWaves) {
        u64 w = 0;
        each_element(row, t * a.tile, std::min(a.V, (t + 1) * a.tile), lane, 64, [&](float l, uint32_t i) {
            if constexpr (BORDER) {
                const uint32_t key = key_of(l);
                if (!candidate(l) || key < klo || !inside(in, key, i)) return;
                if (key <= khi) {
                    const uint32_t at = atomicAdd(&sh.n_list, 1u);
                    if (at < kList) sh.list[at] = entry(key, i);
                    return;
                }
            }
            w += kept_weight(r, in, l, i, sh.tab);
        });
        w = wave_incl(w);
        if (lane == 63) sh.tile[t] = w;
    }
    __syncthreads();
    return sh.n_list <= kList;
}

template <typename T>
__device__ __forceinline__ void whole_row(const SampleArgs& a, int64_t b, Shared& sh) {
    const T* row = (const T*)a.logits + b * a.ld;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Row r = settings(a, b);
    Border in = {0, 0};                                              // key 0 is below every candidate: all are inside
    const float own = thread_max(row, 0, a.V, threadIdx.x, kThreads);
    float top = own;
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (lane == 0) sh.wmax[wave] = top;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, sh.wmax[i]);
    if (!candidate(top)) return draw_nothing(a, b);
    if (a.V <= kSmall || by_maxima(r, kThreads)) {
        set_scale(a, r, top, 1.f, (float)kList);
        uint32_t klo = kLowestKey;
        if (a.V > kSmall) {
            sh.group[threadIdx.x] = own;
            klo = key_by_maxima(r, sh.group, kThreads, sh);
        }
        if (klo && gather(a, row, in, klo, 0xffffffffu, sh)) return draw_from_list(a, r, b, sh.n_list, sh);
    }
    // the maxima of the threads bound the mass from below and, as often as a thread has elements, from above
    {
        const float c = (float)(1.4426950408889634 * r.inv_t);
        float sum = own == top ? 1.f : candidate(own) ? __builtin_amdgcn_exp2f((own - top) * c) : 0.f;
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
        __syncthreads();
        if (lane == 0) sh.wmax[wave] = sum;
        __syncthreads();
        sum = 0.f;
        for (int i = 0; i < kWaves; ++i) sum += sh.wmax[i];
        set_scale(a, r, top, sum * 0.99f, sum * 1.01f * 4.f * (float)((a.V + 4 * kThreads - 1) / (4 * kThreads)));
    }
    if (r.k > 0) {
        histogram<T, kCount, false>(a, row, r, in, 0, 0, 0, sh);
        find_bin<kCount>((u64)r.k, -1.0, sh);
        const u64 above = sh.above, here = sh.in_bin, total = sh.total;
        const int bin = sh.bin;
        const uint32_t klo = (u64)r.k >= total ? kLowestKey : first_key_of_bin(r, bin);
        if (std::min(above + here, total) <= kList) {
            gather(a, row, in, klo, 0xffffffffu, sh);
            return draw_from_list(a, r, b, sh.n_list, sh);
        }
        if ((u64)r.k < total) in = border_in<T, kCount>(a, row, r, in, klo, last_key_of_bin(r, bin), (u64)r.k - above, sh);
    }
    bool summed = false;
    if (r.p < 1.0) {
        histogram<T, kMass, false>(a, row, r, in, 0, 0, 0, sh);
        find_bin<kMass>(0, r.p > 0.0 ? r.p : 0.0, sh);
        const u64 need = sh.target - sh.above;
        const int bin = sh.bin;
        const uint32_t klo = first_key_of_bin(r, bin), khi = last_key_of_bin(r, bin);
        summed = sum_tiles<T, true>(a, row, r, in, klo, khi, sh);
        if (summed) {                                                // the border's bin: its kept elements join their tiles
            const uint32_t n = sh.n_list;
            sort_list<true>(n, sh.list);
            const uint32_t last = place_of_mass(r, n, need, sh);
            const u64 x = sh.list[last];
            for (uint32_t i = threadIdx.x; i <= last; i += kThreads) {
                const u64 y = sh.list[i];
                const float l = entry_value(y);
                if (log_weight(r, l) >= r.log_min_p) atomicAdd(&sh.tile[~(uint32_t)y / a.tile], weight(r, l, sh.tab));
            }
            in = Border{(uint32_t)(x >> 32), ~(uint32_t)x};
        } else {
            in = border_in<T, kMass>(a, row, r, in, klo, khi, need, sh);
        }
    }
    if (!summed) sum_tiles<T, false>(a, row, r, in, 0, 0, sh);
    draw_from_tiles(a, row, r, in, b, sh);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ Shared sh;
    make_table(sh);
    whole_row<T>(a, blockIdx.x, sh);
}

}  // namespace

// ================================================================================ C ABI
extern "C" int hmx_sample_logits(const void* logits, int64_t ld, int64_t B, int64_t V, int bf16, const void* u, int u_f64,
                                 int64_t draws, const float* temperature, const int32_t* top_k, const float* top_p,
                                 const float* min_p, double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all,
                                 int64_t* ids, float* probs, void* stream) {
    HMX_ENTER();
    if (B < 0 || V < 1 || V >= (int64_t)1 << 31 || draws < 0 || draws >= (int64_t)1 << 31 || ld < 0 || B >= (int64_t)1 << 22)
        return HMX_EINVAL;
    if (B == 0 || draws == 0) return HMX_OK;
    if (!logits || !u || !ids || !probs) return HMX_EINVAL;
    SampleArgs a = {logits, ld, (uint32_t)V, u, u_f64 != 0, (int)draws, temperature, top_p, min_p, top_k, temperature_all,
                    top_p_all, min_p_all, top_k_all, ids, probs, (uint32_t)(hmx_ceil_div(V, (int64_t)kTiles * 256) * 256)};
    if (bf16)
        hipLaunchKernelGGL(sample_row_kernel<__bf16>, dim3((unsigned)B), dim3(kThreads), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(sample_row_kernel<float>, dim3((unsigned)B), dim3(kThreads), 0, (hipStream_t)stream, a);
    HMX_CHECK_LAUNCH();
    return HMX_OK;
}
