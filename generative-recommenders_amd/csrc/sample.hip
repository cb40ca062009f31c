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
// The border is found on counts and masses of 2048 bins: first bins of T / 64 in l below the maximum, then, inside one
// bin, equal ranges of the ordered 32-bit key, until the border's bin fits a list in LDS (sorted there) or is one key
// (ties: the border is the index of the r-th).  When the whole kept set fits the list, all is done in it.
#include "hmx_common.h"

#include <algorithm>

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;                // two per thread
constexpr int kList = 4096;
constexpr int kTiles = 1024;               // tiles of a row at most (running sums in LDS)
constexpr uint32_t kLowestKey = 0x00800000u;        // the key after that of -infinity

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
        for (int e = 0; e < 4; ++e) v[e] = i + e < V ? (float)row[i + e] : __builtin_nanf("");
    }
}

// What a row's weights and bins are computed with.
struct Row {
    float lmax, bin_scale;          // bins of T / 64
    double inv_t;
    double log_min_p;               // -infinity: off
    double unit;                    // 2^s
};

__device__ __forceinline__ int bin_of(const Row& r, float l) {      // ascending as l falls; kBins: all that lies lower
    const float t = l == r.lmax ? 0.f : (r.lmax - l) * r.bin_scale;
    return t < (float)kBins ? (int)t : kBins;
}

__device__ __forceinline__ double log_weight(const Row& r, float l) {
    return l == r.lmax ? 0.0 : ((double)l - (double)r.lmax) * r.inv_t;
}

// exp(z), z <= 0: z = (64 q + i) ln2 / 64 + x, |x| <= ln2 / 128: 2^q * 2^(i / 64) * (1 + x + ... + x^5 / 120); the series
// leaves off x^6 / 720 < 4e-17, ln2 / 64 is taken as the sum of two doubles.
__device__ __forceinline__ double exp_neg(double z, const double* tab) {
    if (!(z > -708.0)) return 0.0;
    const double n = rint(z * 92.33248261689366);                   // 64 / ln 2
    const double x = fma(n, -3.623510646634843e-19, fma(n, -0.010830424696249145, z));
    const int k = (int)n;
    double e = fma(x, 1.0 / 120, 1.0 / 24);
    e = fma(x, e, 1.0 / 6);
    e = fma(x, e, 0.5);
    e = fma(x, e, 1.0);
    e = fma(x, e, 1.0);
    return ldexp(tab[k & 63] * e, k >> 6);
}

__device__ __forceinline__ u64 to_units(const Row& r, double w) {   // w * 2^s rounded to an integer (< 2^52)
    return __double_as_longlong(w * r.unit + 4503599627370496.0) & 0xfffffffffffffull;
}
__device__ __forceinline__ u64 weight(const Row& r, float l, const double* tab) {
    return to_units(r, exp_neg(log_weight(r, l), tab));
}

// The kept set so far: keys above `key`, and of those equal to it the indices up to `idx`.
struct Border {
    uint32_t key, idx;
};
__device__ __forceinline__ bool inside(const Border& b, uint32_t key, uint32_t i) {
    return key > b.key || (key == b.key && i <= b.idx);
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
    double tab[64];
    union {
        struct {
            u64 mass[kBins];
            uint32_t count[kBins];
        };
        u64 run[kList];
    };
    union {
        u64 list[kList];
        struct {
            u64 sum[kTiles];
            uint32_t ties[kTiles];
        } tiles;
    };
    u64 wsum[kWaves];
    float wmax[kWaves], wexp[kWaves];
    u64 found_mass, found_total, rest_mass;
    uint32_t found_bin, found_above, found_count, n_list, rest_count, found_tile;
};

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
// Counts and masses of a row's elements by bin.  SUB false: bins of bin_of(), the rest apart; true: ranges of 2^shift keys
// below khi, elements from klo to khi only.
template <typename T, bool SUB>
__device__ void histogram(const SampleArgs& a, const T* row, const Row& r, const Border& in, uint32_t klo, uint32_t khi,
                          int shift, Shared& sh) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) sh.mass[b] = 0, sh.count[b] = 0;
    if (threadIdx.x == 0) sh.rest_mass = 0, sh.rest_count = 0;
    __syncthreads();
    u64 rest = 0;
    uint32_t n_rest = 0;
    for (uint32_t i = threadIdx.x * 4; i < a.V; i += kThreads * 4) {
        float v[4];
        load4(row, i, a.V, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!candidate(v[e])) continue;
            const uint32_t key = key_of(v[e]);
            if (!inside(in, key, i + e)) continue;
            int b;
            if constexpr (SUB) {
                if (key < klo || key > khi) continue;
                b = (int)((khi - key) >> shift);
            } else {
                b = bin_of(r, v[e]);
            }
            const u64 w = weight(r, v[e], sh.tab);
            if (!SUB && b == kBins) {
                rest += w;
                ++n_rest;
            } else {
                atomicAdd(&sh.mass[b], w);
                atomicAdd(&sh.count[b], 1u);
            }
        }
    }
    if (!SUB && n_rest) {
        atomicAdd(&sh.rest_mass, rest);
        atomicAdd(&sh.rest_count, n_rest);
    }
    __syncthreads();
}

// The first bin at which the running count (mass) reaches `target` (> 0): its number, what lies above it, and its count.
// kBins where the bins do not reach it.  *total_mass: of all bins and the rest.
__device__ void find_bin(bool by_mass, u64 target, double share, Shared& sh) {
    const uint32_t c0 = sh.count[2 * threadIdx.x], c1 = sh.count[2 * threadIdx.x + 1];
    const u64 m0 = sh.mass[2 * threadIdx.x], m1 = sh.mass[2 * threadIdx.x + 1];
    u64 n_all, m_all;
    const u64 n_in = block_incl((u64)c0 + c1, sh, &n_all), n_ex = n_in - c0 - c1;
    const u64 m_in = block_incl(m0 + m1, sh, &m_all), m_ex = m_in - m0 - m1;
    const u64 total = m_all + sh.rest_mass;
    if (by_mass && share >= 0.0) {
        target = (u64)ceil(share * (double)total);
        target = target < 1 ? 1 : target > total ? total : target;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sh.found_bin = kBins;
        sh.found_above = (uint32_t)n_all;
        sh.found_mass = m_all;
        sh.found_count = sh.rest_count;
        sh.found_total = target;
    }
    __syncthreads();
    const u64 ex = by_mass ? m_ex : n_ex, first = by_mass ? m0 : c0, in = by_mass ? m_in : n_in;
    if (ex < target && target <= in) {
        const bool second = ex + first < target;
        sh.found_bin = 2 * threadIdx.x + second;
        sh.found_above = (uint32_t)(second ? n_ex + c0 : n_ex);
        sh.found_mass = second ? m_ex + m0 : m_ex;
        sh.found_count = second ? c1 : c0;
    }
    __syncthreads();
}

// The largest key with bin_of >= b (kLowestKey - 1: none); every wave searches for itself, 64 keys at a time.
__device__ uint32_t last_key_of_bin(const Row& r, int b) {
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

__device__ __forceinline__ u64 entry(uint32_t key, uint32_t i) { return ((u64)key << 32) | (uint32_t)~i; }

// Sorts the list's first n entries (padded with zeros to a power of two); DESC: the largest first.
template <bool DESC>
__device__ void sort_list(uint32_t n, Shared& sh) {
    uint32_t m = 2;
    while (m < n) m <<= 1;
    for (uint32_t i = n + threadIdx.x; i < m; i += kThreads) sh.list[i] = DESC ? 0 : ~0ull;
    __syncthreads();
    for (uint32_t size = 2; size <= m; size <<= 1)
        for (uint32_t stride = size / 2; stride > 0; stride >>= 1) {
            for (uint32_t t = threadIdx.x; t < m / 2; t += kThreads) {
                const uint32_t i = 2 * t - (t & (stride - 1)), j = i + stride;
                const u64 x = sh.list[i], y = sh.list[j];
                const bool up = ((i & size) != 0) == DESC;
                if ((x > y) == up && x != y) sh.list[i] = y, sh.list[j] = x;
            }
            __syncthreads();
        }
}

// Appends the elements of `in` with klo <= key <= khi to the list (their number is known to fit).
template <typename T>
__device__ void gather(const SampleArgs& a, const T* row, const Border& in, uint32_t klo, uint32_t khi, Shared& sh) {
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x * 4; i < a.V; i += kThreads * 4) {
        float v[4];
        load4(row, i, a.V, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!candidate(v[e])) continue;
            const uint32_t key = key_of(v[e]);
            if (key < klo || key > khi || !inside(in, key, i + e)) continue;
            const uint32_t at = atomicAdd(&sh.n_list, 1u);
            if (at < kList) sh.list[at] = entry(key, i + e);
        }
    }
    __syncthreads();
}

// Narrows `in` to its first elements in (l descending, index ascending) order: as many as hold `target` (by count), or the
// share `share` of the mass (by mass).  Returns true when the result's bin and all above fit the list: then nothing is
// narrowed, *klo is the lowest key that the list needs, and *units the mass that the share stands for.
template <typename T>
__device__ bool narrow(const SampleArgs& a, const T* row, const Row& r, Border& in, bool by_mass, u64 target, double share,
                       uint32_t* klo_out, u64* units, Shared& sh) {
    histogram<T, false>(a, row, r, in, 0, 0, 0, sh);
    find_bin(by_mass, target, share, sh);
    target = sh.found_total;
    *units = target;
    const uint32_t bin = sh.found_bin;
    uint32_t above = sh.found_above, count = sh.found_count;
    u64 mass_above = sh.found_mass;
    uint32_t khi = last_key_of_bin(r, bin), klo = bin == kBins ? kLowestKey : last_key_of_bin(r, bin + 1) + 1;
    __syncthreads();
    if (!by_mass && bin == kBins && target >= (u64)above + count) {  // there are no more candidates than that
        *klo_out = kLowestKey;
        return above + count <= kList;
    }
    if (above + count <= kList) {
        *klo_out = klo;
        return true;
    }
    while (count > kList && klo < khi) {
        const uint32_t span = khi - klo;
        const int bits = 32 - __clz(span), shift = bits > 11 ? bits - 11 : 0;
        histogram<T, true>(a, row, r, in, klo, khi, shift, sh);
        find_bin(by_mass, target - (by_mass ? mass_above : above), -1.0, sh);
        const uint32_t sub = sh.found_bin;
        above += sh.found_above;
        mass_above += sh.found_mass;
        count = sh.found_count;
        khi -= sub << shift;
        klo = khi - klo > (1u << shift) - 1 ? khi - ((1u << shift) - 1) : klo;
        __syncthreads();
    }
    const u64 need = target - (by_mass ? mass_above : above);       // of the border's bin, > 0
    if (count <= kList) {
        gather(a, row, in, klo, khi, sh);
        sort_list<true>(count, sh);
        u64 last;
        if (by_mass) {
            u64 carry = 0;
            if (threadIdx.x == 0) sh.found_bin = count - 1;
            for (uint32_t i0 = 0; i0 < count; i0 += kThreads) {
                const uint32_t i = i0 + threadIdx.x;
                const u64 w = i < count ? weight(r, value_of((uint32_t)(sh.list[i] >> 32)), sh.tab) : 0;
                u64 all;
                const u64 upto = carry + block_incl(w, sh, &all);
                if (i < count && upto >= need && upto - w < need) sh.found_bin = i;
                carry += all;
            }
            __syncthreads();
            last = sh.list[sh.found_bin];
        } else {
            last = sh.list[need - 1];
        }
        in.key = (uint32_t)(last >> 32);
        in.idx = ~(uint32_t)last;
        __syncthreads();
        return false;
    }
    // one key: the r-th of its indices, by counts of tiles
    u64 rank = need;
    if (by_mass) {
        const u64 w = weight(r, value_of(khi), sh.tab);
        rank = w ? (need + w - 1) / w : 1;
    }
    rank = rank > count ? count : rank;
    const uint32_t tiles = (a.V + a.tile - 1) / a.tile;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t t = wave; t < tiles; t += kWaves) {
        uint32_t n = 0;
        const uint32_t end = a.V - t * a.tile < a.tile ? a.V : (t + 1) * a.tile;
        for (uint32_t i = t * a.tile + lane * 4; i < end; i += 256) {
            float v[4];
            load4(row, i, end, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) n += candidate(v[e]) && key_of(v[e]) == khi && inside(in, khi, i + e);
        }
        for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
        if (lane == 0) sh.tiles.ties[t] = n;
    }
    __syncthreads();
    {
        const u64 n = threadIdx.x < tiles ? sh.tiles.ties[threadIdx.x] : 0;
        u64 all;
        const u64 upto = block_incl(n, sh, &all);
        if (upto >= rank && upto - n < rank) sh.found_tile = threadIdx.x, sh.found_mass = upto - n;
        __syncthreads();
    }
    {
        const uint32_t t = sh.found_tile;
        uint32_t left = (uint32_t)(rank - sh.found_mass);           // the left-th tie of this tile
        const uint32_t end = a.V - t * a.tile < a.tile ? a.V : (t + 1) * a.tile;
        if (wave == 0) {
            for (uint32_t i0 = t * a.tile; i0 < end; i0 += 64) {
                const uint32_t i = i0 + lane;
                const bool tie = i < end && candidate((float)row[i]) && key_of((float)row[i]) == khi && inside(in, khi, i);
                const u64 ties = __ballot(tie);
                const uint32_t n = __popcll(ties);
                if (n < left) {
                    left -= n;
                    continue;
                }
                if (tie && __popcll(ties & ((1ull << lane) - 1)) == left - 1) sh.found_bin = i;
                break;
            }
        }
        __syncthreads();
        in.key = khi;
        in.idx = sh.found_bin;
        __syncthreads();
    }
    return false;
}

__device__ __forceinline__ u64 draw_target(const SampleArgs& a, int64_t at, u64 total) {
    const double u = a.u64bit ? ((const double*)a.u)[at] : (double)((const float*)a.u)[at];
    const double t = u > 0.0 ? u * (double)total : 0.0;             // NaN counts as 0
    return t < (double)total ? ((u64)t < total ? (u64)t : total - 1) : total - 1;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int64_t b = blockIdx.x;
    const T* row = (const T*)a.logits + b * a.ld;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x < 64) sh.tab[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
    double t = a.temperature ? (double)a.temperature[b] : a.t;
    int64_t k = a.top_k ? a.top_k[b] : a.k;
    const double p = a.top_p ? (double)a.top_p[b] : a.p, mp = a.min_p ? (double)a.min_p[b] : a.mp;
    if (!(t > 0.0) || t > 3e38) t = 1.0, k = 1;
    // ---- the maximum, and the mass as far as fp32 tells it (for the scale alone)
    const float c = (float)(1.4426950408889634 / t);
    float m = -__builtin_inff(), s = 0.f;
    for (uint32_t i = threadIdx.x * 4; i < a.V; i += kThreads * 4) {
        float v[4];
        load4(row, i, a.V, v);
        float vm = m;
#pragma unroll
        for (int e = 0; e < 4; ++e) vm = fmaxf(vm, v[e]);
        if (vm > m) {
            s = candidate(m) ? s * exp2f((m - vm) * c) : 0.f;
            m = vm;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (candidate(v[e])) s += v[e] == m ? 1.f : exp2f((v[e] - m) * c);
    }
    auto join = [&](float om, float os) {
        const float top = fmaxf(m, om);
        if (!candidate(top)) return;
        s = (m == top ? s : candidate(m) ? s * exp2f((m - top) * c) : 0.f) +
            (om == top ? os : candidate(om) ? os * exp2f((om - top) * c) : 0.f);
        m = top;
    };
    for (int d = 1; d < 64; d <<= 1) join(__shfl_xor(m, d), __shfl_xor(s, d));
    if (lane == 0) sh.wmax[wave] = m, sh.wexp[wave] = s;
    __syncthreads();
    m = sh.wmax[0], s = sh.wexp[0];
    for (int i = 1; i < kWaves; ++i) join(sh.wmax[i], sh.wexp[i]);
    if (!candidate(m)) {                                             // nothing to draw from
        for (int q = threadIdx.x; q < a.draws; q += kThreads) a.ids[b * a.draws + q] = -1, a.probs[b * a.draws + q] = 0.f;
        return;
    }
    int ex;
    (void)frexpf(s * 1.25f, &ex);                                    // the mass is below 2^ex, rounding of s included
    Row r;
    r.lmax = m;
    r.inv_t = 1.0 / t;
    r.bin_scale = (float)(64.0 / t);
    r.log_min_p = mp > 0.0 ? log(mp < 1.0 ? mp : 1.0) : -__builtin_inf();
    r.unit = ldexp(1.0, min(51, 62 - ex));
    // ---- the border of the kept set
    Border in = {0, 0};                                              // key 0 is below every candidate: all are inside
    uint32_t klo = kLowestKey;
    u64 units = 0, unused;                                           // units: the mass top_p stands for, once it is known
    bool listed = a.V <= kList;
    if (!listed && k > 0 && k < a.V) listed = narrow<T>(a, row, r, in, false, (u64)k, -1.0, &klo, &unused, sh);
    if (!listed && p < 1.0) listed = narrow<T>(a, row, r, in, true, 0, p > 0.0 ? p : 0.0, &klo, &units, sh);
    if (listed) {
        gather(a, row, in, klo, 0xffffffffu, sh);
        const uint32_t n = sh.n_list;
        uint32_t keep = n;
        if ((k > 0 && k < n) || p < 1.0) {
            sort_list<true>(n, sh);
            if (k > 0 && k < n) keep = (uint32_t)k;
        }
        if (p < 1.0) {
            u64 target = units, all, carry = 0;
            if (target == 0) {
                u64 total = 0;
                for (uint32_t i0 = 0; i0 < keep; i0 += kThreads) {
                    const uint32_t i = i0 + threadIdx.x;
                    block_incl(i < keep ? weight(r, value_of((uint32_t)(sh.list[i] >> 32)), sh.tab) : 0, sh, &all);
                    total += all;
                }
                target = (u64)ceil((p > 0.0 ? p : 0.0) * (double)total);
                target = target < 1 ? 1 : target > total ? total : target;
            }
            if (threadIdx.x == 0) sh.found_bin = keep - 1;
            for (uint32_t i0 = 0; i0 < keep; i0 += kThreads) {
                const uint32_t i = i0 + threadIdx.x;
                const u64 w = i < keep ? weight(r, value_of((uint32_t)(sh.list[i] >> 32)), sh.tab) : 0;
                const u64 upto = carry + block_incl(w, sh, &all);
                if (i < keep && upto >= target && upto - w < target) sh.found_bin = i;
                carry += all;
            }
            __syncthreads();
            keep = sh.found_bin + 1;
            __syncthreads();
        }
        // the kept entries in index order, those below min_p with weight zero
        for (uint32_t i = threadIdx.x; i < keep; i += kThreads) {
            const u64 x = sh.list[i];
            sh.list[i] = ((u64)(~(uint32_t)x) << 32) | (uint32_t)(x >> 32);
        }
        __syncthreads();
        sort_list<false>(keep, sh);
        u64 carry = 0;
        for (uint32_t i0 = 0; i0 < keep; i0 += kThreads) {
            const uint32_t i = i0 + threadIdx.x;
            u64 w = 0, all;
            if (i < keep) {
                const float l = value_of((uint32_t)sh.list[i]);
                if (log_weight(r, l) >= r.log_min_p) w = weight(r, l, sh.tab);
            }
            const u64 upto = carry + block_incl(w, sh, &all);
            if (i < keep) sh.run[i] = upto;
            carry += all;
        }
        __syncthreads();
        const u64 total = carry;
        for (int q = threadIdx.x; q < a.draws; q += kThreads) {
            const u64 want = draw_target(a, b * a.draws + q, total);
            uint32_t lo = 0, hi = keep - 1;                          // the first with a running sum above `want`
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (sh.run[mid] > want) hi = mid;
                else lo = mid + 1;
            }
            const u64 x = sh.list[lo];
            a.ids[b * a.draws + q] = (int64_t)(x >> 32);
            a.probs[b * a.draws + q] = (float)(exp_neg(log_weight(r, value_of((uint32_t)x)), sh.tab) * r.unit / (double)total);
        }
        return;
    }
    // ---- a kept set that does not fit the list: running sums of tiles, then the tile that holds the draw
    const uint32_t tiles = (a.V + a.tile - 1) / a.tile;
    auto kept_weight = [&](float l, uint32_t i) -> u64 {
        if (!candidate(l) || !inside(in, key_of(l), i)) return 0;
        const double z = log_weight(r, l);
        return z >= r.log_min_p ? to_units(r, exp_neg(z, sh.tab)) : 0;
    };
    for (uint32_t tl = wave; tl < tiles; tl += kWaves) {
        u64 w = 0;
        const uint32_t end = a.V - tl * a.tile < a.tile ? a.V : (tl + 1) * a.tile;
        for (uint32_t i = tl * a.tile + lane * 4; i < end; i += 256) {
            float v[4];
            load4(row, i, end, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) w += kept_weight(v[e], i + e);
        }
        w = wave_incl(w);
        if (lane == 63) sh.tiles.sum[tl] = w;
    }
    __syncthreads();
    u64 total;
    {
        const u64 w = threadIdx.x < tiles ? sh.tiles.sum[threadIdx.x] : 0;
        const u64 upto = block_incl(w, sh, &total);
        if (threadIdx.x < tiles) sh.tiles.sum[threadIdx.x] = upto;
        __syncthreads();
    }
    for (int q = wave; q < a.draws; q += kWaves) {
        const u64 want = draw_target(a, b * a.draws + q, total);
        uint32_t lo = 0, hi = tiles - 1;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (sh.tiles.sum[mid] > want) hi = mid;
            else lo = mid + 1;
        }
        u64 before = lo ? sh.tiles.sum[lo - 1] : 0;
        const uint32_t end = a.V - lo * a.tile < a.tile ? a.V : (lo + 1) * a.tile;
        for (uint32_t i0 = lo * a.tile; i0 < end; i0 += 64) {
            const uint32_t i = i0 + lane;
            const float l = i < end ? (float)row[i] : __builtin_nanf("");
            const u64 w = kept_weight(l, i);
            const u64 upto = before + wave_incl(w);
            const u64 hit = __ballot(upto > want);
            if (hit) {
                if (lane == __ffsll((long long)hit) - 1) {
                    a.ids[b * a.draws + q] = i;
                    a.probs[b * a.draws + q] = (float)(exp_neg(log_weight(r, l), sh.tab) * r.unit / (double)total);
                }
                break;
            }
            before = ((u64)__shfl((uint32_t)(upto >> 32), 63) << 32) | __shfl((uint32_t)upto, 63);
        }
    }
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
