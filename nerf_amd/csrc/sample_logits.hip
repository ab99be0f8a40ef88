// Indices drawn from rows of logits: temperature, top-k, top-p, min-p, then the inverse of the distribution at given uniform
// numbers, in the order of the index (sample_pdf's rule for a discrete distribution).
//
// Row x[V], maximum M, masses e_i = exp((x_i - M) / T).  The entries stand in falling order, ties by rising index; kept are the
// first k of them, of those the shortest prefix that holds p of their mass, and of that the ones with e_i >= m (the first one
// always).  A draw is the first kept index whose running mass exceeds u times the kept mass S; prob = e / S.
//
// An index has to be exact, so masses and running sums are f64: errors near 1e-15 against gaps of e / S.  exp is a table of
// 16 values of 2^(j/16) and a polynomial, about 14 f64 instructions (the library's is several times that), and entries
// that the filters have already excluded are not evaluated.
//
// The cut (the last kept entry, by value and index) is found among few entries:
//   - top-k with k up to some 1500: the row is split into 4096 groups, and the k-th largest of the groups' maxima bounds the k-th
//     largest entry from below.  The entries above that bound (a few more than k) go into a list in LDS.
//   - else a histogram of the row, 2048 bins of equal width below the maximum, counts and masses.  Masses are added there as 64-bit
//     integers, because these give the same sums in any order, in units that go down with the bin's masses, and are f64 from then on:
//     an entry is right to 2^-42 of the largest mass its bin could hold, however small that is.  The bin of the cut, or all entries
//     down to it, go into the list.  A bin that holds more than the list (many equal values, far outliers) is split again by the bits of
//     its values until it does not, or holds one value only.
// The list (up to 2048 entries) is sorted.  Where it holds everything that is kept, the draws come from it; else from the
// masses of the row's tiles of 1024 entries.
//
// Three forms: short rows without a cut, a wave each (4096 rows of 1001 f32: 11 us); one block a row; and, for few long rows, 32 or 64
// blocks a row over several launches (4096 draws from 640000 f32, top-p: 48 us in five; one of 131072 by top-k: 16 us in two), where the
// block that arrives last at a stage's end does what needs the whole row.
// Of one block a row, 256 rows of 131072 bf16: by top-k 1000 and top-p 34 us, of which 15 are the pass for the maximum (4.5 TB/s), 3 the
// bound, 6 the list and 11 its two sorts, cuts and the draw, with no other block on the CU and the vector units busy 30 % of the whole; by
// top-p alone 127 us, vector units busy 66 %: 12 maximum, 45 histogram, 21 cut (bf16 ties overflow the list), 49 masses of the tiles and the draw.
#include <algorithm>
#include "nrf_types.h"

using namespace nrf;

namespace {

constexpr int kBins = 2048, kList = 2048, kGroups = 4096, kMaxTiles = 1024;
constexpr int kMaxSize = 1 << 28, kMaxRows = 1 << 21;
constexpr int kSegment = 1 << 20;           // entries whose masses a word of the histogram holds
constexpr int kParts = 32;                  // blocks of a row, many-block form
constexpr int kCrowd = 160;                 // entries of a bucket from which sort_list falls back
constexpr int kGroupsMaxK = 1500;           // above it the groups' bound lets more entries through than the list holds

struct SampleArgs {
    const void *logits;
    int64_t stride;
    const float *u;                                  // [rows, draws]
    const float *temperature_v, *top_p_v, *min_p_v;  // per row, or null: the scalars below
    const int32_t *top_k_v;
    float temperature, top_p, min_p;
    int32_t top_k;
    int32_t rows, size, draws;
    int64_t *ids;
    float *prob;
};

// ---- values
// Order-preserving key of a logit: larger value, larger key; -0 and +0 alike.  0 stands for entries that are never drawn (NaN, -inf).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    return x > -__builtin_inff() ? k : 0u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// 2^(j/16)
__constant__ double kRoots[16] = {
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0, 0x1.306fe0a31b715p+0,
    0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0, 0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0,
    0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0, 0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0,
    0x1.ea4afa2a490dap+0};

struct Row {
    double top, inv_t;      // M and 1 / T (0 at T = 0)
    float topf;
    bool flat;              // M = +inf or T = 0: mass 1 at M, 0 elsewhere
    const double *tab;      // 2^(j/16), LDS
};

// exp(y), y = (x - M) / T <= 0: y = (16 q + j) ln2 / 16 + r, |r| <= ln2 / 32, exp = 2^q tab[j] exp(r); the Taylor polynomial of
// degree 6 leaves r^7 / 5040 < 5e-16.  x = M gives 1 exactly; -inf and NaN end in the clamp's 2^-4328, which is 0.  2^up (up to 2^2200)
// times that, with the one rounding.
__device__ __forceinline__ double mass_of(const Row &w, float x, int up = 0) {
    if (w.flat) return x == w.topf ? __builtin_ldexp(1.0, up) : 0.0;
    const double y = fmax(((double)x - w.top) * w.inv_t, -3000.0);
    const double n = __builtin_rint(y * (16.0 * 1.44269504088896340736));
    const double r = fma(n, -0.69314718055994530942 / 16.0, y);
    double s = fma(r, 1.0 / 720.0, 1.0 / 120.0);
    s = fma(r, s, 1.0 / 24.0);
    s = fma(r, s, 1.0 / 6.0);
    s = fma(r, s, 0.5);
    s = fma(r, s, 1.0);
    s = fma(r, s, 1.0);
    const int q = (int)n;
    return __builtin_ldexp(s * w.tab[q & 15], (q >> 4) + up);
}

// Bin of the first histogram: equal widths below the maximum, the last bin open.  Every step is monotone in x.
__device__ __forceinline__ int bin_of(const Row &w, float scale, float x) {
    return (int)fminf((w.topf - x) * scale, (float)(kBins - 1));
}

// 16-byte pieces of a row, at any alignment of its elements
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    static constexpr int E = 16 / sizeof(T);
    T e[E];
};

// f(x, i, u) for the entries begin .. end of a row, 16 bytes a load (at any alignment of the elements), four loads in flight;
// u: which of the four the entry came in (0 for the odd ones at the end).
template <int BLOCK, int U = 4, typename T, typename F>
__device__ __forceinline__ void for_each(const T *row, int begin, int end, F f) {
    constexpr int E = Vec<T>::E;
    const Vec<T> *v = reinterpret_cast<const Vec<T> *>(row + begin);
    const int n = (end - begin) / E;
    for (int j = threadIdx.x; j < n; j += BLOCK * U) {
        Vec<T> p[U];
#pragma unroll
        for (int u = 0; u < U; ++u) p[u] = v[min(j + u * BLOCK, n - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u * BLOCK < n) {
#pragma unroll
                for (int e = 0; e < E; ++e) f(to_f32(p[u].e[e]), begin + (j + u * BLOCK) * E + e, u);
            }
    }
    const int i = begin + n * E + threadIdx.x;
    if (i < end) f(to_f32(row[i]), i, 0);
}

// What is the same in all lanes, into scalar registers.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(uniform(__float_as_uint(v))); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) {
    return ((uint64_t)uniform((uint32_t)(v >> 32)) << 32) | uniform((uint32_t)v);
}

// ---- block-wide helpers (BLOCK threads, all of them call)
template <int BLOCK> struct Shared {
    static constexpr int kWaves = BLOCK / 64;
    double tab[16];
    double wave_d[kWaves];
    uint64_t wave_u[kWaves];
    uint32_t wave_a[kWaves];
    int32_t wave_last[kWaves];
    uint32_t count;                    // entries in `list`
    uint64_t found[3];                 // what one thread found for all
    int32_t first, back;               // find_bin
    uint32_t crowded, bucket[kBins];   // sort_list
    uint64_t list[kList];
    double mass[kList];
};
struct Histogram {
    uint32_t cnt[kBins];
    union {
        uint64_t word[kBins];          // while entries are added: fixed point, see `raise`
        double mass[kBins];            // afterwards
    };
};

// The value of the lane that DPP control CTRL names, 0 where there is none (4- and 8-byte types)
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V dpp(V v) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    } else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(V, ((uint64_t)hi << 32) | lo);
    }
}

// Inclusive sums over the lanes of a wave: shifts inside rows of 16, then the rows' last lanes (all lanes must be active)
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
    v += dpp<0x111, 0xf>(v);      // row_shr:1
    v += dpp<0x112, 0xf>(v);      // row_shr:2
    v += dpp<0x114, 0xf>(v);      // row_shr:4
    v += dpp<0x118, 0xf>(v);      // row_shr:8
    v += dpp<0x142, 0xa>(v);      // row_bcast:15 into rows 1 and 3
    v += dpp<0x143, 0xc>(v);      // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ double last_lane(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)b, 63), hi = __builtin_amdgcn_readlane((uint32_t)(b >> 32), 63);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// Largest of the lanes (the same moves; lanes without a source keep their own value)
__device__ __forceinline__ float wave_max(float v) {
#define NRF_DPP_MAX(ctrl, rows) \
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), ctrl, rows, 0xf, false)))
    NRF_DPP_MAX(0x111, 0xf);
    NRF_DPP_MAX(0x112, 0xf);
    NRF_DPP_MAX(0x114, 0xf);
    NRF_DPP_MAX(0x118, 0xf);
    NRF_DPP_MAX(0x142, 0xa);
    NRF_DPP_MAX(0x143, 0xc);
#undef NRF_DPP_MAX
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}
template <typename V>
__device__ __forceinline__ V lane_before(V v) { return dpp<0x138, 0xf>(v); }      // wave_shr:1

// Sum of the values of the threads before this one, in a fixed order of additions; *total = the sum of all.
template <int BLOCK, typename V, typename S>
__device__ __forceinline__ V block_scan(V v, S *sums, V *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    if (lane == 63) sums[wave] = v;
    const V before = lane_before(v);
    __syncthreads();
    V base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) {
        if (w == wave) base = all;
        all += sums[w];
    }
    __syncthreads();
    *total = all;
    return base + before;
}

template <int BLOCK>
__device__ __forceinline__ void block_max_min(float &hi, float &lo, Shared<BLOCK> &s) {
    hi = wave_max(hi), lo = -wave_max(-lo);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *w_hi = reinterpret_cast<float *>(s.wave_a), *w_lo = reinterpret_cast<float *>(s.wave_u);
    if (lane == 0) w_hi[wave] = hi, w_lo[wave] = lo;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) hi = fmaxf(hi, w_hi[w]), lo = fminf(lo, w_lo[w]);
    hi = uniform(hi), lo = uniform(lo);
    __syncthreads();
}

// Order of the entries: larger value first, then smaller index.
__device__ __forceinline__ uint64_t by_value(uint32_t key, int i) { return ((uint64_t)~key << 32) | (uint32_t)i; }

// list[0 .. n) into rising order, n <= kList.  bucket(c): 0 .. kBins - 1, rising with c.
//   few entries: each counts the smaller ones;
//   else: buckets (about as many as entries), each entry counting within its own;
//   where a bucket is crowded (equal values): bitonic, 66 steps of a barrier each for 2048 entries (18 us against 4).
template <int BLOCK, typename F>
__device__ __forceinline__ void sort_list(Shared<BLOCK> &s, int n, F bucket) {
    constexpr int kPer = kList / BLOCK;
    uint64_t c[kPer];
    if (n <= 256) {
        static_assert(BLOCK >= 256, "one entry a thread");
        const int i = threadIdx.x;
        uint32_t rank = 0;
        if (i < n) {
            c[0] = s.list[i];
#pragma unroll 8
            for (int j = 0; j < n; ++j) rank += s.list[j] < c[0];
        }
        __syncthreads();
        if (i < n) s.list[rank] = c[0];
        __syncthreads();
        return;
    }
    uint32_t *count = s.bucket;
#pragma unroll
    for (int j = 0; j < kPer; ++j) count[j * BLOCK + threadIdx.x] = 0;
    if (threadIdx.x == 0) s.crowded = 0;
    __syncthreads();
    int b[kPer];
    uint32_t at[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = j * BLOCK + threadIdx.x;
        if (i < n) {
            c[j] = s.list[i];
            b[j] = bucket(c[j]);
            at[j] = atomicAdd(&count[b[j]], 1u);
            if (at[j] == kCrowd) s.crowded = 1;
        }
    }
    __syncthreads();
    if (s.crowded) {
        int size = 512;
        while (size < n) size <<= 1;
        for (int i = n + threadIdx.x; i < size; i += BLOCK) s.list[i] = ~0ull;
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int p = threadIdx.x; p < size / 2; p += BLOCK) {
                    const int x = ((p & ~(j - 1)) << 1) | (p & (j - 1)), y = x | j;
                    const uint64_t u = s.list[x], v = s.list[y];
                    if ((u > v) == ((x & k) == 0)) s.list[x] = v, s.list[y] = u;
                }
                __syncthreads();
            }
        return;
    }
    // bucket sizes -> first places
    uint32_t mine[kPer], run = 0, all;
#pragma unroll
    for (int j = 0; j < kPer; ++j) mine[j] = count[threadIdx.x * kPer + j], run += mine[j];
    uint32_t first = block_scan<BLOCK, uint32_t>(run, s.wave_a, &all);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        count[threadIdx.x * kPer + j] = first;
        first += mine[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (j * BLOCK + (int)threadIdx.x < n) s.list[count[b[j]] + at[j]] = c[j];
    __syncthreads();
    uint32_t place[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (j * BLOCK + (int)threadIdx.x < n) {
            const uint32_t lo = count[b[j]], hi = b[j] + 1 < kBins ? count[b[j] + 1] : n;
            place[j] = lo;
#pragma unroll 8
            for (uint32_t q = lo; q < hi; ++q) place[j] += s.list[q] < c[j];
        }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (j * BLOCK + (int)threadIdx.x < n) s.list[place[j]] = c[j];
    __syncthreads();
}

// The list in the order of value, largest first: entries between base and base - kBins / mul.
template <int BLOCK>
__device__ __forceinline__ void sort_by_value(Shared<BLOCK> &s, int n, float base, float mul) {
    sort_list<BLOCK>(s, n, [=](uint64_t c) {
        return (int)fminf(fmaxf((base - value_of(~(uint32_t)(c >> 32))) * mul, 0.0f), (float)(kBins - 1));
    });
}

// Entries 0 .. n of the list from the order of value to that of the index, as (index, key).
template <int BLOCK>
__device__ __forceinline__ void list_by_index(Shared<BLOCK> &s, int n, int size) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += BLOCK) {
        const uint64_t c = s.list[i];
        s.list[i] = (c << 32) | (uint32_t)~(uint32_t)(c >> 32);
    }
    __syncthreads();
    int shift = 0;
    while ((size - 1) >> shift >= kBins) ++shift;
    sort_list<BLOCK>(s, n, [=](uint64_t c) { return (int)((uint32_t)(c >> 32) >> shift); });
}

struct Filter {
    int k;                  // entries kept by top-k: 1 .. size
    double p;               // < 1: top-p
    double m;
    bool cut;               // k or p leaves something out
    uint32_t key;           // the last kept entry
    int32_t idx;
    __device__ __forceinline__ bool keeps(uint32_t x, int i) const { return x > key || (x == key && i <= idx); }
};

__device__ __forceinline__ double kept_mass(const Row &w, const Filter &f, float x, int i) {
    if (f.cut && !f.keeps(key_of(x), i)) return 0.0;
    const double e = mass_of(w, x);
    return e >= f.m ? e : 0.0;
}

// What stands before a place in the order: entries and their mass.
struct Above {
    uint32_t cnt;
    double mass;
};

// ---- a row's parameters
struct RowState {
    Row w;
    Filter f;
    bool valid, use_p;      // use_p: top-p leaves something out, if anything does
    float t, scale;         // scale: bins of the first histogram
    float lift;             // log2 of how much smaller a bin's masses are than those of the bin before
    int shift;              // bits behind the point of a histogram's word, bin 0
    __device__ __forceinline__ bool plain() const { return !valid || t == 0.0f; }
};

// top, low: the largest and the smallest logit (NaN aside)
__device__ __forceinline__ RowState row_state(const SampleArgs &a, int r, float top, float low, const double *tab) {
    RowState o;
    const float p = a.top_p_v ? a.top_p_v[r] : a.top_p, m = a.min_p_v ? a.min_p_v[r] : a.min_p;
    const int k = a.top_k_v ? a.top_k_v[r] : a.top_k;
    o.t = a.temperature_v ? a.temperature_v[r] : a.temperature;
    top += 0.0f;                                           // -0 as +0
    o.valid = top > -__builtin_inff() && o.t >= 0.0f && o.t < __builtin_inff() && p == p && m == m;
    o.w.topf = top, o.w.top = top, o.w.tab = tab;
    o.w.flat = o.t == 0.0f || top == __builtin_inff();
    o.w.inv_t = o.w.flat ? 0.0 : 1.0 / (double)o.t;
    o.f.k = k <= 0 || k > a.size ? a.size : k;
    o.f.p = p, o.f.m = fmin((double)m, 1.0);
    o.use_p = p < 1.0f;
    o.f.cut = o.f.k < a.size || o.use_p;
    o.f.key = 0, o.f.idx = a.size;
    // 64 temperatures reach masses of 1e-28; top-k, which does not look at masses, gets some room where they are narrow
    o.scale = fminf((float)kBins / fminf(top - low, fmaxf(64.0f * o.t, 16.0f)), 1e30f);
    // (scale 0, or so small that bins end beyond f32's range, leaves bins without an order of mass: no lift)
    o.lift = o.w.flat || o.scale == 0.0f ? 0.0f : fminf(1.44269504f / (o.scale * o.t), 1.0f);
    o.shift = 62;
    for (int v = min(a.size, kSegment); v > 0; v >>= 1) --o.shift;
    o.shift = min(o.shift, 50);
    return o;
}

// Masses of a histogram are added as 64-bit integers, which give the same sums in any order.  A bin's unit goes down with its masses:
// the entries of bin b weigh at most 2^(-b lift) (but for some 1e-3 that f32 rounds into the bin), so e * 2^raise <= 2^shift * 1.001 and
// the words of kSegment entries stay below 2^63.  An entry is held to half a unit, 2^-42 of its bin's largest at kSegment entries
// (the last bin has no lower end, but what begins there weighs e^-64 and less).
__device__ __forceinline__ int raise(const RowState &o, int bin) { return o.shift + (int)((float)bin * o.lift); }
// Nearest integer of 0 <= v < 2^52: the bits of 2^52 + v behind those of 2^52 (shift is at most 50: rows in a histogram have more than
// 2048 entries)
__device__ __forceinline__ uint64_t fixed(double v) { return __builtin_bit_cast(uint64_t, v + 0x1p52) - __builtin_bit_cast(uint64_t, 0x1p52); }

// Lowest index in begin .. end that holds x (size where none does)
template <int BLOCK, typename T>
__device__ __forceinline__ int find_value(Shared<BLOCK> &s, const T *row, int begin, int end, float x, int size) {
    int at = size;
    for_each<BLOCK>(row, begin, end, [&](float v, int i, int) { at = v == x ? min(at, i) : at; });
#pragma unroll
    for (int d = 32; d; d >>= 1) at = min(at, __shfl_xor(at, d));
    if ((threadIdx.x & 63) == 0) s.wave_a[threadIdx.x >> 6] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) at = min(at, (int)s.wave_a[w]);
    __syncthreads();
    return at;
}

template <int BLOCK>
__device__ __forceinline__ void clear_histogram(Histogram &h) {
    for (int b = threadIdx.x; b < kBins; b += BLOCK) h.cnt[b] = 0, h.word[b] = 0;
    __syncthreads();
}

template <int BLOCK, typename T>
__device__ __forceinline__ void add_counts(Histogram &h, const RowState &o, const T *row, int begin, int end) {
    for_each<BLOCK>(row, begin, end, [&](float x, int, int) {
        if (key_of(x)) atomicAdd(&h.cnt[bin_of(o.w, o.scale, x)], 1u);
    });
    __syncthreads();
}

// Counts and words of begin .. end, at most kSegment entries.  bin(x, key): below 0 for entries of no bin; up(b): the unit of bin b
template <int BLOCK, typename T, typename B, typename X>
__device__ __forceinline__ void add_words(Histogram &h, const RowState &o, const T *row, int begin, int end, B bin, X up) {
    for_each<BLOCK, 1>(row, begin, end, [&](float x, int, int) {
        const uint32_t key = key_of(x);
        const int b = bin(x, key);
        if (b >= 0) {
            atomicAdd(&h.cnt[b], 1u);
            atomicAdd((unsigned long long *)&h.word[b], (unsigned long long)fixed(mass_of(o.w, x, up(b))));
        }
    });
    __syncthreads();
}

// Counts and masses of a whole row; a thread adds up its bins' words behind each segment.
template <int BLOCK, typename T, typename B, typename X>
__device__ __forceinline__ void fill_histogram(Histogram &h, const RowState &o, const T *row, int size, B bin, X up) {
    constexpr int kPer = kBins / BLOCK;
    double sum[kPer] = {};
    clear_histogram<BLOCK>(h);
    for (int begin = 0; begin < size; begin += kSegment) {
        add_words<BLOCK, T>(h, o, row, begin, min(size, begin + kSegment), bin, up);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int b = j * BLOCK + threadIdx.x;
            sum[j] += __builtin_ldexp((double)h.word[b], -up(b));
            h.word[b] = 0;
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) h.mass[j * BLOCK + threadIdx.x] = sum[j];
    __syncthreads();
}
template <int BLOCK, typename T>
__device__ __forceinline__ void fill_histogram(Histogram &h, const RowState &o, const T *row, int size) {
    fill_histogram<BLOCK, T>(h, o, row, size, [&](float x, uint32_t key) { return key ? bin_of(o.w, o.scale, x) : -1; },
                             [&](int b) { return raise(o, b); });
}

// ---- the cut
// In a sorted list whose first entry has `above` before it: the last of the entries that are among the first `last` and have less
// than `want` of mass before them (by_mass).  Returns how many entries of the list that keeps; mass_at: mass up to entry `last`.
template <int BLOCK>
__device__ __forceinline__ int cut_list(Shared<BLOCK> &s, const RowState &o, Filter &f, int n, Above above, int last, bool by_mass, double p,
                        double want, double *mass_at) {
    constexpr int kPer = kList / BLOCK;
    double e[kPer], run = 0.0, all;
    const int i0 = threadIdx.x * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        e[j] = i0 + j < n ? mass_of(o.w, value_of(~(uint32_t)(s.list[i0 + j] >> 32))) : 0.0;
        run += e[j];
    }
    double before = above.mass + block_scan<BLOCK, double>(run, s.wave_d, &all);
    if (last <= n) {
        double b = before;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            b += e[j];
            if (i0 + j == last - 1) s.found[0] = __builtin_bit_cast(uint64_t, b);
        }
        __syncthreads();
        *mass_at = __builtin_bit_cast(double, uniform(s.found[0]));
        __syncthreads();
        if (p >= 0.0) want = p * *mass_at;                             // top-p of the mass found here
    }
    uint32_t mine = 0, kept;                                           // a prefix: counting is enough
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const bool first = above.cnt == 0 && i0 + j == 0;
        if (i0 + j < min(n, last) && (!by_mass || before < want || first)) ++mine;
        before += e[j];
    }
    block_scan<BLOCK, uint32_t>(mine, s.wave_a, &kept);
    kept = uniform(kept);
    const uint64_t c = uniform(s.list[kept > 0 ? kept - 1 : 0]);
    f.key = ~(uint32_t)(c >> 32);
    f.idx = (int)(uint32_t)c;
    __syncthreads();
    return (int)kept;
}

// The bin that takes the running count to `want` (by_count), or the running mass to `wantm`; adds what stands before it to
// `above` (masses only where the histogram has them).  kBins: none does by count, or all are empty.
template <int BLOCK>
__device__ __forceinline__ int find_bin(Shared<BLOCK> &s, const Histogram &h, bool by_count, bool masses, uint32_t want, double wantm, Above &above) {
    constexpr int kPer = kBins / BLOCK;
    const int b0 = threadIdx.x * kPer;
    uint32_t c[kPer], cs = 0, call;
    double m[kPer], ms = 0.0, mb = 0.0, mall;
#pragma unroll
    for (int j = 0; j < kPer; ++j) c[j] = h.cnt[b0 + j], m[j] = masses ? h.mass[b0 + j] : 0.0, cs += c[j], ms += m[j];
    if (threadIdx.x == 0) s.found[0] = kBins, s.first = kBins, s.back = -1;
    uint32_t cb = above.cnt + block_scan<BLOCK, uint32_t>(cs, s.wave_a, &call);
    if (masses) mb = above.mass + block_scan<BLOCK, double>(ms, s.wave_d, &mall);
    const uint32_t cb0 = cb;
    const double mb0 = mb;
    int hit = kBins;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (hit == kBins && c[j] && (by_count ? cb < want && cb + c[j] >= want : mb + m[j] >= wantm)) hit = b0 + j;
        cb += c[j], mb += m[j];
    }
    if (!by_count) {
        // the first of all threads' (their running masses differ by roundings, so several may see the crossing); where no one sees it,
        // the sums of a bin's parts having rounded below its own, the last bin that holds anything
        int back = -1;
#pragma unroll
        for (int j = 0; j < kPer; ++j) back = c[j] ? b0 + j : back;
        const uint64_t over = __ballot(hit < kBins), some = __ballot(back >= 0);
        const int lane = threadIdx.x & 63;
        if (over && lane == __builtin_ctzll(over)) atomicMin(&s.first, hit);
        if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&s.back, back);
        __syncthreads();
        const int bin = s.first < kBins ? s.first : s.back;
        hit = bin >= b0 && bin < b0 + kPer ? bin : kBins;
    }
    if (hit < kBins) {
        uint32_t cnt = cb0;
        double mass = mb0;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (b0 + j < hit) cnt += c[j], mass += m[j];
        s.found[0] = hit, s.found[1] = cnt, s.found[2] = __builtin_bit_cast(uint64_t, mass);
    }
    __syncthreads();
    const int bin = (int)uniform(s.found[0]);
    if (bin < kBins) above.cnt = (uint32_t)uniform(s.found[1]), above.mass = __builtin_bit_cast(double, uniform(s.found[2]));
    __syncthreads();
    return bin;
}

// One of the two cuts as the first histogram sees it: the bin it lies in, and which bins' entries to sort.
struct Step {
    bool any, by_count, prefix, fits;     // prefix: all entries down to the bin fit the list; fits: they or the bin's do
    int from, bin;
    uint32_t n;                           // entries of the bin
    Above above;                          // before bin `from`
    double wantm;
};

template <int BLOCK>
__device__ __forceinline__ Step make_step(Shared<BLOCK> &s, const Histogram &h, const RowState &o, bool by_count, double mass_k) {
    Step st;
    st.by_count = by_count;
    st.wantm = o.f.p * mass_k;
    st.above = Above{0, 0.0};
    st.bin = find_bin<BLOCK>(s, h, by_count, true, o.f.k, st.wantm, st.above);
    st.any = st.bin < kBins;
    st.n = st.any ? uniform(h.cnt[st.bin]) : 0;
    st.prefix = st.above.cnt + st.n <= (uint32_t)kList;
    st.fits = st.prefix || st.n <= (uint32_t)kList;
    st.from = st.prefix ? 0 : st.bin;
    if (st.prefix) st.above = Above{0, 0.0};
    return st;
}

// Top-k where it leaves something out, else top-p of the whole mass (known if the histogram has masses).
template <int BLOCK>
__device__ __forceinline__ Step first_step(Shared<BLOCK> &s, const Histogram &h, RowState &o) {
    constexpr int kPer = kBins / BLOCK;
    uint32_t c = 0, total;
    double m = 0.0, mass;
#pragma unroll
    for (int j = 0; j < kPer; ++j) c += h.cnt[threadIdx.x * kPer + j], m += h.mass[threadIdx.x * kPer + j];
    block_scan<BLOCK, uint32_t>(c, s.wave_a, &total);
    block_scan<BLOCK, double>(m, s.wave_d, &mass);
    total = uniform(total), mass = __builtin_bit_cast(double, uniform(__builtin_bit_cast(uint64_t, mass)));
    if (o.f.k < (int)total) return make_step<BLOCK>(s, h, o, true, 0.0);
    o.f.k = (int)total;
    if (o.use_p && mass > 0.0) return make_step<BLOCK>(s, h, o, false, mass);
    Step none{};
    return none;
}

// What a list is gathered by: all entries of the bins from .. to, or (a superset of bins 0 .. to) all entries from `least` up.
struct Reach {
    int from, to;
    float least;
    __device__ __forceinline__ Reach(int f, int t) : from(f), to(t), least(0.0f) {}
    __device__ __forceinline__ Reach(const RowState &o, int t) : from(-1), to(t) {
        // the widths of the bins, and some roundings more; never -inf
        const float width = (float)(t + 1) / o.scale;
        least = t == kBins - 1 ? -3.402823466e38f : fmaxf(o.w.topf - width * 1.000001f - fabsf(o.w.topf) * 3e-7f, -3.402823466e38f);
    }
};

__device__ __forceinline__ bool reached(const Reach &want, const RowState &o, float x) {
    if (want.from < 0) return x >= want.least;
    // before the rounding down to whole bins; the last bin has no end
    const float b = fminf((o.w.topf - x) * o.scale, (float)(kBins - 1));
    return b >= (float)want.from && b < (want.to == kBins - 1 ? __builtin_inff() : (float)(want.to + 1)) && x > -__builtin_inff();
}

// What is reached in four pieces (place j of the row and every BLOCK-th behind it), a bit an entry
template <int BLOCK, typename T>
__device__ __forceinline__ uint32_t reach_mask(const RowState &o, const Vec<T> *p, int j, int pieces, const Reach &want) {
    constexpr int E = Vec<T>::E;
    uint32_t mask = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) m |= reached(want, o, to_f32(p[u].e[e])) ? 1u << e : 0u;
        mask |= j + u * BLOCK < pieces ? m << (u * E) : 0u;
    }
    return mask;
}

// Places in the list for `n` entries of each lane: one addition a wave (all lanes call; an atomicAdd of different amounts would
// be serialised lane by lane)
__device__ __forceinline__ uint32_t reserve(uint32_t *count, uint32_t n) {
    const uint32_t to = wave_scan(n), all = __builtin_amdgcn_readlane(to, 63);
    uint32_t base = 0;
    if (all) {
        if ((threadIdx.x & 63) == 0) base = atomicAdd(count, all);
        base = uniform(base);
    }
    return base + to - n;
}

// The indices of a mask's entries into the list from place `at` on
template <int BLOCK, typename T>
__device__ __forceinline__ uint32_t put_mask(uint32_t *index, uint32_t mask, uint32_t at, int j, int begin) {
    constexpr int E = Vec<T>::E;
    while (mask) {
        const int bit = __builtin_ctz(mask);
        if (at < (uint32_t)kList) index[at] = begin + (j + bit / E * BLOCK) * E + bit % E;
        ++at;
        mask &= mask - 1;
    }
    return at;
}

// The odd entries at the end, then the values by their indices: list[0 ..), in any order, as by_value.  Returns how many are reached
// (those beyond kList are counted only).
template <int BLOCK, typename T>
__device__ __forceinline__ uint32_t finish_list(Shared<BLOCK> &s, const RowState &o, const T *row, int i, int end, const Reach &want) {
    uint32_t *index = reinterpret_cast<uint32_t *>(s.mass);
    if (i < end && reached(want, o, to_f32(row[i]))) {
        const uint32_t at = atomicAdd(&s.count, 1u);
        if (at < (uint32_t)kList) index[at] = i;
    }
    __syncthreads();
    const uint32_t n = uniform(s.count);
    for (uint32_t q = threadIdx.x; q < n && q < (uint32_t)kList; q += BLOCK) s.list[q] = by_value(key_of(to_f32(row[index[q]])), index[q]);
    __syncthreads();
    return n;
}

template <int BLOCK, typename T>
__device__ __forceinline__ uint32_t gather(Shared<BLOCK> &s, const RowState &o, const T *row, int begin, int end, const Reach &want) {
    constexpr int E = Vec<T>::E;
    const Vec<T> *v = reinterpret_cast<const Vec<T> *>(row + begin);
    const int pieces = (end - begin) / E;
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    for (int j0 = 0; j0 < pieces; j0 += BLOCK * 4) {
        const int j = j0 + threadIdx.x;
        Vec<T> p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u] = v[min(j + u * BLOCK, pieces - 1)];
        const uint32_t mask = reach_mask<BLOCK, T>(o, p, j, pieces, want), at = reserve(&s.count, __popc(mask));
        put_mask<BLOCK, T>(reinterpret_cast<uint32_t *>(s.mass), mask, at, j, begin);
    }
    return finish_list<BLOCK, T>(s, o, row, begin + pieces * E + threadIdx.x, end, want);
}

// A cut inside a bin that holds more than the list: the bin's range of keys is split again (whole row per step) until the
// entries fit, or share one value.  Uses up the histogram.
template <int BLOCK, typename T>
__device__ __forceinline__ void cut_range(Shared<BLOCK> &s, Histogram &h, const RowState &o, Filter &f, const T *row, int size, const Step &st,
                          double *mass_at) {
    uint32_t hi = 0, lo = 0xffffffffu, n = st.n;
    {
        float top = -__builtin_inff(), low = __builtin_inff();
        for_each<BLOCK>(row, 0, size, [&](float x, int, int) {
            if (key_of(x) && bin_of(o.w, o.scale, x) == st.bin) top = fmaxf(top, x), low = fminf(low, x);
        });
        block_max_min<BLOCK>(top, low, s);
        hi = key_of(top), lo = key_of(low);
    }
    Above above = st.above;
    while (n > (uint32_t)kList && lo < hi) {
        int bits = 0;
        while (((hi - lo) >> bits) >= (uint32_t)kBins) ++bits;
        const int up = raise(o, st.bin);                 // all of these entries lie in that bin
        fill_histogram<BLOCK, T>(h, o, row, size, [=](float, uint32_t key) { return key >= lo && key <= hi ? (int)((hi - key) >> bits) : -1; },
                                 [=](int) { return up; });
        const int bin = min(find_bin<BLOCK>(s, h, st.by_count, true, f.k, st.wantm, above), kBins - 1);
        n = uniform(h.cnt[bin]);
        hi -= (uint32_t)bin << bits;
        if (hi - lo > (1u << bits) - 1) lo = hi - ((1u << bits) - 1);
        __syncthreads();
    }
    if (n <= (uint32_t)kList) {
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        for_each<BLOCK>(row, 0, size, [&](float x, int i, int) {
            const uint32_t key = key_of(x);
            if (key >= lo && key <= hi) s.list[atomicAdd(&s.count, 1u)] = by_value(key, i);
        });
        __syncthreads();
        sort_by_value<BLOCK>(s, n, value_of(hi), fminf((float)kBins / (value_of(hi) - value_of(lo)), 1e30f));
        cut_list<BLOCK>(s, o, f, n, above, st.by_count ? (int)(f.k - above.cnt) : kList + 1, !st.by_count, -1.0, st.wantm, mass_at);
        return;
    }
    // one value, more than kList times: the first q of them by index
    const double e = mass_of(o.w, value_of(hi));
    uint32_t q = n;
    if (st.by_count) q = f.k - above.cnt;
    else if (e > 0.0) {
        // as many as have less than the target before them; the quotient's rounding is mended
        q = (uint32_t)fmin((double)n, fmax(1.0, __builtin_ceil((st.wantm - above.mass) / e)));
        if (q > 1 && above.mass + (q - 1) * e >= st.wantm) --q;
        else if (q < n && above.mass + q * e < st.wantm) ++q;
    }
    *mass_at = above.mass + q * e;
    f.key = hi;
    uint32_t seen = 0;                                   // entries of that value in the chunks before
    for (int i0 = 0; i0 < size && seen < q; i0 += BLOCK) {
        const int i = i0 + threadIdx.x;
        const uint32_t is = i < size && key_of(to_f32(row[i])) == hi;
        uint32_t all;
        const uint32_t before = seen + block_scan<BLOCK, uint32_t>(is, s.wave_a, &all);
        if (is && before + 1 == q) s.found[0] = i;
        seen += all;
    }
    __syncthreads();
    f.idx = (int)uniform(s.found[0]);
    __syncthreads();
}

// Mass of the entries that top-k's cut keeps
template <int BLOCK, typename T>
__device__ __forceinline__ double mass_of_first(Shared<BLOCK> &s, const RowState &o, const T *row, int size) {
    double mine = 0.0, all;
    for_each<BLOCK, 1>(row, 0, size, [&](float x, int i, int) {
        const uint32_t key = key_of(x);
        if (key && o.f.keeps(key, i)) mine += mass_of(o.w, x);
    });
    block_scan<BLOCK, double>(mine, s.wave_d, &all);
    return __builtin_bit_cast(double, uniform(__builtin_bit_cast(uint64_t, all)));
}

// Both cuts of a long row, from its histogram (used up where a bin is too full).  gathered: the entries of the first step are in
// the list already.  Returns the number of kept entries where the list holds all of them, sorted by value; else -1.
template <int BLOCK, typename T>
__device__ __forceinline__ int select_cut(Shared<BLOCK> &s, Histogram &h, RowState &o, const T *row, int size, Step st, bool gathered) {
    while (st.any) {
        double mass_at = 0.0;
        if (st.fits) {
            const int n = gathered ? uniform(s.count) : gather<BLOCK, T>(s, o, row, 0, size, Reach(st.from, st.bin));
            gathered = false;
            // the bins from .. bin, stretched over the buckets
            sort_by_value<BLOCK>(s, n, o.w.topf - (float)st.from / o.scale, o.scale * ((float)kBins / (float)(st.bin - st.from + 1)));
            int kept;
            if (st.by_count) {
                // with the whole prefix in the list, top-p is decided by it too
                const bool both = st.prefix && o.use_p;
                kept = cut_list<BLOCK>(s, o, o.f, n, st.above, (int)(o.f.k - st.above.cnt), both, both ? o.f.p : -1.0, 0.0, &mass_at);
            } else {
                kept = cut_list<BLOCK>(s, o, o.f, n, st.above, kList + 1, true, -1.0, st.wantm, &mass_at);
            }
            if (st.prefix) return kept;
        } else {
            cut_range<BLOCK, T>(s, h, o, o.f, row, size, st, &mass_at);
        }
        if (!(st.by_count && o.use_p)) break;
        // top-k's list was not the whole prefix: top-p by masses, which a histogram for top-k's sake has not got
        fill_histogram<BLOCK, T>(h, o, row, size);
        mass_at = mass_of_first<BLOCK, T>(s, o, row, size);
        st = make_step<BLOCK>(s, h, o, false, mass_at);
    }
    if (!st.any) o.f.cut = false;
    return -1;
}

// ---- draws
__device__ __forceinline__ double mass_or_zero(const RowState &o, uint32_t key) {
    const double e = mass_of(o.w, value_of(key));
    return e >= o.f.m ? e : 0.0;
}

// What a running mass has to exceed.  u = 1, and what is clamped to it, lies behind all of them, whatever their roundings, and so names
// the last entry with mass; below, u <= 1 - 2^-24 keeps far from the total.
__device__ __forceinline__ double target(float u, double total) {
    return u >= 1.0f ? __builtin_inf() : (double)fmaxf(u, 0.0f) * total;
}

// From the list, kept entries 0 .. n by index as (index, key), and their running masses: draws first, first + step ...
template <int BLOCK>
__device__ __forceinline__ void draw_by_search(Shared<BLOCK> &s, const RowState &o, int n, double total, const float *u, int draws, int64_t *ids,
                                               float *prob, int first, int step) {
    for (int j = first; j < draws; j += step) {
        const float uj = u[j];
        const double want = target(uj, total);
        int a = 0, b = n - 1;                          // first entry whose running mass exceeds `want`
        while (a < b) {
            const int mid = (a + b) >> 1;
            if (s.mass[mid] > want) b = mid;
            else a = mid + 1;
        }
        // back from the end of the list (u = 1), or from a running sum that an entry without mass rounds up
        while (a > 0 && mass_or_zero(o, (uint32_t)s.list[a]) == 0.0) --a;
        const double m = mass_or_zero(o, (uint32_t)s.list[a]);
        ids[j] = uj == uj ? (int64_t)(s.list[a] >> 32) : -1;
        prob[j] = uj == uj ? (float)(m / total) : 0.0f;
    }
}

// The kept entries' running masses, then a thread a draw.
template <int BLOCK>
__device__ __forceinline__ void draw_from_list(Shared<BLOCK> &s, const RowState &o, int n, const float *u, int draws, int64_t *ids, float *prob) {
    constexpr int kPer = kList / BLOCK;
    double e[kPer], run = 0.0, total;
    const int tid = threadIdx.x, i0 = tid * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        e[j] = i0 + j < n ? mass_or_zero(o, (uint32_t)s.list[i0 + j]) : 0.0;
        run += e[j];
    }
    double cum = block_scan<BLOCK, double>(run, s.wave_d, &total);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        cum += e[j];
        s.mass[i0 + j] = cum;
    }
    __syncthreads();
    total = s.mass[n - 1];
    draw_by_search(s, o, n, total, u, draws, ids, prob, tid, BLOCK);
}

// Tiles of a row: 1024 entries, or a multiple of them where a row has more than kMaxTiles; 16 consecutive entries a lane.
__device__ __forceinline__ int tile_of(int size) {
    int tile = 1024;
    while ((size + tile - 1) / tile > kMaxTiles) tile <<= 1;
    return tile;
}

// This lane's 16 kept masses of the 1024 entries from `base`; their sum
template <typename T>
__device__ __forceinline__ double lane_masses(const RowState &o, const T *row, int size, int base, double *e) {
    constexpr int E = Vec<T>::E;
    const int i0 = base + (threadIdx.x & 63) * 16;
    T x[16];
    if (i0 + 16 <= size) {
#pragma unroll
        for (int v = 0; v < 16 / E; ++v) {
            const Vec<T> p = *reinterpret_cast<const Vec<T> *>(row + i0 + v * E);
#pragma unroll
            for (int j = 0; j < E; ++j) x[v * E + j] = p.e[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = i0 + j < size ? row[i0 + j] : from_f32<T>(-__builtin_inff());
    }
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        e[j] = kept_mass(o.w, o.f, to_f32(x[j]), i0 + j);
        sum += e[j];
        if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // 16 exponentials interleaved need more registers than there are
    }
    return sum;
}

template <typename T>
__device__ __forceinline__ double tile_mass(const RowState &o, const T *row, int size, int tile, int q) {
    double e[16], sum = 0.0;
    const int end = min(size, (q + 1) * tile);
    for (int base = q * tile; base < end; base += 1024) sum += lane_masses<T>(o, row, size, base, e);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    return sum;
}

// Of the lanes' entries (base + 16 lane + j, masses e, inclusive lane sums `cum` on top of `before`) the first whose running sum
// exceeds `want`; where rounding leaves none, the last one with mass.  Returns whether one exceeds.
template <int P>
__device__ __forceinline__ bool pick_entry(const double *e, double sum, double cum, double before, double want, int base, int &at,
                                           double &mass) {
    const uint64_t over = __ballot(sum > 0.0 && before + cum > want), some = __ballot(sum > 0.0);
    if (some == 0) return false;
    const int src = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
    double run = before + lane_before(cum), m = 0.0;
    int in = 0;
    bool found = false;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        run += e[j];
        if (e[j] > 0.0 && !found) in = j, m = e[j], found = over != 0 && run > want;
    }
    at = base + src * P + __shfl(in, src);
    mass = __shfl(m, src);
    return over != 0;
}

// tiles[0 .. n) -> running sums; load(q): tile q.  Returns the last tile with mass.
template <int BLOCK, typename S, typename L>
__device__ __forceinline__ int scan_tiles(S &s, double *tiles, int n, L load) {
    constexpr int kPer = kMaxTiles / BLOCK;
    const int q0 = threadIdx.x * kPer;
    double v[kPer], run = 0.0, total;
    int last = -1;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        v[j] = q0 + j < n ? load(q0 + j) : 0.0, run += v[j];
        last = v[j] > 0.0 ? q0 + j : last;
    }
    const uint64_t some = __ballot(last >= 0);
    last = some ? __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(some)) : 0;
    if ((threadIdx.x & 63) == 0) s.wave_last[threadIdx.x >> 6] = last;
    double cum = block_scan<BLOCK, double>(run, s.wave_d, &total);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        cum += v[j];
        if (q0 + j < n) tiles[q0 + j] = cum;
    }
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) last = max(last, s.wave_last[w]);
    __syncthreads();
    return last;
}

// One draw by a wave: the tile by its running sum, then the entry.
template <typename T>
__device__ __forceinline__ void draw_from_tiles(const RowState &o, const T *row, int size, int tile, const double *tiles, int n_tiles, int last,
                                float uj, int64_t *id, float *prob) {
    const int lane = threadIdx.x & 63;
    const double total = tiles[n_tiles - 1];
    double want = target(uj, total);
    // the first tile whose running sum exceeds `want` (u = 1: the last with mass): 64 probes, 16 tiles apart, then 16
    static_assert(kMaxTiles == 64 * 16, "two steps");
    const uint64_t far = __ballot(tiles[min(lane * 16 + 15, n_tiles - 1)] > want);
    const int from = (far ? __builtin_ctzll(far) : 63) * 16;
    const uint64_t near = __ballot(tiles[min(from + (lane & 15), n_tiles - 1)] > want);
    int a = near ? min(from + __builtin_ctzll(near), n_tiles - 1) : last, at = 0;
    double mass = 0.0, e[16];
    // The sums are added in another order from thread to thread, so an empty tile's may lie a rounding above that of the tile before:
    // where that much led to it, the draw is the last entry with mass before it.  (There is one: the sums of empty tiles are exactly 0 up to
    // the first tile with mass.)
    for (;; --a, want = __builtin_inf()) {
        double before = a > 0 ? tiles[a - 1] : 0.0;
        const int end = min(size, (a + 1) * tile);
        for (int base = a * tile; base < end; base += 1024) {
            const double sum = lane_masses<T>(o, row, size, base, e), cum = wave_scan(sum);
            if (pick_entry<16>(e, sum, cum, before, want, base, at, mass)) break;
            before += __shfl(cum, 63);
        }
        if (mass > 0.0 || a == 0) break;
    }
    if (lane == 0) {
        *id = uj == uj ? at : -1;
        *prob = uj == uj ? (float)(mass / total) : 0.0f;
    }
}

// Rows without anything to draw (id -1), and T = 0 (the first maximum).
__device__ __forceinline__ void draw_plain(const RowState &o, int at, const float *u, int draws, int64_t *ids, float *prob, int first,
                                           int step) {
    for (int j = first; j < draws; j += step) {
        const bool ok = o.valid && u[j] == u[j];
        ids[j] = ok ? at : -1;
        prob[j] = ok ? 1.0f : 0.0f;
    }
}

// LDS written by lanes of this wave before, read by others behind (a wave's LDS accesses are in order; this holds the compiler to it)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// n <= 64 P entries of the list into rising order, by one wave: each counts the smaller ones; c: entries P * lane + j
template <int P>
__device__ __forceinline__ void wave_sort(uint64_t *list, int n, uint64_t *c) {
    const int i0 = (threadIdx.x & 63) * P;
    uint32_t rank[P] = {};
#pragma unroll 16
    for (int q = 0; q < n; ++q) {
        const uint64_t v = list[q];
#pragma unroll
        for (int j = 0; j < P; ++j) rank[j] += v < c[j];
    }
    wave_sync();
#pragma unroll
    for (int j = 0; j < P; ++j)
        if (i0 + j < n) list[rank[j]] = c[j];
    wave_sync();
#pragma unroll
    for (int j = 0; j < P; ++j) c[j] = list[min(i0 + j, n - 1)];
}

// draw_top_k by one wave, for a list of at most 64 P entries and few draws: no barriers.  One row of 131072, top-k 50: 15.6 us a
// call against 18.2 by the block's steps, 256 rows of 32768 11.8 against 13.5; lists of 200 with four entries a lane 23.6 against 21.6.
template <int P, int BLOCK>
__device__ __forceinline__ void draw_few(Shared<BLOCK> &s, const RowState &o, int n, const float *u, int draws, int64_t *ids, float *prob) {
    const int lane = threadIdx.x & 63, i0 = lane * P, last = min(o.f.k, n);
    uint64_t c[P];
    double e[P], run = 0.0, at_last = 0.0;
#pragma unroll
    for (int j = 0; j < P; ++j) c[j] = s.list[min(i0 + j, n - 1)];
    wave_sort<P>(s.list, n, c);
#pragma unroll
    for (int j = 0; j < P; ++j) {
        e[j] = i0 + j < n ? mass_of(o.w, value_of(~(uint32_t)(c[j] >> 32))) : 0.0;
        run += e[j];
        if (i0 + j == last - 1) at_last = run;
    }
    double before = lane_before(wave_scan(run));
    const double want = o.f.p * __shfl(before + at_last, (last - 1) / P);
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        if (i0 + j < last && (!o.use_p || before < want || i0 + j == 0)) ++mine;
        before += e[j];
    }
    const int kept = (int)__builtin_amdgcn_readlane(wave_scan(mine), 63);
    wave_sync();
#pragma unroll
    for (int j = 0; j < P; ++j) {
        c[j] = (c[j] << 32) | (uint32_t)~(uint32_t)(c[j] >> 32);
        if (i0 + j < kept) s.list[i0 + j] = c[j];
    }
    wave_sync();
    wave_sort<P>(s.list, kept, c);
    double m[P], sum = 0.0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        m[j] = i0 + j < kept ? mass_or_zero(o, (uint32_t)c[j]) : 0.0;
        sum += m[j];
    }
    double cum = lane_before(wave_scan(sum));          // (not a difference: a small mass before a large one would be lost)
#pragma unroll
    for (int j = 0; j < P; ++j) {
        cum += m[j];
        if (i0 + j < kept) s.mass[i0 + j] = cum;
    }
    wave_sync();
    draw_by_search(s, o, kept, s.mass[kept - 1], u, draws, ids, prob, lane, 64);
}

// The list holds all that top-k can keep (values down to `low`): both cuts and the draws from it.
template <int BLOCK>
__device__ __forceinline__ void draw_top_k(Shared<BLOCK> &s, RowState &o, int n, float low, int size, const float *u, int draws, int64_t *ids, float *prob) {
    if (n <= 128 && draws <= 64) {
        if (threadIdx.x < 64) draw_few<2>(s, o, n, u, draws, ids, prob);
        return;
    }
    double mass_at;
    sort_by_value<BLOCK>(s, n, o.w.topf, fminf((float)kBins / (o.w.topf - low), 1e30f));
    const int kept = cut_list<BLOCK>(s, o, o.f, n, Above{0, 0.0}, min(o.f.k, n), o.use_p, o.f.p, 0.0, &mass_at);
    list_by_index<BLOCK>(s, kept, size);
    draw_from_list<BLOCK>(s, o, kept, u, draws, ids, prob);
}

template <int BLOCK, typename T>
__device__ __forceinline__ void draw_whole_row(Shared<BLOCK> &s, double *tiles, const RowState &o, const T *row, int size, const float *u, int draws,
                               int64_t *ids, float *prob) {
    const int tid = threadIdx.x, tile = tile_of(size), n_tiles = (size + tile - 1) / tile;
    for (int q = tid >> 6; q < n_tiles; q += BLOCK / 64) {
        const double m = tile_mass<T>(o, row, size, tile, q);
        if ((tid & 63) == 0) tiles[q] = m;
    }
    __syncthreads();
    const int last = scan_tiles<BLOCK>(s, tiles, n_tiles, [&](int q) { return tiles[q]; });
    for (int j = tid >> 6; j < draws; j += BLOCK / 64) draw_from_tiles<T>(o, row, size, tile, tiles, n_tiles, last, u[j], ids + j, prob + j);
}

// ---- one block a row
template <typename T>
struct RowIO {
    const T *row;
    const float *u;
    int64_t *ids;
    float *prob;
    __device__ __forceinline__ RowIO(const SampleArgs &a, int r)
        : row((const T *)a.logits + (int64_t)r * a.stride), u(a.u + (int64_t)r * a.draws), ids(a.ids + (int64_t)r * a.draws),
          prob(a.prob + (int64_t)r * a.draws) {}
};

// A long row by its histogram, from the start.
template <int BLOCK, typename T>
__device__ __forceinline__ void draw_long_row(Shared<BLOCK> &s, Histogram &h, double *tiles, RowState &o, const RowIO<T> &io, const SampleArgs &a) {
    if (o.f.cut) {
        const bool by_k = o.f.k < a.size;
        if (by_k) {
            clear_histogram<BLOCK>(h);
            add_counts<BLOCK, T>(h, o, io.row, 0, a.size);
        } else {
            fill_histogram<BLOCK, T>(h, o, io.row, a.size);
        }
        Step st = first_step<BLOCK>(s, h, o);
        if (by_k && !st.any && o.use_p) {          // fewer than k can be drawn: top-p of them all
            fill_histogram<BLOCK, T>(h, o, io.row, a.size);
            st = first_step<BLOCK>(s, h, o);
        }
        const int listed = select_cut<BLOCK, T>(s, h, o, io.row, a.size, st, false);
        if (listed > 0) {
            list_by_index<BLOCK>(s, listed, a.size);
            return draw_from_list<BLOCK>(s, o, listed, io.u, a.draws, io.ids, io.prob);
        }
    }
    draw_whole_row<BLOCK, T>(s, tiles, o, io.row, a.size, io.u, a.draws, io.ids, io.prob);
}

// Rows of up to kList entries: the whole row goes into the list.
template <typename T>
__global__ void __launch_bounds__(256) sample_short_kernel(const SampleArgs a) {
    constexpr int BLOCK = 256;
    __shared__ Shared<BLOCK> s;
    const int tid = threadIdx.x, size = a.size;
    const RowIO<T> io(a, blockIdx.x);
    float top = -__builtin_inff(), low = __builtin_inff();
    for_each<BLOCK>(io.row, 0, size, [&](float x, int, int) { top = fmaxf(top, x), low = fminf(low, x); });
    if (tid < 16) s.tab[tid] = kRoots[tid];
    block_max_min<BLOCK>(top, low, s);
    RowState o = row_state(a, blockIdx.x, top, low, s.tab);
    if (o.plain()) {
        const int at = find_value<BLOCK, T>(s, io.row, 0, size, o.w.topf, size);
        return draw_plain(o, at, io.u, a.draws, io.ids, io.prob, tid, BLOCK);
    }
    if (!o.f.cut) {
        for_each<BLOCK>(io.row, 0, size, [&](float x, int i, int) { s.list[i] = ((uint64_t)i << 32) | key_of(x); });
        __syncthreads();
        return draw_from_list<BLOCK>(s, o, size, io.u, a.draws, io.ids, io.prob);
    }
    if (tid == 0) s.count = 0;
    __syncthreads();
    for_each<BLOCK>(io.row, 0, size, [&](float x, int i, int) {
        const uint32_t key = key_of(x);
        if (key) s.list[atomicAdd(&s.count, 1u)] = by_value(key, i);
    });
    __syncthreads();
    draw_top_k<BLOCK>(s, o, uniform(s.count), fmaxf(low, -3e38f), size, io.u, a.draws, io.ids, io.prob);
}

// HELD: 16-byte pieces a thread keeps in registers from the pass for the maximum to that for the list, 0 where the row is read again
template <typename T, int HELD>
__global__ void __launch_bounds__(1024) sample_row_kernel(const SampleArgs a) {
    constexpr int BLOCK = 1024, E = Vec<T>::E;
    __shared__ Shared<BLOCK> s;
    __shared__ Histogram h;
    __shared__ double tiles[kMaxTiles];
    const int tid = threadIdx.x, size = a.size, pieces = size / E;
    const RowIO<T> io(a, blockIdx.x);
    float group[4] = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()}, low = __builtin_inff();
    typedef uint32_t Raw __attribute__((ext_vector_type(4)));
    Raw held[HELD > 0 ? HELD : 1];
    if constexpr (HELD > 0) {
        const Vec<T> *v = reinterpret_cast<const Vec<T> *>(io.row);
#pragma unroll
        for (int u = 0; u < HELD; ++u)
            if (u * BLOCK < pieces) held[u] = __builtin_bit_cast(Raw, v[min(u * BLOCK + tid, pieces - 1)]);
#pragma unroll
        for (int u = 0; u < HELD; ++u)
            if (u * BLOCK + tid < pieces) {
                const Vec<T> p = __builtin_bit_cast(Vec<T>, held[u]);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = to_f32(p.e[e]);
                    group[u & 3] = fmaxf(group[u & 3], x), low = fminf(low, x);
                }
            }
        if (pieces * E + tid < size) {
            const float x = to_f32(io.row[pieces * E + tid]);
            group[0] = fmaxf(group[0], x), low = fminf(low, x);
        }
    } else {
        for_each<BLOCK>(io.row, 0, size, [&](float x, int, int u) { group[u] = fmaxf(group[u], x), low = fminf(low, x); });
    }
    if (tid < 16) s.tab[tid] = kRoots[tid];
    float top = fmaxf(fmaxf(group[0], group[1]), fmaxf(group[2], group[3]));
    block_max_min<BLOCK>(top, low, s);
    RowState o = row_state(a, blockIdx.x, top, low, s.tab);
    if (o.plain()) {
        const int at = find_value<BLOCK, T>(s, io.row, 0, size, o.w.topf, size);
        return draw_plain(o, at, io.u, a.draws, io.ids, io.prob, tid, BLOCK);
    }
    if (o.f.cut && o.f.k <= kGroupsMaxK) {
        if (tid == 0) s.count = 0;
        clear_histogram<BLOCK>(h);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (group[u] > -__builtin_inff()) atomicAdd(&h.cnt[bin_of(o.w, o.scale, group[u])], 1u);
        __syncthreads();
        Above above{0, 0.0};
        // where fewer than k groups hold anything: all entries, if they fit
        const int bin = min(find_bin<BLOCK>(s, h, true, false, o.f.k, 0.0, above), kBins - 1);
        const Reach want(o, bin);
        uint32_t n;
        if constexpr (HELD > 0) {
            uint32_t mask[HELD / 4], hits = 0;
#pragma unroll
            for (int u = 0; u < HELD; u += 4) {
                mask[u / 4] = 0;
                if (u * BLOCK < pieces) {
                    Vec<T> p[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        // opaque: else the widened values of the first pass would be kept, in twice the registers
                        asm volatile("" : "+v"(held[u + k]));
                        p[k] = __builtin_bit_cast(Vec<T>, held[u + k]);
                    }
                    mask[u / 4] = reach_mask<BLOCK, T>(o, p, u * BLOCK + tid, pieces, want);
                    hits += __popc(mask[u / 4]);
                }
            }
            uint32_t at = reserve(&s.count, hits);
#pragma unroll
            for (int u = 0; u < HELD; u += 4)
                at = put_mask<BLOCK, T>(reinterpret_cast<uint32_t *>(s.mass), mask[u / 4], at, u * BLOCK + tid, 0);
            n = finish_list<BLOCK, T>(s, o, io.row, pieces * E + tid, size, want);
        } else {
            n = gather<BLOCK, T>(s, o, io.row, 0, size, want);
        }
        if (n <= (uint32_t)kList) return draw_top_k<BLOCK>(s, o, n, o.w.topf - (float)(bin + 1) / o.scale, size, io.u, a.draws, io.ids, io.prob);
    }
    draw_long_row<BLOCK, T>(s, h, tiles, o, io, a);
}

// Whether a chunk behind c has mass
template <int C>
__device__ __forceinline__ bool more_after(const double *all, int c) {
    bool more = false;
#pragma unroll
    for (int k = 0; k < C; ++k) more = more || (k > c && all[k] > 0.0);
    return more;
}

// ---- short rows without a cut: a wave a row of up to 64 P entries, in chunks of 16 bytes a lane (entry: chunk, lane, place)
template <typename T, int P>
__global__ void __launch_bounds__(256) sample_wave_kernel(const SampleArgs a) {
    constexpr int E = Vec<T>::E, C = P / E;
    __shared__ double tab[16];
    const int lane = threadIdx.x & 63, r = min((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), a.rows - 1), size = a.size;
    const RowIO<T> io(a, r);
    float x[C][E], top = -__builtin_inff(), u = io.u[0];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * 64 + lane) * E;
        if (i + E <= size) {
            const Vec<T> p = *reinterpret_cast<const Vec<T> *>(io.row + i);
#pragma unroll
            for (int j = 0; j < E; ++j) x[c][j] = to_f32(p.e[j]);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) x[c][j] = i + j < size ? to_f32(io.row[i + j]) : -__builtin_inff();
        }
    }
    if (threadIdx.x < 16) tab[threadIdx.x] = kRoots[threadIdx.x];
    __syncthreads();
    if ((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6) >= a.rows) return;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j) top = fmaxf(top, x[c][j]);
    const RowState o = row_state(a, r, wave_max(top), 0.0f, tab);
    if (o.plain()) {
        int at = size;
#pragma unroll
        for (int c = C - 1; c >= 0; --c) {
            const int i = (c * 64 + lane) * E;
            int mine = E;
#pragma unroll
            for (int j = E - 1; j >= 0; --j) mine = x[c][j] == o.w.topf ? j : mine;
            const uint64_t has = __ballot(mine < E);
            if (has) at = __builtin_amdgcn_readlane(i + mine, __builtin_ctzll(has));
        }
        return draw_plain(o, at, io.u, a.draws, io.ids, io.prob, lane, 64);
    }
    double e[C][E], sum[C], cum[C], all[C], total = 0.0;      // per chunk: this lane's mass, with the lanes before, the wave's
#pragma unroll
    for (int c = 0; c < C; ++c) {
        sum[c] = 0.0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            e[c][j] = kept_mass(o.w, o.f, x[c][j], (c * 64 + lane) * E + j);
            sum[c] += e[c][j];
        }
        cum[c] = wave_scan(sum[c]);
        all[c] = last_lane(cum[c]);
        total += all[c];
    }
    for (int d = 0; d < a.draws; ++d) {
        if (d > 0) u = io.u[d];
        const double want = target(u, total);
        int at = 0;
        double mass = 0.0, before = 0.0;
        bool found = false;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            // the chunk that exceeds; until one does, the last place with mass (all of this is wave-uniform)
            if (!found && all[c] > 0.0 && (before + all[c] > want || c == C - 1 || !more_after<C>(all, c)))
                found = pick_entry<E>(e[c], sum[c], cum[c], before, want, c * 64 * E, at, mass);
            before += all[c];
        }
        if (lane == 0) {
            io.ids[d] = u == u ? at : -1;
            io.prob[d] = u == u ? (float)(mass / total) : 0.0f;
        }
    }
}

// ---- few long rows: kParts blocks a row and stage.  What a stage leaves for the next, per row:
struct RowWork {
    float top[kParts], low[kParts];        // of each part
    int32_t first[kParts];                 // lowest index of the part's maximum (T = 0)
    uint32_t count[2];                     // entries in `list`: from the groups' bound / from the histogram
    uint32_t arrived[3];
    uint32_t done;                         // the draws are out
    uint32_t cut, cut_key;
    int32_t cut_idx, last_tile;
    alignas(256) float group[kGroups];
    Histogram h;
    uint64_t high[kBins];                  // upper halves of the words, apart where more than kSegment entries could pass 64 bits
    uint64_t list[kList];
    double tiles[kMaxTiles];
};

struct Part {
    int begin, end;
};
__device__ __forceinline__ Part part_of(int size, int part, int parts) {
    const int each = ((size + parts - 1) / parts + 15) / 16 * 16;
    return Part{(int)min((int64_t)size, (int64_t)part * each), (int)min((int64_t)size, (int64_t)(part + 1) * each)};
}

__device__ __forceinline__ RowState state_of(const SampleArgs &a, int r, const RowWork &w, const double *tab) {
    const int part = threadIdx.x & (kParts - 1);               // a lane a part
    return row_state(a, r, wave_max(w.top[part]), -wave_max(-w.low[part]), tab);
}

// What blocks of one launch hand to the last of them goes through the memory that all XCDs see, word by word (their L2s do not see
// each other's writes).  A fence at device scope instead writes back a whole L2 for each block: 33 us for 1024 blocks.
template <typename V>
__device__ __forceinline__ void publish(V *p, V v) {
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V>
__device__ __forceinline__ V fetch(const V *p) {
    return __builtin_bit_cast(V, __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Whether this block is the last of its row at this point: what the others published before is there then.  Every wave waits for
// its stores to arrive before the barrier, and the count is raised behind it.
template <typename S>
__device__ __forceinline__ bool last_to_arrive(S &s, uint32_t *counter) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) s.found[0] = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == gridDim.x;
    __syncthreads();
    const bool last = uniform((uint32_t)s.found[0]);
    __syncthreads();
    return last;
}

// This part's entries behind those of the other parts in the row's list (entries beyond kList: counted only).
template <int BLOCK, typename T>
__device__ __forceinline__ void gather_part(Shared<BLOCK> &s, const RowState &o, const T *row, Part p, const Reach &want, uint64_t *list,
                                            uint32_t *count) {
    const uint32_t n = gather<BLOCK, T>(s, o, row, p.begin, p.end, want);
    if (threadIdx.x == 0) s.found[0] = n ? atomicAdd(count, n) : 0;
    __syncthreads();
    const uint32_t at = uniform((uint32_t)s.found[0]);
    for (uint32_t i = threadIdx.x; i < n && i < (uint32_t)kList && at + i < (uint32_t)kList; i += BLOCK) publish(&list[at + i], s.list[i]);
}

// The row's whole list into LDS; its length
template <int BLOCK>
__device__ __forceinline__ uint32_t load_list(Shared<BLOCK> &s, const uint64_t *list, const uint32_t *count) {
    uint64_t c[kList / BLOCK];                             // in flight together with the length
#pragma unroll
    for (int j = 0; j < kList / BLOCK; ++j) c[j] = fetch(&list[j * BLOCK + threadIdx.x]);
    const uint32_t n = uniform(__hip_atomic_load(count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
#pragma unroll
    for (int j = 0; j < kList / BLOCK; ++j) s.list[j * BLOCK + threadIdx.x] = c[j];
    if (threadIdx.x == 0) s.count = n;
    __syncthreads();
    return n;
}

// Stage 1: maximum, minimum, groups' maxima; clears what later stages add to.
template <typename T>
__global__ void __launch_bounds__(1024) sample_max_kernel(const SampleArgs a, RowWork *work) {
    constexpr int BLOCK = 1024;
    __shared__ Shared<BLOCK> s;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    RowWork &w = work[r];
    const RowIO<T> io(a, r);
    const Part p = part_of(a.size, part, kParts);
    float top = -__builtin_inff(), low = __builtin_inff();
    for_each<BLOCK>(io.row, p.begin, p.end, [&](float x, int, int) { top = fmaxf(top, x), low = fminf(low, x); });
    constexpr int kEach = kGroups / kParts, kOf = BLOCK / kEach;       // groups of a part, threads of a group
    float g = top;
#pragma unroll
    for (int d = 1; d < kOf; d <<= 1) g = fmaxf(g, __shfl_xor(g, d));
    if (tid % kOf == 0) w.group[part * kEach + tid / kOf] = g;
    for (int i = tid; i < kBins / kParts; i += BLOCK) {
        const int b = part * (kBins / kParts) + i;
        w.h.cnt[b] = 0, w.h.word[b] = 0, w.high[b] = 0;
    }
    block_max_min<BLOCK>(top, low, s);
    const float t = a.temperature_v ? a.temperature_v[r] : a.temperature;
    const int first = t == 0.0f ? find_value<BLOCK, T>(s, io.row, p.begin, p.end, top, a.size) : 0;
    if (tid == 0) {
        w.top[part] = top, w.low[part] = low, w.first[part] = first;
        if (part == 0) {
            w.count[0] = w.count[1] = w.done = w.cut = 0;
            w.arrived[0] = w.arrived[1] = w.arrived[2] = 0;
        }
    }
}

// Stage 2, rows whose top-k the groups' maxima bound: the list, and by the last block the draws.  Where the list overflows, the
// next stages see to the row, or (alone) the last block by itself.
template <typename T>
__global__ void __launch_bounds__(1024) sample_groups_kernel(const SampleArgs a, RowWork *work, bool alone) {
    constexpr int BLOCK = 1024;
    __shared__ Shared<BLOCK> s;
    __shared__ Histogram h;
    __shared__ double tiles[kMaxTiles];
    const int tid = threadIdx.x, r = blockIdx.y;
    RowWork &w = work[r];
    const RowIO<T> io(a, r);
    if (tid < 16) s.tab[tid] = kRoots[tid];
    float group[kGroups / BLOCK];
#pragma unroll
    for (int u = 0; u < kGroups / BLOCK; ++u) group[u] = w.group[u * BLOCK + tid];
    RowState o = state_of(a, r, w, s.tab);
    if (o.plain()) {                                           // the list holds nothing: one block writes the row
        if (blockIdx.x > 0) return;
        int at = a.size;
        for (int i = 0; i < kParts; ++i)
            if (w.top[i] == o.w.topf) at = min(at, w.first[i]);
        draw_plain(o, at, io.u, a.draws, io.ids, io.prob, tid, BLOCK);
        if (tid == 0) w.done = 1;
        return;
    }
    if (o.f.k > kGroupsMaxK && !alone) return;
    clear_histogram<BLOCK>(h);
#pragma unroll
    for (int u = 0; u < kGroups / BLOCK; ++u) {
        if (group[u] > -__builtin_inff()) atomicAdd(&h.cnt[bin_of(o.w, o.scale, group[u])], 1u);
    }
    __syncthreads();
    Above above{0, 0.0};
    const int bin = min(find_bin<BLOCK>(s, h, true, false, o.f.k, 0.0, above), kBins - 1);
    const Part p = part_of(a.size, blockIdx.x, gridDim.x);
    gather_part<BLOCK, T>(s, o, io.row, p, Reach(o, bin), w.list, &w.count[0]);
    if (!last_to_arrive(s, &w.arrived[0])) return;
    const uint32_t n = load_list<BLOCK>(s, w.list, &w.count[0]);
    if (n <= (uint32_t)kList) {
        draw_top_k<BLOCK>(s, o, n, o.w.topf - (float)(bin + 1) / o.scale, a.size, io.u, a.draws, io.ids, io.prob);
        if (tid == 0) w.done = 1;
    } else if (alone) {
        draw_long_row<BLOCK, T>(s, h, tiles, o, io, a);
    }
}

// Stage 3: the histogram.
template <typename T>
__global__ void __launch_bounds__(1024) sample_bins_kernel(const SampleArgs a, RowWork *work) {
    constexpr int BLOCK = 1024;
    __shared__ Histogram h;
    __shared__ double tab[16];
    const int tid = threadIdx.x, r = blockIdx.y;
    RowWork &w = work[r];
    if (w.done) return;
    if (tid < 16) tab[tid] = kRoots[tid];
    const RowState o = state_of(a, r, w, tab);
    if (o.plain() || !o.f.cut) return;
    const RowIO<T> io(a, r);
    const Part p = part_of(a.size, blockIdx.x, gridDim.x);
    for (int begin = p.begin; begin < p.end; begin += kSegment) {
        const int end = min(p.end, begin + kSegment);
        clear_histogram<BLOCK>(h);
        if (o.use_p)
            add_words<BLOCK, T>(h, o, io.row, begin, end, [&](float x, uint32_t key) { return key ? bin_of(o.w, o.scale, x) : -1; },
                                [&](int b) { return raise(o, b); });
        else add_counts<BLOCK, T>(h, o, io.row, begin, end);
        for (int b = tid; b < kBins; b += BLOCK) {
            const unsigned long long v = h.word[b];
            if (h.cnt[b]) atomicAdd(&w.h.cnt[b], h.cnt[b]);
            if (v == 0) continue;
            const bool apart = a.size > kSegment;
            atomicAdd((unsigned long long *)&w.h.word[b], apart ? v & 0xffffffffu : v);
            if (apart) atomicAdd((unsigned long long *)&w.high[b], v >> 32);
        }
        __syncthreads();
    }
}

// Stage 4: the entries around the first cut into the list; the last block finds the cut.
template <typename T>
__global__ void __launch_bounds__(1024) sample_cut_kernel(const SampleArgs a, RowWork *work) {
    constexpr int BLOCK = 1024;
    __shared__ Shared<BLOCK> s;
    __shared__ Histogram h;
    const int tid = threadIdx.x, r = blockIdx.y;
    RowWork &w = work[r];
    if (w.done) return;
    if (tid < 16) s.tab[tid] = kRoots[tid];
    RowState o = state_of(a, r, w, s.tab);
    if (o.plain() || !o.f.cut) return;
    for (int b = tid; b < kBins; b += BLOCK) {
        h.cnt[b] = w.h.cnt[b];
        const double high = a.size > kSegment ? (double)w.high[b] * 0x1p32 : 0.0;
        h.mass[b] = __builtin_ldexp(high + (double)w.h.word[b], -raise(o, b));
    }
    __syncthreads();
    const RowIO<T> io(a, r);
    const Part p = part_of(a.size, blockIdx.x, gridDim.x);
    const Step st = first_step<BLOCK>(s, h, o);
    if (st.any && st.fits) gather_part<BLOCK, T>(s, o, io.row, p, Reach(st.from, st.bin), w.list, &w.count[1]);
    if (!last_to_arrive(s, &w.arrived[1])) return;
    if (st.any && st.fits) load_list<BLOCK>(s, w.list, &w.count[1]);       // as many as the histogram counted: they fit
    const int listed = select_cut<BLOCK, T>(s, h, o, io.row, a.size, st, st.any && st.fits);
    if (listed > 0) {
        list_by_index<BLOCK>(s, listed, a.size);
        draw_from_list<BLOCK>(s, o, listed, io.u, a.draws, io.ids, io.prob);
    }
    if (tid == 0) w.done = listed > 0, w.cut = o.f.cut, w.cut_key = o.f.key, w.cut_idx = o.f.idx;
}

// What is kept, for the stages after the cut
__device__ __forceinline__ RowState cut_state(const SampleArgs &a, int r, const RowWork &w, const double *tab) {
    RowState o = state_of(a, r, w, tab);
    o.f.cut = w.cut, o.f.key = w.cut_key, o.f.idx = w.cut_idx;
    return o;
}

// Stage 5: masses of the tiles, a wave each (64 rows of 524288: 44 us, vector units busy 66 %); by the last block their running sums.
struct TileShared {
    double tab[16], wave_d[4];
    int32_t wave_last[4];
    uint64_t found[1];
};
template <typename T>
__global__ void __launch_bounds__(256) sample_tiles_kernel(const SampleArgs a, RowWork *work) {
    constexpr int BLOCK = 256;
    __shared__ TileShared s;
    const int tid = threadIdx.x, r = blockIdx.y, tile = tile_of(a.size), n = (a.size + tile - 1) / tile;
    RowWork &w = work[r];
    if (w.done) return;
    if (tid < 16) s.tab[tid] = kRoots[tid];
    __syncthreads();
    const RowState o = cut_state(a, r, w, s.tab);
    if (o.plain()) return;
    const RowIO<T> io(a, r);
    for (int q = blockIdx.x * 4 + (tid >> 6); q < n; q += gridDim.x * 4) {
        const double m = tile_mass<T>(o, io.row, a.size, tile, q);
        if ((tid & 63) == 0) publish(&w.tiles[q], m);
    }
    if (!last_to_arrive(s, &w.arrived[2])) return;
    const int last = scan_tiles<BLOCK>(s, w.tiles, n, [&](int q) { return fetch(&w.tiles[q]); });
    if (tid == 0) w.last_tile = last;
}

// Stage 6: the draws, a wave each.
template <typename T>
__global__ void __launch_bounds__(256) sample_draw_kernel(const SampleArgs a, const RowWork *work) {
    __shared__ double tab[16], tiles[kMaxTiles];
    const int tid = threadIdx.x, r = blockIdx.y, tile = tile_of(a.size), n = (a.size + tile - 1) / tile;
    const RowWork &w = work[r];
    if (w.done) return;
    if (tid < 16) tab[tid] = kRoots[tid];
    const RowState o = cut_state(a, r, w, tab);
    const RowIO<T> io(a, r);
    if (o.plain()) {
        int at = a.size;
        for (int i = 0; i < kParts; ++i)
            if (w.top[i] == o.w.topf) at = min(at, w.first[i]);
        return draw_plain(o, at, io.u, a.draws, io.ids, io.prob, blockIdx.x * 256 + tid, gridDim.x * 256);
    }
    for (int q = tid; q < n; q += 256) tiles[q] = w.tiles[q];
    __syncthreads();
    for (int j = blockIdx.x * 4 + (tid >> 6); j < a.draws; j += gridDim.x * 4)
        draw_from_tiles<T>(o, io.row, a.size, tile, tiles, n, w.last_tile, io.u[j], io.ids + j, io.prob + j);
}

// ---- host
enum Form { kWaveForm, kShortForm, kRowForm, kPartsForm };
enum Cut { kNoCut, kListCut, kWideCut };       // kListCut: a top-k that the groups' maxima bound

// Long rows: with many of them, a block each fills the chip and is done in one launch; few of them are split.  Measured, bf16, one block
// a row against split rows, us a call (one draw; 64; 256):
//   no cut  65536 x 64 rows: 26 / 24, 47 / 27, 116 / 43    131072 x 96: 45 / 38, 65 / 44, 135 / 67    524288 x 32: 155 / 36, 176 / 38, 245 / 45
//   top-k 50  131072 x 4: 17 / 16  131072 x 16: 17 / 29  262144 x 4: 25 / 16  524288 x 16: 40 / 30  524288 x 32: 41 / 50
//   top-p 0.9  32768 x 16: 41 / 61, 66 / 62, 149 / 65    131072 x 32: 117 / 109, 141 / 110, 224 / 119    524288 x 64: 439 / 302, 463 / 306, 546 / 323
// Without a list that holds all that is kept, one block draws 16 at a time.
Form form_of(int64_t rows, int size, int draws, Cut cut) {
    if (size <= kList) return cut == kNoCut && draws <= 16 ? kWaveForm : kShortForm;
    bool parts;
    if (cut == kNoCut) parts = draws > 16 ? rows <= 96 : size >= 65536 && rows <= 128 - (1 << 22) / size;
    else if (cut == kListCut) parts = size >= 131072 && rows <= std::min(size / 32768, 64);
    else parts = rows <= std::min(size / 4096 + draws / 8, std::clamp(draws / 8, 64, 512));
    return parts ? kPartsForm : kRowForm;
}

// (a k of each row is unknown here: taken for a small one, but where many draws would make a large one slow)
Cut cut_of(const SampleArgs &a, bool may_k, bool may_p) {
    if (may_k && (a.top_k_v ? a.draws <= 64 : a.top_k <= kGroupsMaxK)) return kListCut;
    return may_k || may_p ? kWideCut : kNoCut;
}

template <typename T>
void launch_sample(const SampleArgs &a, bool may_k, bool may_p, RowWork *work, hipStream_t s) {
    const Form form = form_of(a.rows, a.size, a.draws, cut_of(a, may_k, may_p));
    if (form == kWaveForm) {
        if (a.size <= 1024) sample_wave_kernel<T, 16><<<(a.rows + 3) / 4, 256, 0, s>>>(a);
        else sample_wave_kernel<T, 32><<<(a.rows + 3) / 4, 256, 0, s>>>(a);
    } else if (form == kShortForm) {
        sample_short_kernel<T><<<a.rows, 256, 0, s>>>(a);
    } else if (form == kRowForm) {
        // 16 pieces of 1024 threads hold 131072 16-bit or 65536 f32 logits; they pay where top-k reads the row twice (256 rows of
        // 131072, top-k 1000: 34.0 us against 36.7)
        if (may_k && a.size <= 16 * 1024 * Vec<T>::E) sample_row_kernel<T, 16><<<a.rows, 1024, 0, s>>>(a);
        else sample_row_kernel<T, 0><<<a.rows, 1024, 0, s>>>(a);
    } else {
        const dim3 parts(kParts, a.rows);
        sample_max_kernel<T><<<parts, 1024, 0, s>>>(a, work);
        // one k for all rows, within the groups' reach: nothing is left for later stages (but many draws, where the list overflows)
        const bool alone = !a.top_k_v && may_k && a.top_k <= kGroupsMaxK && a.draws <= 64;
        if (may_k) sample_groups_kernel<T><<<parts, 1024, 0, s>>>(a, work, alone);
        if (alone) return;
        if (may_k || may_p) {
            // 4096 draws from one row of 640000 by top-p: 51.2 us with 32 blocks a row, 47.5 with 64, 48.7 with 128
            const dim3 more(std::clamp(128 / a.rows, kParts, 64), a.rows);
            sample_bins_kernel<T><<<more, 1024, 0, s>>>(a, work);
            sample_cut_kernel<T><<<more, 1024, 0, s>>>(a, work);
        }
        int tile = 1024;
        while ((a.size + tile - 1) / tile > kMaxTiles) tile <<= 1;
        const int n_tiles = (a.size + tile - 1) / tile;
        const int tile_blocks = std::min((n_tiles + 3) / 4, std::max(1, 2048 / a.rows));
        sample_tiles_kernel<T><<<dim3(tile_blocks, a.rows), 256, 0, s>>>(a, work);
        const int draw_blocks = (a.draws + 3) / 4 < 1024 ? (a.draws + 3) / 4 : 1024;
        sample_draw_kernel<T><<<dim3(draw_blocks, a.rows), 256, 0, s>>>(a, work);
    }
}

}  // namespace

extern "C" int64_t nrf_sample_logits_workspace_bytes(int64_t n_rows, int32_t size, int32_t n_draws) {
    bool parts = false;
    for (const Cut cut : {kNoCut, kListCut, kWideCut}) parts |= n_rows > 0 && form_of(n_rows, size, n_draws, cut) == kPartsForm;
    return parts ? n_rows * (int64_t)sizeof(RowWork) : 0;
}

extern "C" int nrf_sample_logits(const void *logits, int64_t row_stride, int32_t dtype, int64_t n_rows, int32_t size, int32_t n_draws,
                                 float temperature, int32_t top_k, float top_p, float min_p, const float *temperature_rows,
                                 const int32_t *top_k_rows, const float *top_p_rows, const float *min_p_rows, const float *u,
                                 int64_t *ids, float *prob, void *workspace, void *stream) {
    NRF_REQUIRE(n_rows >= 0 && size >= 1 && n_draws >= 0, "nrf_sample_logits: n_rows %lld, size %d, n_draws %d", (long long)n_rows, size, n_draws);
    NRF_REQUIRE(dtype_size(dtype), "nrf_sample_logits: dtype %d", dtype);
    NRF_REQUIRE(row_stride >= 0, "nrf_sample_logits: row_stride %lld", (long long)row_stride);
    NRF_REQUIRE(temperature_rows || (temperature >= 0.0f && temperature < __builtin_inff()), "nrf_sample_logits: temperature must be finite and not negative");
    NRF_REQUIRE(top_p_rows || top_p == top_p, "nrf_sample_logits: top_p is NaN");
    NRF_REQUIRE(min_p_rows || min_p <= 1.0f, "nrf_sample_logits: min_p must be at most 1");
    if (size > kMaxSize || n_rows > kMaxRows || n_rows * n_draws > INT32_MAX)
        return fail(NRF_ERR_UNSUPPORTED, "nrf_sample_logits: size at most 2^28, n_rows at most 2^21, n_rows * n_draws below 2^31");
    if (n_rows == 0 || n_draws == 0) return NRF_OK;
    NRF_REQUIRE(logits && u && ids && prob, "nrf_sample_logits: null pointer");
    SampleArgs a;
    a.logits = logits, a.stride = row_stride, a.u = u;
    a.temperature_v = temperature_rows, a.top_k_v = top_k_rows, a.top_p_v = top_p_rows, a.min_p_v = min_p_rows;
    a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
    a.rows = (int)n_rows, a.size = size, a.draws = n_draws, a.ids = ids, a.prob = prob;
    NRF_REQUIRE(workspace || nrf_sample_logits_workspace_bytes(n_rows, size, n_draws) == 0, "nrf_sample_logits: null pointer (workspace)");
    NRF_REQUIRE(((uintptr_t)workspace & 15) == 0, "nrf_sample_logits: workspace must be 16-byte aligned");
    const bool may_k = top_k_rows || (top_k > 0 && top_k < size), may_p = top_p_rows || top_p < 1.0f;
    RowWork *work = (RowWork *)workspace;
    hipStream_t s = as_stream(stream);
    if (dtype == NRF_F32) launch_sample<float>(a, may_k, may_p, work, s);
    else if (dtype == NRF_BF16) launch_sample<bf16_t>(a, may_k, may_p, work, s);
    else launch_sample<f16_t>(a, may_k, may_p, work, s);
    return check_launch("nrf_sample_logits");
}
