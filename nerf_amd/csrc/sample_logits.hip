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
// The cut (the last kept entry, by value and index) comes from a histogram of the row: 2048 bins of equal width below the maximum,
// counts and masses.  Masses there are 64-bit fixed point (2^62 / V for e = 1), because integer atomics give the same
// sums in any order.  The entries around the cut (up to 2048 of them) are then sorted in LDS.  A bin that holds more (many equal
// values, far outliers) is split again by the bits of its values until it does not, or holds one value only.
#include "nrf_types.h"

using namespace nrf;

namespace {

constexpr int kBins = 2048, kList = 2048, kMaxTiles = 1024;
constexpr int kMaxSize = 1 << 28, kMaxRows = 1 << 21;

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

struct Row {
    double top, inv_t;      // M and 1 / T (0 at T = 0)
    float topf;
    uint32_t top_key;
    bool flat;              // M = +inf or T = 0: mass 1 at M, 0 elsewhere
    const double *tab;      // 2^(j/16), LDS
};

// exp(y), y = (x - M) / T <= 0: y = (16 q + j) ln2 / 16 + r, |r| <= ln2 / 32, exp = 2^q tab[j] exp(r); the Taylor polynomial of
// degree 6 leaves r^7 / 5040 < 5e-16.
__device__ __forceinline__ double mass_of(const Row &w, uint32_t key) {
    if (key == w.top_key) return 1.0;
    if (w.flat || key == 0) return 0.0;
    const double y = fmax(((double)value_of(key) - w.top) * w.inv_t, -800.0);
    const double n = __builtin_rint(y * (16.0 * 1.44269504088896340736));
    const double r = fma(n, -0.69314718055994530942 / 16.0, y);
    double s = fma(r, 1.0 / 720.0, 1.0 / 120.0);
    s = fma(r, s, 1.0 / 24.0);
    s = fma(r, s, 1.0 / 6.0);
    s = fma(r, s, 0.5);
    s = fma(r, s, 1.0);
    s = fma(r, s, 1.0);
    const int q = (int)n;
    return __builtin_ldexp(s * w.tab[q & 15], q >> 4);
}

// Bin of the first histogram: equal widths below the maximum, the last bin open.  Every step is monotone in x.
__device__ __forceinline__ int bin_of(const Row &w, float scale, uint32_t key) {
    return (int)fminf((w.topf - value_of(key)) * scale, (float)(kBins - 1));
}

template <typename T>
__device__ __forceinline__ uint32_t load_key(const T *row, int i) { return key_of(to_f32(row[i])); }

// ---- block-wide helpers (BLOCK threads, all of them call)
template <int BLOCK> struct Shared {
    static constexpr int kWaves = BLOCK / 64;
    double tab[16];
    double wave_d[kWaves];
    uint64_t wave_u[kWaves];
    uint32_t wave_a[kWaves];
    uint32_t count;                    // entries in `list`
    uint64_t found[3];                 // what one thread found for all
    uint64_t list[kList];
    double mass[kList];
};
struct Histogram {
    uint32_t cnt[kBins];
    uint64_t mass[kBins];
};

// Sum of the values of the threads before this one, in a fixed order of additions; *total = the sum of all.
template <int BLOCK, typename V, typename S>
__device__ __forceinline__ V block_scan(V v, S *sums, V *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const V y = __shfl_up(v, d);
        if (lane >= d) v += y;
    }
    if (lane == 63) sums[wave] = v;
    V before = __shfl_up(v, 1);
    if (lane == 0) before = 0;
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
__device__ __forceinline__ void block_max_min(uint64_t &best, uint32_t &lo, Shared<BLOCK> &s) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, d));
        lo = min(lo, (uint32_t)__shfl_xor(lo, d));
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) s.wave_u[wave] = best, s.wave_a[wave] = lo;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) best = max(best, s.wave_u[w]), lo = min(lo, s.wave_a[w]);
    __syncthreads();
}

// list[0 .. n) into rising order; n <= kList.  Bitonic, padded with ~0 to a power of two.
template <int BLOCK>
__device__ void sort_list(Shared<BLOCK> &s, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += BLOCK) s.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int p = threadIdx.x; p < size / 2; p += BLOCK) {
                const int a = ((p & ~(j - 1)) << 1) | (p & (j - 1)), b = a | j;
                const uint64_t x = s.list[a], y = s.list[b];
                if ((x > y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;
            }
            __syncthreads();
        }
}

// Order of the entries: larger value first, then smaller index.
__device__ __forceinline__ uint64_t by_value(uint32_t key, int i) { return ((uint64_t)~key << 32) | (uint32_t)i; }

// Entries 0 .. n of the list from the order of value to that of the index, as (index, key).
template <int BLOCK>
__device__ __forceinline__ void list_by_index(Shared<BLOCK> &s, int n) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += BLOCK) {
        const uint64_t c = s.list[i];
        s.list[i] = (c << 32) | (uint32_t)~(uint32_t)(c >> 32);
    }
    __syncthreads();
    sort_list<BLOCK>(s, n);
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

__device__ __forceinline__ double kept_mass(const Row &w, const Filter &f, uint32_t key, int i) {
    if (key == 0 || (f.cut && !f.keeps(key, i))) return 0.0;
    const double e = mass_of(w, key);
    return e >= f.m ? e : 0.0;
}

// What stands before a place in the order: entries and their mass.
struct Above {
    uint32_t cnt;
    uint64_t mass;
};

// Fixed-point masses: e * 2^shift, the sum of a whole row stays below 2^63.
__device__ __forceinline__ uint64_t fixed(double e, int shift) { return (uint64_t)__builtin_ldexp(e, shift); }

// ---- a row's parameters
struct RowState {
    Row w;
    Filter f;
    bool valid, use_p;      // use_p: top-p leaves something out, if anything does
    float t, scale;         // scale: bins of the first histogram
    int shift, first;       // first: the lowest index of the maximum
};

// best: the largest key and, in the low half, ~(its lowest index); lo: the smallest key that can be drawn.
__device__ __forceinline__ RowState row_state(const SampleArgs &a, int r, uint64_t best, uint32_t lo, const double *tab) {
    RowState o;
    const float p = a.top_p_v ? a.top_p_v[r] : a.top_p, m = a.min_p_v ? a.min_p_v[r] : a.min_p;
    const int k = a.top_k_v ? a.top_k_v[r] : a.top_k;
    o.t = a.temperature_v ? a.temperature_v[r] : a.temperature;
    const uint32_t hi = (uint32_t)(best >> 32);
    o.valid = hi != 0 && o.t >= 0.0f && o.t < __builtin_inff() && p == p && m == m;
    o.first = (int)~(uint32_t)best;
    o.w.topf = value_of(hi), o.w.top = o.w.topf, o.w.top_key = hi, o.w.tab = tab;
    o.w.flat = o.t == 0.0f || o.w.topf == __builtin_inff();
    o.w.inv_t = o.w.flat ? 0.0 : 1.0 / (double)o.t;
    o.f.k = k <= 0 || k > a.size ? a.size : k;
    o.f.p = p, o.f.m = fmin((double)m, 1.0);
    o.use_p = p < 1.0f;
    o.f.cut = o.f.k < a.size || o.use_p;
    o.f.key = 0, o.f.idx = a.size;
    o.scale = fminf((float)kBins / fminf(o.w.topf - value_of(lo), 64.0f * o.t), 1e30f);
    o.shift = 62;
    for (int v = a.size; v > 0; v >>= 1) --o.shift;
    return o;
}

template <typename T>
__device__ __forceinline__ void scan_max_min(const T *row, int begin, int end, uint64_t &best, uint32_t &lo) {
    for (int i = begin + threadIdx.x; i < end; i += blockDim.x) {
        const uint32_t key = load_key(row, i);
        const uint64_t c = ((uint64_t)key << 32) | (uint32_t)~i;
        if (key) best = max(best, c), lo = min(lo, key);
    }
}

template <typename T>
__device__ __forceinline__ void add_to_histogram(Histogram &h, const RowState &o, const T *row, int begin, int end) {
    for (int i = begin + threadIdx.x; i < end; i += blockDim.x) {
        const uint32_t key = load_key(row, i);
        if (key) {
            const int b = bin_of(o.w, o.scale, key);
            atomicAdd(&h.cnt[b], 1u);
            if (o.use_p)      // masses only where top-p asks for them
                atomicAdd((unsigned long long *)&h.mass[b], (unsigned long long)fixed(mass_of(o.w, key), o.shift));
        }
    }
}

// ---- the cut
// In a sorted list whose first entry has `above` before it: the last of the entries that are among the first `last` and have less
// than `want` of mass before them (by_mass).  Returns how many entries of the list that keeps; mass_at: mass up to entry `last`.
template <int BLOCK>
__device__ int cut_list(Shared<BLOCK> &s, const RowState &o, Filter &f, int n, Above above, int last, bool by_mass, double p,
                        double want, uint64_t *mass_at) {
    constexpr int kPer = kList / BLOCK;
    uint64_t e[kPer], run = 0;
    const int i0 = threadIdx.x * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        e[j] = i0 + j < n ? fixed(mass_of(o.w, ~(uint32_t)(s.list[i0 + j] >> 32)), o.shift) : 0;
        run += e[j];
    }
    unsigned long long all;
    uint64_t before = above.mass + block_scan<BLOCK, unsigned long long>(run, (unsigned long long *)s.wave_u, &all);
    if (last <= n) {
        uint64_t b = before;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            b += e[j];
            if (i0 + j == last - 1) s.found[0] = b;
        }
        __syncthreads();
        *mass_at = s.found[0];
        __syncthreads();
        if (p >= 0.0) want = p * (double)*mass_at;                     // top-p of the mass found here
    }
    uint32_t mine = 0, kept;                                           // a prefix: counting is enough
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const bool first = above.cnt == 0 && i0 + j == 0;
        if (i0 + j < min(n, last) && (!by_mass || (double)before < want || first)) ++mine;
        before += e[j];
    }
    block_scan<BLOCK, uint32_t>(mine, s.wave_a, &kept);
    const uint64_t c = s.list[kept > 0 ? kept - 1 : 0];
    f.key = ~(uint32_t)(c >> 32);
    f.idx = (int)(uint32_t)c;
    __syncthreads();
    return (int)kept;
}

// The bin that takes the running count to `want` (by_count), or the running mass to `wantm`; adds what stands before it to
// `above`.  kBins: none does.
template <int BLOCK>
__device__ int find_bin(Shared<BLOCK> &s, const Histogram &h, bool by_count, uint32_t want, double wantm, Above &above) {
    constexpr int kPer = kBins / BLOCK;
    const int b0 = threadIdx.x * kPer;
    uint32_t c[kPer], cs = 0, call;
    uint64_t m[kPer], ms = 0;
    unsigned long long mall;
#pragma unroll
    for (int j = 0; j < kPer; ++j) c[j] = h.cnt[b0 + j], m[j] = h.mass[b0 + j], cs += c[j], ms += m[j];
    uint64_t cb = above.cnt + block_scan<BLOCK, uint32_t>(cs, s.wave_a, &call);
    uint64_t mb = above.mass + block_scan<BLOCK, unsigned long long>(ms, (unsigned long long *)s.wave_u, &mall);
    if (threadIdx.x == 0) s.found[0] = kBins;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const bool hit = by_count ? cb < want && cb + c[j] >= want : (double)mb < wantm && (double)(mb + m[j]) >= wantm;
        if (hit) s.found[0] = b0 + j, s.found[1] = cb, s.found[2] = mb;
        cb += c[j], mb += m[j];
    }
    __syncthreads();
    const int bin = (int)s.found[0];
    if (bin < kBins) above.cnt = (uint32_t)s.found[1], above.mass = s.found[2];
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
__device__ Step make_step(Shared<BLOCK> &s, const Histogram &h, const RowState &o, bool by_count, uint64_t mass_k) {
    Step st;
    st.by_count = by_count;
    st.wantm = fmax(o.f.p * (double)mass_k, 0.5);          // top-p keeps at least the first
    st.above = Above{0, 0};
    st.bin = find_bin<BLOCK>(s, h, by_count, o.f.k, st.wantm, st.above);
    st.any = st.bin < kBins;
    st.n = st.any ? h.cnt[st.bin] : 0;
    st.prefix = st.above.cnt + st.n <= (uint32_t)kList;
    st.fits = st.prefix || st.n <= (uint32_t)kList;
    st.from = st.prefix ? 0 : st.bin;
    if (st.prefix) st.above = Above{0, 0};
    return st;
}

// Top-k where it leaves something out, else top-p of the whole mass.
template <int BLOCK>
__device__ Step first_step(Shared<BLOCK> &s, const Histogram &h, RowState &o) {
    constexpr int kPer = kBins / BLOCK;
    uint32_t c = 0, total;
    unsigned long long m = 0, mass;
#pragma unroll
    for (int j = 0; j < kPer; ++j) c += h.cnt[threadIdx.x * kPer + j], m += h.mass[threadIdx.x * kPer + j];
    block_scan<BLOCK, uint32_t>(c, s.wave_a, &total);
    block_scan<BLOCK, unsigned long long>(m, (unsigned long long *)s.wave_u, &mass);
    if (o.f.k > (int)total) o.f.k = (int)total;
    if (o.f.k == (int)total && !o.use_p) {
        Step none;
        none.any = none.fits = none.prefix = false;
        return none;
    }
    return make_step<BLOCK>(s, h, o, o.f.k < (int)total, mass);
}

template <int BLOCK, typename T>
__device__ void gather_list(Shared<BLOCK> &s, const RowState &o, const T *row, int size, const Step &st) {
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < size; i += BLOCK) {
        const uint32_t key = load_key(row, i);
        if (key) {
            const int b = bin_of(o.w, o.scale, key);
            if (b >= st.from && b <= st.bin) s.list[atomicAdd(&s.count, 1u)] = by_value(key, i);
        }
    }
    __syncthreads();
}

template <int BLOCK>
__device__ __forceinline__ void clear_histogram(Histogram &h) {
    for (int b = threadIdx.x; b < kBins; b += BLOCK) h.cnt[b] = 0, h.mass[b] = 0;
    __syncthreads();
}

// A cut inside a bin that holds more than the list: the bin's range of keys is split again (whole row per step) until the
// entries fit, or share one value.  Uses up the histogram.
template <int BLOCK, typename T>
__device__ void cut_range(Shared<BLOCK> &s, Histogram &h, const RowState &o, Filter &f, const T *row, int size, const Step &st,
                          uint64_t *mass_at) {
    uint64_t best = 0;
    uint32_t lo = 0xffffffffu;
    for (int i = threadIdx.x; i < size; i += BLOCK) {
        const uint32_t key = load_key(row, i);
        if (key && bin_of(o.w, o.scale, key) == st.bin) best = max(best, (uint64_t)key << 32), lo = min(lo, key);
    }
    block_max_min<BLOCK>(best, lo, s);
    uint32_t hi = (uint32_t)(best >> 32), n = st.n;
    Above above = st.above;
    while (n > (uint32_t)kList && lo < hi) {
        int bits = 0;
        while (((hi - lo) >> bits) >= (uint32_t)kBins) ++bits;
        clear_histogram<BLOCK>(h);
        for (int i = threadIdx.x; i < size; i += BLOCK) {
            const uint32_t key = load_key(row, i);
            if (key >= lo && key <= hi) {
                atomicAdd(&h.cnt[(hi - key) >> bits], 1u);
                atomicAdd((unsigned long long *)&h.mass[(hi - key) >> bits], (unsigned long long)fixed(mass_of(o.w, key), o.shift));
            }
        }
        __syncthreads();
        const int bin = min(find_bin<BLOCK>(s, h, st.by_count, f.k, st.wantm, above), kBins - 1);
        n = h.cnt[bin];
        hi -= (uint32_t)bin << bits;
        if (hi - lo > (1u << bits) - 1) lo = hi - ((1u << bits) - 1);
        __syncthreads();
    }
    if (n <= (uint32_t)kList) {
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < size; i += BLOCK) {
            const uint32_t key = load_key(row, i);
            if (key >= lo && key <= hi) s.list[atomicAdd(&s.count, 1u)] = by_value(key, i);
        }
        __syncthreads();
        sort_list<BLOCK>(s, n);
        cut_list<BLOCK>(s, o, f, n, above, st.by_count ? (int)(f.k - above.cnt) : kList + 1, !st.by_count, -1.0, st.wantm, mass_at);
        return;
    }
    // one value, more than kList times: the first q of them by index
    const uint64_t e = fixed(mass_of(o.w, hi), o.shift);
    uint32_t q = n;
    if (st.by_count) q = f.k - above.cnt;
    else if (e > 0) {
        // the smallest q whose mass reaches the target; the quotient's rounding is mended
        q = (uint32_t)fmin((double)n, fmax(1.0, __builtin_ceil((st.wantm - (double)above.mass) / (double)e)));
        while (q > 1 && (double)(above.mass + (q - 1) * e) >= st.wantm) --q;
        while (q < n && (double)(above.mass + q * e) < st.wantm) ++q;
    }
    *mass_at = above.mass + q * e;
    f.key = hi;
    uint32_t seen = 0;                                   // entries of that value in the chunks before
    for (int i0 = 0; i0 < size && seen < q; i0 += BLOCK) {
        const int i = i0 + threadIdx.x;
        const uint32_t is = i < size && load_key(row, i) == hi;
        uint32_t all;
        const uint32_t before = seen + block_scan<BLOCK, uint32_t>(is, s.wave_a, &all);
        if (is && before + 1 == q) s.found[0] = i;
        seen += all;
    }
    __syncthreads();
    f.idx = (int)s.found[0];
    __syncthreads();
}

// Both cuts of a long row, from its histogram (used up where a bin is too full).  gathered: the entries of the first step are in
// the list already.  Returns the number of kept entries where the list holds all of them, sorted by value; else -1.
template <int BLOCK, typename T>
__device__ int select_cut(Shared<BLOCK> &s, Histogram &h, RowState &o, const T *row, int size, Step st, bool gathered) {
    const bool by_k = st.any && st.by_count;
    while (st.any) {
        uint64_t mass_at = 0;
        if (st.fits) {
            if (!gathered) gather_list<BLOCK, T>(s, o, row, size, st);
            gathered = false;
            const int n = s.count;
            sort_list<BLOCK>(s, n);
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
            if (by_k && st.by_count && o.use_p) {
                clear_histogram<BLOCK>(h);
                add_to_histogram<T>(h, o, row, 0, size);
                __syncthreads();
            }
        }
        if (!(st.by_count && o.use_p)) break;
        st = make_step<BLOCK>(s, h, o, false, mass_at);
    }
    if (!st.any) o.f.cut = false;
    return -1;
}

// ---- draws
__device__ __forceinline__ double mass_or_zero(const RowState &o, uint32_t key) {
    const double e = mass_of(o.w, key);
    return e >= o.f.m ? e : 0.0;
}

// From the list: kept entries 0 .. n by index as (index, key); a thread a draw.
template <int BLOCK>
__device__ void draw_from_list(Shared<BLOCK> &s, const RowState &o, int n, const float *u, int draws, int64_t *ids, float *prob) {
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
    for (int j = tid; j < draws; j += BLOCK) {
        const float uj = u[j];
        const double want = (double)fminf(fmaxf(uj, 0.0f), 1.0f) * total;
        int a = 0, b = n - 1;                          // first entry whose running mass exceeds `want`
        while (a < b) {
            const int mid = (a + b) >> 1;
            if (s.mass[mid] > want) b = mid;
            else a = mid + 1;
        }
        // u = 1, or a product that rounds up to the total: back to the last entry that has mass
        while (a > 0 && mass_or_zero(o, (uint32_t)s.list[a]) == 0.0) --a;
        const double m = mass_or_zero(o, (uint32_t)s.list[a]);
        ids[j] = uj == uj ? (int64_t)(s.list[a] >> 32) : -1;
        prob[j] = uj == uj ? (float)(m / total) : 0.0f;
    }
}

// Tiles of a row: their masses, added lane by lane, then over the wave.
__device__ __forceinline__ int tile_of(int size) {
    int tile = 1024;
    while ((size + tile - 1) / tile > kMaxTiles) tile <<= 1;
    return tile;
}

template <typename T>
__device__ __forceinline__ double tile_mass(const RowState &o, const T *row, int size, int tile, int q) {
    const int lane = threadIdx.x & 63, end = min(size, (q + 1) * tile);
    double sum = 0.0;
    for (int i = q * tile + lane; i < end; i += 64) sum += kept_mass(o.w, o.f, load_key(row, i), i);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    return sum;
}

// tiles[0 .. n) -> running sums
template <int BLOCK>
__device__ void scan_tiles(Shared<BLOCK> &s, double *tiles, int n) {
    constexpr int kPer = kMaxTiles / BLOCK;
    const int q0 = threadIdx.x * kPer;
    double v[kPer], run = 0.0, total;
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = q0 + j < n ? tiles[q0 + j] : 0.0, run += v[j];
    double cum = block_scan<BLOCK, double>(run, s.wave_d, &total);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        cum += v[j];
        if (q0 + j < n) tiles[q0 + j] = cum;
    }
    __syncthreads();
}

// One draw by a wave: the tile by its running sum, then the entry.
template <typename T>
__device__ void draw_from_tiles(const RowState &o, const T *row, int size, int tile, const double *tiles, int n_tiles, float uj,
                                int64_t *id, float *prob) {
    const int lane = threadIdx.x & 63;
    const double total = tiles[n_tiles - 1], want = (double)fminf(fmaxf(uj, 0.0f), 1.0f) * total;
    int a = 0, b = n_tiles - 1;
    while (a < b) {
        const int mid = (a + b) >> 1;
        if (tiles[mid] > want) b = mid;
        else a = mid + 1;
    }
    while (a > 0 && tiles[a] <= tiles[a - 1]) --a;       // u = 1: back to the last tile that has mass
    double cum = a > 0 ? tiles[a - 1] : 0.0, mass = 0.0;
    int at = 0;
    const int end = min(size, (a + 1) * tile);
    for (int i0 = a * tile; i0 < end; i0 += 64) {
        const int i = i0 + lane;
        const double e = i < end ? kept_mass(o.w, o.f, load_key(row, i), i) : 0.0;
        double c = e;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double y = __shfl_up(c, d);
            if (lane >= d) c += y;
        }
        const uint64_t over = __ballot(e > 0.0 && cum + c > want), some = __ballot(e > 0.0);
        // the first that exceeds; where the sums' rounding leaves none, the last one with mass
        if (some) {
            const int src = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
            at = i0 + src, mass = __shfl(e, src);
        }
        if (over) break;
        cum += __shfl(c, 63);
    }
    if (lane == 0) {
        *id = uj == uj ? at : -1;
        *prob = uj == uj ? (float)(mass / total) : 0.0f;
    }
}

// Rows without anything to draw (id -1), and T = 0 (the first maximum): true if this was one of them.
__device__ __forceinline__ bool plain_row(const RowState &o, const float *u, int draws, int64_t *ids, float *prob, int first, int step) {
    if (o.valid && o.t > 0.0f) return false;
    for (int j = first; j < draws; j += step) {
        const bool ok = o.valid && u[j] == u[j];
        ids[j] = ok ? o.first : -1;
        prob[j] = ok ? 1.0f : 0.0f;
    }
    return true;
}

// ---- one block a row
// LONG: rows beyond kList entries, by the histogram; otherwise the whole row goes into the list.
template <typename T, int BLOCK, bool LONG>
__global__ void __launch_bounds__(BLOCK) sample_row_kernel(const SampleArgs a) {
    __shared__ Shared<BLOCK> s;
    const int tid = threadIdx.x, r = blockIdx.x, size = a.size;
    const T *row = (const T *)a.logits + (int64_t)r * a.stride;
    const float *u = a.u + (int64_t)r * a.draws;
    int64_t *ids = a.ids + (int64_t)r * a.draws;
    float *prob = a.prob + (int64_t)r * a.draws;

    uint64_t best = 0;
    uint32_t lo = 0xffffffffu;
    scan_max_min<T>(row, 0, size, best, lo);
    if (tid < 16) s.tab[tid] = exp2(tid / 16.0);
    block_max_min<BLOCK>(best, lo, s);
    RowState o = row_state(a, r, best, lo, s.tab);
    if (plain_row(o, u, a.draws, ids, prob, tid, BLOCK)) return;

    int listed = -1;
    if constexpr (!LONG) {
        if (!o.f.cut) {
            for (int i = tid; i < size; i += BLOCK) s.list[i] = ((uint64_t)i << 32) | load_key(row, i);
            __syncthreads();
            return draw_from_list<BLOCK>(s, o, size, u, a.draws, ids, prob);
        }
        if (tid == 0) s.count = 0;
        __syncthreads();
        for (int i = tid; i < size; i += BLOCK) {
            const uint32_t key = load_key(row, i);
            if (key) s.list[atomicAdd(&s.count, 1u)] = by_value(key, i);
        }
        __syncthreads();
        const int n = s.count;
        sort_list<BLOCK>(s, n);
        uint64_t mass_at;
        listed = cut_list<BLOCK>(s, o, o.f, n, Above{0, 0}, min(o.f.k, n), o.use_p, o.f.p, 0.0, &mass_at);
    } else if (o.f.cut) {
        __shared__ Histogram h;
        clear_histogram<BLOCK>(h);
        add_to_histogram<T>(h, o, row, 0, size);
        __syncthreads();
        const Step st = first_step<BLOCK>(s, h, o);
        listed = select_cut<BLOCK, T>(s, h, o, row, size, st, false);
    }
    if (listed > 0) {
        list_by_index<BLOCK>(s, listed);
        return draw_from_list<BLOCK>(s, o, listed, u, a.draws, ids, prob);
    }
    if constexpr (LONG) {
        __shared__ double tiles[kMaxTiles];
        const int tile = tile_of(size), n_tiles = (size + tile - 1) / tile;
        for (int q = tid >> 6; q < n_tiles; q += BLOCK / 64) {
            const double m = tile_mass<T>(o, row, size, tile, q);
            if ((tid & 63) == 0) tiles[q] = m;
        }
        __syncthreads();
        scan_tiles<BLOCK>(s, tiles, n_tiles);
        for (int j = tid >> 6; j < a.draws; j += BLOCK / 64)
            draw_from_tiles<T>(o, row, size, tile, tiles, n_tiles, u[j], ids + j, prob + j);
    }
}

template <typename T>
void launch_sample(const SampleArgs &a, hipStream_t s) {
    if (a.size <= kList) sample_row_kernel<T, 256, false><<<a.rows, 256, 0, s>>>(a);
    else sample_row_kernel<T, 1024, true><<<a.rows, 1024, 0, s>>>(a);
}

}  // namespace

extern "C" int nrf_sample_logits(const void *logits, int64_t row_stride, int32_t dtype, int64_t n_rows, int32_t size, int32_t n_draws,
                                 float temperature, int32_t top_k, float top_p, float min_p, const float *temperature_rows,
                                 const int32_t *top_k_rows, const float *top_p_rows, const float *min_p_rows, const float *u,
                                 int64_t *ids, float *prob, void *stream) {
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
    hipStream_t s = as_stream(stream);
    if (dtype == NRF_F32) launch_sample<float>(a, s);
    else if (dtype == NRF_BF16) launch_sample<bf16_t>(a, s);
    else launch_sample<f16_t>(a, s);
    return check_launch("nrf_sample_logits");
}
