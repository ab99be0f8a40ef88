// Code tables: out[i] = scale * table[ids[i]] and its gradient grad[v] = scale * sum of g[i] over the i with ids[i] = v.
//
// Forward: every output element is one load, one product, one store; HBM-bound.  The output is cut into chunks of up to 16
// bytes, consecutive lanes on consecutive chunks, so narrow rows (two features) and wide ones take the same path.  16384 rows of
// 4096 bf16: 34 us (134 MB written, repeated rows read once); 2^21 rows of two f32 from 524288: 17.5 us, a cache line a row.
//
// Gradient: the sum over equal ids is taken in a fixed order (no float atomics: results repeat bit for bit).
//   1. a stable sort of the pairs (id, position): least significant digit first, digits of up to 10 bits.  The blocks of the
//      first launch that do not sort write the zeros of the dense gradient meanwhile.
//   2. the sorted list is cut into tiles of T tokens; a team of threads owns a tile and up to 256 vectors of columns, gathers the
//      tokens' rows and adds runs of equal ids in f32 registers.  A run inside the tile goes straight to its row of grad; one
//      that reaches beyond an end of it leaves a partial sum (at most two per tile).
//   3. the team whose tile a crossing run starts in adds up the run's partial sums.
// Few rows and up to 16384 tokens go without the sort, narrow rows of g travel with their ids instead of being gathered: below.
// Any distribution of ids costs the same in 2, and a run of n tokens costs n / T partial sums in 3.  16384 rows of 4096 bf16 into
// 131072: 231 us, 154 of them the zeros (7.0 TB/s), 70 the sums; 786432 rows of 33 f32 into 200: 55 us, of which 21 to 26 are 2 (4 to
// 5 TB/s) and 22 the sort.
#include "nrf_types.h"

using namespace nrf;

namespace {

constexpr int kMaxDim = 32768;

// Rows are taken in vectors of VW elements at any alignment (the hardware splits what crosses a line); where VW does not divide a row,
// its last vector overlaps the one before and both give the shared elements the same bits.  The gradient of 786432 x 33 f32 over 200 rows:
// 49 us a call against 58 by single elements.
template <int VW>
__device__ __forceinline__ int column(int vector, int dim) { return min(vector * VW, dim - VW); }

// ---------------------------------------------------------------------------------------------------- forward
constexpr int kFwdUnroll = 4;

// A store past the caches, in words of up to 16 bytes
template <int BYTES> struct Word;
template <> struct Word<2> { typedef uint16_t type; };
template <> struct Word<4> { typedef uint32_t type __attribute__((aligned(2))); };
template <> struct Word<8> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Word<16> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <typename V>
__device__ __forceinline__ void store_once(V *p, V v) {
    constexpr int W = sizeof(V) < 16 ? sizeof(V) : 16, N = sizeof(V) / W;
    typedef typename Word<W>::type U;
    struct All { U w[N]; };
    const All all = __builtin_bit_cast(All, v);
#pragma unroll
    for (int k = 0; k < N; ++k) __builtin_nontemporal_store(all.w[k], reinterpret_cast<U *>(p) + k);
}

// blockDim 256; chunk = VW elements of one row; `per_row` = dim / VW, up; magic = ceil(2^32 / per_row).  An output that the L2s could not
// hold (32 MB) goes past them, which leaves them to rows that are met again: 16384 ids x 4096 bf16 32.8 us against 34.9.
template <typename T, typename O, int VW, typename I>
__global__ void __launch_bounds__(256) lookup_fwd_kernel(const T *__restrict__ table, int64_t stride, int64_t n_rows,
                                                         const I *__restrict__ ids, int64_t chunks, int dim, uint32_t per_row,
                                                         uint32_t magic, float scale, O *__restrict__ out) {
    const int64_t c0 = (int64_t)blockIdx.x * (256 * kFwdUnroll);
    const int64_t r0 = c0 / per_row;                       // block-uniform: one 64-bit division a block
    const uint32_t rem = (uint32_t)(c0 - r0 * per_row);
    const bool once = chunks * (int64_t)sizeof(Pack<O, VW>) > 32 << 20;
    Pack<T, VW> v[kFwdUnroll];
    int64_t id[kFwdUnroll];
    int col[kFwdUnroll];
    int64_t row[kFwdUnroll];
    // loads without branches between them: chunks behind the last one read the last one's row, ids outside the table row 0
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
        uint32_t local = u * 256 + threadIdx.x;
        if (c0 + local >= chunks) local = (uint32_t)(chunks - 1 - c0);
        const uint32_t off = rem + local;
        // off < per_row + 1024 and per_row <= 32768: off * per_row < 2^32, where the product with the magic is exact
        const uint32_t q = per_row == 1 ? off : __umulhi(off, magic);
        row[u] = r0 + q;
        id[u] = (int64_t)ids[row[u]];
        col[u] = column<VW>((int)(off - q * per_row), dim);
    }
    if (n_rows > 0) {
#pragma unroll
        for (int u = 0; u < kFwdUnroll; ++u) {
            const int64_t r = (uint64_t)id[u] < (uint64_t)n_rows ? id[u] : 0;
            v[u] = *reinterpret_cast<const Pack<T, VW> *>(table + r * stride + col[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
        const int64_t c = c0 + u * 256 + threadIdx.x;
        if (c < chunks) {
            Pack<O, VW> o;
#pragma unroll
            for (int j = 0; j < VW; ++j)
                o.e[j] = from_f32<O>((uint64_t)id[u] < (uint64_t)n_rows ? to_f32(v[u].e[j]) * scale : __uint_as_float(0x7fc00000u));
            Pack<O, VW> *to = reinterpret_cast<Pack<O, VW> *>(out + row[u] * dim + col[u]);
            if (once) store_once(to, o);
            else *to = o;
        }
    }
}

template <typename T, typename O, int VW>
void launch_fwd(const void *table, int64_t stride, int64_t n_rows, const void *ids, bool i64, int64_t n, int dim, float scale,
                void *out, hipStream_t s) {
    const uint32_t per_row = (uint32_t)((dim + VW - 1) / VW);
    const uint32_t magic = (uint32_t)(((1ull << 32) + per_row - 1) / per_row);
    const int64_t chunks = n * per_row;
    const int blocks = (int)((chunks + 256 * kFwdUnroll - 1) / (256 * kFwdUnroll));
    if (i64)
        lookup_fwd_kernel<T, O, VW, int64_t><<<blocks, 256, 0, s>>>((const T *)table, stride, n_rows, (const int64_t *)ids, chunks,
                                                                    dim, per_row, magic, scale, (O *)out);
    else
        lookup_fwd_kernel<T, O, VW, int32_t><<<blocks, 256, 0, s>>>((const T *)table, stride, n_rows, (const int32_t *)ids, chunks,
                                                                    dim, per_row, magic, scale, (O *)out);
}

template <typename T, typename O>
void pick_fwd(int vw, const void *table, int64_t stride, int64_t n_rows, const void *ids, bool i64, int64_t n, int dim,
              float scale, void *out, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (vw == 8) return launch_fwd<T, O, 8>(table, stride, n_rows, ids, i64, n, dim, scale, out, s);
    if (vw >= 4) return launch_fwd<T, O, 4>(table, stride, n_rows, ids, i64, n, dim, scale, out, s);
    if (vw == 2) return launch_fwd<T, O, 2>(table, stride, n_rows, ids, i64, n, dim, scale, out, s);
    launch_fwd<T, O, 1>(table, stride, n_rows, ids, i64, n, dim, scale, out, s);
}

// ---------------------------------------------------------------------------------------------------- sort of (id, position)
// Pair: x = key (the id; n_rows for tokens that take no part: ids outside the table, the padding id), y = position.
constexpr int kItems = 16;                  // most items of a thread, one-block sort
constexpr int kSmall = 1024 * kItems;       // most items the one-block sort takes
constexpr int kTileItems = 4;               // items of a thread, many-block sort: 1024 threads, two blocks fill a CU's waves ...
constexpr int kFewItems = 2;                // ... and where few blocks have work, when the ranking's chain of items takes the time
constexpr int kTile = 1024 * kTileItems;
constexpr int kFewTiles = 64;               // blocks up to which each sums the counters of all (a scan launch costs 5 us)
constexpr int kMaxDigit = 10;               // bits of a digit: 16 waves' counters and the one-block sort's pairs fit LDS

template <typename I>
__device__ __forceinline__ uint32_t key_of(I id, uint32_t n_rows, int64_t padding) {
    const int64_t v = (int64_t)id;
    return (uint64_t)v < (uint64_t)n_rows && v != padding ? (uint32_t)v : n_rows;
}

// Lanes of the wave that hold the same digit (inactive lanes: never counted)
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, bool active) {
    uint64_t m = __ballot(active);
    for (int b = 0; b < bits; ++b) {
        const bool one = (d >> b) & 1;
        const uint64_t w = __ballot(one);
        m &= one ? w : ~w;
    }
    return m;
}

__device__ __forceinline__ int lanes_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// Rank of an item among the items of its digit that this wave saw before it; moves the wave's counter (one leader a digit).
// The counter is read by all lanes of the digit before the leader writes it: one wave, LDS accesses in order.
__device__ __forceinline__ uint32_t wave_rank(uint16_t *cnt, uint32_t d, int bits, bool active) {
    const uint64_t m = same_digit(d, bits, active);
    uint32_t r = 0;
    if (active) {
        const int below = lanes_below(m);
        const uint32_t c = *(volatile uint16_t *)&cnt[d];
        r = c + below;
        __builtin_amdgcn_wave_barrier();
        if (below == 0) *(volatile uint16_t *)&cnt[d] = (uint16_t)(c + __popcll(m));
    }
    __builtin_amdgcn_wave_barrier();
    return r;
}

// Exclusive scan of one value a thread over the block (WAVES waves); `sums`: WAVES words of LDS.
template <int WAVES>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    uint32_t base = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
        if (w < wave) base += sums[w];
    __syncthreads();
    return base + x - v;
}

// Zeros of the dense gradient, by the blocks of a launch that do not sort: kFill bytes each (blockDim 1024).
constexpr int kFill = 1024 * 16;
__device__ __forceinline__ void fill_zero(char *p, int64_t bytes, int b) {
    const int64_t begin = (int64_t)b * kFill, end = begin + kFill < bytes ? begin + kFill : bytes;
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && end - begin == kFill) {
        reinterpret_cast<uint4 *>(p + begin)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    } else {
        for (int64_t i = begin + 2 * threadIdx.x; i < end; i += 2048) *reinterpret_cast<uint16_t *>(p + i) = 0;
    }
}

// One block sorts up to kSmall pairs in LDS; a pass ranks by waves (items in order: wave, item, lane), then moves the pairs.
struct SmallSort {
    uint32_t key[kSmall];
    uint16_t pos[kSmall];
    uint16_t cnt[16][1 << kMaxDigit];
    uint32_t sums[16];
};

template <typename I>
__global__ void __launch_bounds__(1024) sort_small_kernel(const I *__restrict__ ids, int n, uint32_t n_rows, int64_t padding,
                                                          int passes, int digit, uint2 *__restrict__ pairs, void *grad,
                                                          int64_t grad_bytes) {
    if (blockIdx.x > 0) return fill_zero((char *)grad, grad_bytes, blockIdx.x - 1);
    __shared__ SmallSort s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bins = 1 << digit;
    // waves own consecutive ranges of `per` items (a multiple of 64), item k of a lane at wave * per + k * 64 + lane
    const int rounds = (n + 1023) / 1024, per = rounds * 64;
    uint32_t key[kItems], rank[kItems];
    uint16_t pos[kItems];
    for (int k = 0; k < kItems; ++k) {
        const int i = wave * per + k * 64 + lane;
        if (k < rounds && i < n) {
            key[k] = key_of(ids[i], n_rows, padding);
            pos[k] = (uint16_t)i;
        }
    }
    for (int p = 0; p < passes; ++p) {
        for (int b = tid; b < 16 * bins; b += 1024) s.cnt[b >> digit][b & (bins - 1)] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            if (k < rounds) {
                const bool on = wave * per + k * 64 + lane < n;
                rank[k] = wave_rank(s.cnt[wave], on ? (key[k] >> (p * digit)) & (bins - 1) : 0, digit, on);
            }
        __syncthreads();
        // counters -> first place of (digit, wave); digits in order, waves in order inside a digit
        uint32_t total = 0;
        if (tid < bins)
            for (int w = 0; w < 16; ++w) total += s.cnt[w][tid];
        uint32_t base = block_scan<16>(total, s.sums);
        if (tid < bins)
            for (int w = 0; w < 16; ++w) {
                const uint32_t c = s.cnt[w][tid];
                s.cnt[w][tid] = (uint16_t)base;          // places are below kSmall <= 2^14
                base += c;
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            if (k < rounds && wave * per + k * 64 + lane < n) {
                const uint32_t at = s.cnt[wave][(key[k] >> (p * digit)) & (bins - 1)] + rank[k];
                s.key[at] = key[k];
                s.pos[at] = pos[k];
            }
        __syncthreads();
        if (p + 1 < passes) {
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
                const int i = wave * per + k * 64 + lane;
                if (k < rounds && i < n) {
                    key[k] = s.key[i];
                    pos[k] = s.pos[i];
                }
            }
        }
    }
    for (int i = tid; i < n; i += 1024) pairs[i] = make_uint2(s.key[i], s.pos[i]);
}

// Many blocks, one digit: counts[block][bin]; the blocks behind the sorting ones write zeros (first digit only).
template <typename I, bool FIRST, int ITEMS>
__global__ void __launch_bounds__(1024) sort_count_kernel(const I *__restrict__ ids, const uint2 *__restrict__ in, int64_t n,
                                                          uint32_t n_rows, int64_t padding, int shift, int digit, int tiles,
                                                          uint32_t *__restrict__ counts, void *grad, int64_t grad_bytes) {
    if (FIRST && (int)blockIdx.x >= tiles) return fill_zero((char *)grad, grad_bytes, blockIdx.x - tiles);
    __shared__ uint32_t cnt[1 << kMaxDigit];
    const int bins = 1 << digit;
    if ((int)threadIdx.x < bins) cnt[threadIdx.x] = 0;
    const int64_t i0 = (int64_t)blockIdx.x * (1024 * ITEMS) + threadIdx.x;
    uint32_t key[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = i0 + k * 1024 < n ? i0 + k * 1024 : n - 1;
        key[k] = FIRST ? key_of(ids[i], n_rows, padding) : in[i].x;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (i0 + k * 1024 < n) atomicAdd(&cnt[(key[k] >> shift) & (bins - 1)], 1u);
    __syncthreads();
    if ((int)threadIdx.x < bins) counts[(int64_t)blockIdx.x * bins + threadIdx.x] = cnt[threadIdx.x];
}

// counts[*][bin] -> sums over the blocks before, totals[bin].  A block takes 64 bins (a lane each), its 16 waves a strip of
// the blocks each: sums of the strips, their running sum, then the strips again.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t *__restrict__ counts, uint32_t *__restrict__ totals, int bins,
                                                         int tiles) {
    __shared__ uint32_t strip[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bin = blockIdx.x * 64 + lane;
    const int per = (tiles + 15) / 16, t0 = wave * per, t1 = min(tiles, t0 + per);
    const bool on = bin < bins;
    uint32_t sum = 0;
    if (on) {
#pragma unroll 8
        for (int t = t0; t < t1; ++t) sum += counts[(int64_t)t * bins + bin];
    }
    strip[wave][lane] = sum;
    __syncthreads();
    uint32_t run = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        if (w == wave) run = all;
        all += strip[w][lane];
    }
    if (on) {
#pragma unroll 8
        for (int t = t0; t < t1; ++t) {
            const uint32_t c = counts[(int64_t)t * bins + bin];
            counts[(int64_t)t * bins + bin] = run;
            run += c;
        }
        if (wave == 0) totals[bin] = all;
    }
}

template <typename I, bool FIRST, int ITEMS>
__global__ void __launch_bounds__(1024) sort_scatter_kernel(const I *__restrict__ ids, const uint2 *__restrict__ in, int64_t n,
                                                            uint32_t n_rows, int64_t padding, int shift, int digit, int tiles,
                                                            const uint32_t *__restrict__ counts,
                                                            const uint32_t *__restrict__ totals, uint2 *__restrict__ out) {
    __shared__ uint32_t base[1 << kMaxDigit];
    __shared__ uint16_t cnt[16][1 << kMaxDigit], start[1 << kMaxDigit];
    __shared__ uint2 sorted[1024 * ITEMS];
    __shared__ uint32_t sums[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bins = 1 << digit;
    const int64_t i0 = (int64_t)blockIdx.x * (1024 * ITEMS) + wave * (64 * ITEMS) + lane;
    uint2 pair[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = i0 + k * 64 < n ? i0 + k * 64 : n - 1;
        pair[k] = FIRST ? make_uint2(key_of(ids[i], n_rows, padding), (uint32_t)i) : in[i];
    }
    uint32_t total = 0, before = 0;
    if (tid < bins) {
        if (tiles <= kFewTiles) {                          // no scan launch: the blocks before, and all of them
#pragma unroll 8
            for (int t = 0; t < tiles; ++t) {
                const uint32_t c = counts[t * bins + tid];
                total += c;
                before += t < (int)blockIdx.x ? c : 0;
            }
        } else {
            total = totals[tid], before = counts[(int64_t)blockIdx.x * bins + tid];
        }
    }
    for (int b = tid; b < 16 * bins; b += 1024) cnt[b >> digit][b & (bins - 1)] = 0;
    const uint32_t first = block_scan<16>(total, sums);        // first place of bin `tid` (ends in a barrier)
    uint32_t rank[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) rank[k] = wave_rank(cnt[wave], (pair[k].x >> shift) & (bins - 1), digit, i0 + k * 64 < n);
    __syncthreads();
    uint32_t mine = 0;
    if (tid < bins) {
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const uint32_t c = cnt[w][tid];
            cnt[w][tid] = (uint16_t)mine;
            mine += c;
        }
    }
    const uint32_t local = block_scan<16>(mine, sums);         // first place of the bin inside this block
    if (tid < bins) {
        start[tid] = (uint16_t)local;
        base[tid] = first + before - local;
    }
    __syncthreads();
    // in the order of the output through LDS: neighbouring lanes then write neighbouring places
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (i0 + k * 64 < n) {
            const uint32_t d = (pair[k].x >> shift) & (bins - 1);
            sorted[start[d] + cnt[wave][d] + rank[k]] = pair[k];
        }
    __syncthreads();
    const int64_t left = n - (int64_t)blockIdx.x * (1024 * ITEMS);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = k * 1024 + tid;
        if (i < left) {
            const uint2 v = sorted[i];
            out[(int64_t)(base[(v.x >> shift) & (bins - 1)] + i)] = v;
        }
    }
}

// ---------------------------------------------------------------------------------------------------- sums over runs of equal ids
struct SumArgs {
    const uint2 *pairs;
    const void *g;
    int64_t g_stride;
    void *grad;
    float *head, *tail;        // [tiles][dim]: partial sum of a run that began before the tile / that begins in it and goes on
    int64_t n, tiles;
    uint32_t n_rows;
    int dim, tile, lanes, chunks;      // a team of `lanes` threads covers 1 / chunks of the columns
    float scale;
};

constexpr int kBatch = 8;      // rows of g that a team has in flight
constexpr int kAlone = 4;      // batches of partial sums that a team adds alone

template <typename G, typename T, int VW>
__device__ __forceinline__ void store_row(const SumArgs &a, uint32_t key, int col, const float *acc) {
    Pack<T, VW> o;
#pragma unroll
    for (int j = 0; j < VW; ++j) o.e[j] = from_f32<T>(acc[j] * a.scale);
    *reinterpret_cast<Pack<T, VW> *>((T *)a.grad + (int64_t)key * a.dim + col) = o;
}

template <int VW>
__device__ __forceinline__ void store_part(float *p, int64_t tile, int dim, int col, const float *acc) {
#pragma unroll
    for (int j = 0; j < VW; ++j) p[tile * dim + col + j] = acc[j];
}

// Where a thread of the sum kernels works: teams of `lanes` neighbouring threads (no wave boundaries needed: nothing is exchanged
// between lanes), the column chunks of a tile in neighbouring teams.
struct Place {
    int64_t tile;
    int col;           // first column of this thread
    bool on;
};
template <int VW>
__device__ __forceinline__ Place place_of(const SumArgs &a) {
    const int teams = 256 / a.lanes, team = threadIdx.x / a.lanes;
    const int64_t at = (int64_t)blockIdx.x * teams + team;
    Place p;
    p.tile = a.chunks == 1 ? at : at / a.chunks;
    const int vector = (int)((at - p.tile * a.chunks) * a.lanes + (threadIdx.x - team * a.lanes));
    p.col = column<VW>(vector, a.dim);
    p.on = team < teams && p.tile < a.tiles && vector * VW < a.dim;
    return p;
}

template <typename G, typename T, int VW>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const SumArgs a) {
    const Place at = place_of<VW>(a);
    if (!at.on) return;
    const int64_t t = at.tile, i0 = t * a.tile, i1 = i0 + a.tile < a.n ? i0 + a.tile : a.n;
    const int col = at.col;
    const G *g = (const G *)a.g + col;
    uint32_t cur = a.pairs[i0].x;
    if (cur >= a.n_rows) return;                           // sorted: nothing but tokens that take no part from here on
    bool before = i0 > 0 && a.pairs[i0 - 1].x == cur;
    float acc[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) acc[j] = 0.0f;
    uint2 next[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) next[k] = a.pairs[i0 + k < i1 ? i0 + k : i1 - 1];
    for (int64_t i = i0; i < i1; i += kBatch) {
        uint2 p[kBatch];
        Pack<G, VW> v[kBatch];
        // positions are tokens whatever their id: no branch stands between the loads; the next batch's pairs travel with the rows
#pragma unroll
        for (int k = 0; k < kBatch; ++k) p[k] = next[k], v[k] = *reinterpret_cast<const Pack<G, VW> *>(g + (int64_t)p[k].y * a.g_stride);
        if (i + kBatch < i1) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) next[k] = a.pairs[i + kBatch + k < i1 ? i + kBatch + k : i1 - 1];
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (i + k >= i1) break;
            if (p[k].x != cur) {
                if (before) store_part<VW>(a.head, t, a.dim, col, acc);
                else store_row<G, T, VW>(a, cur, col, acc);
                cur = p[k].x;
                before = false;
                if (cur >= a.n_rows) return;
#pragma unroll
                for (int j = 0; j < VW; ++j) acc[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < VW; ++j) acc[j] += to_f32(v[k].e[j]);
        }
    }
    if (before) store_part<VW>(a.head, t, a.dim, col, acc);
    else if (i1 < a.n && a.pairs[i1].x == cur) store_part<VW>(a.tail, t, a.dim, col, acc);
    else store_row<G, T, VW>(a, cur, col, acc);
}

// acc += head[s0 .. s1) in order
template <int VW>
__device__ __forceinline__ void add_heads(const SumArgs &a, int64_t s0, int64_t s1, int col, float *acc) {
    for (int64_t s = s0; s < s1; s += kBatch) {
        float v[kBatch][VW];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
            for (int j = 0; j < VW; ++j) v[k][j] = a.head[(s + k < s1 ? s + k : s1 - 1) * a.dim + col + j];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
            for (int j = 0; j < VW; ++j) acc[j] += s + k < s1 ? v[k][j] : 0.0f;
    }
}

// Runs that cross tiles: the team of the tile a run starts in adds tail[tile] and head[tile + 1 ..]; where the run covers more
// than kAlone * kBatch further tiles, the block's teams take a slice of them each and the slices are added in order.
template <typename G, typename T, int VW>
__global__ void __launch_bounds__(256) sum_join_kernel(const SumArgs a) {
    __shared__ int long_team[256], long_count;
    __shared__ float part[256 * VW];
    const Place at = place_of<VW>(a);
    const int teams = 256 / a.lanes, team = threadIdx.x / a.lanes, lane = threadIdx.x - team * a.lanes;
    const int64_t t = at.tile, i0 = t * a.tile, i1 = i0 + a.tile;
    if (threadIdx.x == 0) long_count = 0;
    __syncthreads();
    bool owner = at.on && i1 < a.n;
    uint32_t cur = 0;
    if (owner) {
        cur = a.pairs[i1 - 1].x;
        owner = cur < a.n_rows && a.pairs[i1].x == cur && !(i0 > 0 && a.pairs[i0 - 1].x == cur);
    }
    if (owner) {
        const int64_t far = t + 1 + kAlone * kBatch;
        if (far < a.tiles && a.pairs[far * a.tile].x == cur) {
            if (lane == 0) long_team[atomicAdd(&long_count, 1)] = team;
        } else {
            // the run's tiles are those whose first token carries its id: batches, keys and sums together
            float acc[VW];
#pragma unroll
            for (int j = 0; j < VW; ++j) acc[j] = a.tail[t * a.dim + at.col + j];
            bool more = true;
            for (int64_t q = t + 1; more && q < far; q += kBatch) {
                uint32_t key[kBatch];
                float v[kBatch][VW];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int64_t e = q + k < a.tiles ? q + k : a.tiles - 1;
                    key[k] = a.pairs[e * a.tile].x;
#pragma unroll
                    for (int j = 0; j < VW; ++j) v[k][j] = a.head[e * a.dim + at.col + j];     // unwritten behind the run's end: unused
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    more = more && q + k < a.tiles && key[k] == cur;
#pragma unroll
                    for (int j = 0; j < VW; ++j) acc[j] = more ? acc[j] + v[k][j] : acc[j];
                }
            }
            store_row<G, T, VW>(a, cur, at.col, acc);
        }
    }
    __syncthreads();
    // long runs, by the whole block: thread (team, lane) takes a slice of the owner's heads at the owner's columns
    const int count = long_count;
    for (int q = 0; q < count; ++q) {
        const int who = long_team[q];
        const int64_t wat = (int64_t)blockIdx.x * teams + who, wt = a.chunks == 1 ? wat : wat / a.chunks;
        const int vector = (int)((wat - wt * a.chunks) * a.lanes + lane), col = column<VW>(vector, a.dim);
        const uint32_t key = a.pairs[wt * a.tile + a.tile - 1].x;
        // tiles of the run behind the first: the last one whose first token carries the id, 256 probes a round
        int64_t lo = wt + 1, hi = a.tiles;                     // lo is one of them; hi is not
        while (hi - lo > 1) {
            const int64_t step = (hi - lo + 255) / 256, probe = lo + threadIdx.x * step;
            const int in = __syncthreads_count(probe < hi && a.pairs[probe * a.tile].x == key);
            const int64_t next = lo + in * step;
            lo = lo + (in - 1) * step;
            hi = next < hi ? next : hi;
        }
        float acc[VW];
#pragma unroll
        for (int j = 0; j < VW; ++j) acc[j] = 0.0f;
        const int64_t heads = lo - wt, slice = (heads + teams - 1) / teams, s0 = wt + 1 + team * slice;
        const int64_t s1 = s0 + slice < lo + 1 ? s0 + slice : lo + 1;
        if (team < teams && vector * VW < a.dim && s0 < s1) add_heads<VW>(a, s0, s1, col, acc);
#pragma unroll
        for (int j = 0; j < VW; ++j) part[threadIdx.x * VW + j] = acc[j];
        __syncthreads();
        if (team == 0 && vector * VW < a.dim) {
            float sum[VW];
#pragma unroll
            for (int j = 0; j < VW; ++j) sum[j] = a.tail[wt * a.dim + col + j];
            for (int w = 0; w < teams; ++w)
#pragma unroll
                for (int j = 0; j < VW; ++j) sum[j] += part[(w * a.lanes + lane) * VW + j];
            store_row<G, T, VW>(a, key, col, sum);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------------- few tokens
// No sort, no workspace: a block takes a row (and up to 256 vectors of its columns), lists the tokens that name it, in order,
// in LDS, and adds their rows of g: teams of threads take every teams-th listed token, their sums are added in order.
// BY_TOKEN: the rows are those that the tokens name, each seen to by its first token's block (the zeros are there already);
// otherwise all rows of the table, in one launch.
// Every block reads all ids, and one block may have to read all of g: for small sizes only (few_tokens below).
constexpr int kScanIds = 16;                           // ids of a thread per round
constexpr int kScanRound = 256 * kScanIds;

__global__ void __launch_bounds__(1024) zero_kernel(char *grad, int64_t bytes) { fill_zero(grad, bytes, blockIdx.x); }

template <typename G, typename T, int VW, typename I, bool BY_TOKEN>
__global__ void __launch_bounds__(256) sum_rows_kernel(const SumArgs a, const I *__restrict__ ids, int64_t padding) {
    __shared__ uint16_t list[kScanRound];
    __shared__ uint32_t waves[4];
    __shared__ float part[256 * VW];
    const int teams = 256 / a.lanes, team = threadIdx.x / a.lanes, lane = threadIdx.x - team * a.lanes;
    const int which = blockIdx.x / a.chunks, vector = (int)(blockIdx.x - which * a.chunks) * a.lanes + lane, col = column<VW>(vector, a.dim);
    const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63, n = (int)a.n;
    const int64_t row = BY_TOKEN ? (int64_t)ids[which] : which;
    if (BY_TOKEN && ((uint64_t)row >= (uint64_t)a.n_rows || row == padding)) return;
    const bool works = team < teams && vector * VW < a.dim;
    const G *g = (const G *)a.g + (works ? col : 0);
    float acc[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) acc[j] = 0.0f;
    for (int i0 = 0; i0 < n && row != padding; i0 += kScanRound) {
        // wave w lists its quarter of the round: ids wl, wl + 64, ... of it
        const int first = i0 + wave * (kScanRound / 4) + wl;
        uint64_t hits[kScanIds];
        uint32_t count = 0;
        I id[kScanIds];
#pragma unroll
        for (int k = 0; k < kScanIds; ++k) id[k] = ids[first + k * 64 < n ? first + k * 64 : n - 1];
#pragma unroll
        for (int k = 0; k < kScanIds; ++k) {
            hits[k] = __ballot(id[k] == (I)row && first + k * 64 < n);
            count += __popcll(hits[k]);
        }
        if (wl == 0) waves[wave] = count;
        __syncthreads();
        uint32_t at = 0, total = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w == wave) at = total;
            total += waves[w];
        }
#pragma unroll
        for (int k = 0; k < kScanIds; ++k) {
            if ((hits[k] >> wl) & 1) list[at + lanes_below(hits[k])] = (uint16_t)(first + k * 64 - i0);
            at += __popcll(hits[k]);
        }
        __syncthreads();
        if (BY_TOKEN && i0 == 0 && list[0] != which) return;           // an earlier token sees to the row
        if (works)
            for (uint32_t q = team; q < total; q += kBatch * teams) {
                Pack<G, VW> v[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const uint32_t e = q + k * teams < total ? q + k * teams : q;
                    v[k] = *reinterpret_cast<const Pack<G, VW> *>(g + (int64_t)(i0 + list[e]) * a.g_stride);
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
#pragma unroll
                    for (int j = 0; j < VW; ++j) acc[j] += q + k * teams < total ? to_f32(v[k].e[j]) : 0.0f;
            }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < VW; ++j) part[threadIdx.x * VW + j] = acc[j];
    __syncthreads();
    if (team == 0 && works) {
        for (int w = 1; w < teams; ++w)
#pragma unroll
            for (int j = 0; j < VW; ++j) acc[j] += part[(w * a.lanes + lane) * VW + j];
        store_row<G, T, VW>(a, (uint32_t)row, col, acc);
    }
}

// ---------------------------------------------------------------------------------------------------- up to 16384 tokens: ranges
// One launch, no workspace: a block for each CU takes 2^low table rows and up to 64 vectors of their columns.  It reads all ids and
// lists its own tokens in order (ballots), ranks them by row in LDS, and writes the sums of its rows, zeros included.  Rows of up to
// kLight tokens are a team's (several to a wave), up to kWaveTokens times a wave's teams a wave's, others the block's; the teams' sums
// are added by halves, the waves' in order.  Its rows lie in groups of 64 bytes or more, 2^bits groups apart: neighbouring rows are
// often met alike (frequent ids first), and 16384 such tokens x 4 bf16 over 74009 rows take 40.5 us in one range, 23.4 in groups of 256
// bytes and 16.5 in groups of 64.  4096 x 10 bf16 over 12011 rows: 8.2 us a call (sorted 22); 16384 x 64 over 8000: 11.2 (24).
constexpr int kLight = 16;
constexpr int kWaveTokens = 64;
constexpr int kMaxLow = 10;
struct Ranges {                // a row is high bits, block (`bits`), place in a group (`group`); its number in the block: first and last
    int bits, group, low;
    __device__ __forceinline__ uint32_t block_of(uint32_t row) const { return (row >> group) & ((1u << bits) - 1); }
    __device__ __forceinline__ uint32_t own_of(uint32_t row) const { return row >> (bits + group) << group | (row & ((1u << group) - 1)); }
    __device__ __forceinline__ uint32_t row_of(uint32_t block, uint32_t own) const {
        return (own >> group << bits | block) << group | (own & ((1u << group) - 1));
    }
};

template <typename G, typename T, int VW, int ITEMS>
__global__ void __launch_bounds__(1024, ITEMS > kTileItems ? 4 : 8) sum_ranges_kernel(const SumArgs a, const void *__restrict__ ids,
                                                                                        int wide, int64_t padding, const Ranges w) {
    __shared__ uint32_t list[1024 * ITEMS];                // row in the range << 14 | position; then positions by row
    __shared__ union {
        uint16_t cnt[16][1 << kMaxLow];
        float part[16][64 * VW];
    } u;
    __shared__ uint16_t start[(1 << kMaxLow) + 1], heavy[1 << kMaxLow];
    __shared__ uint32_t sums[16], heavy_count;
    uint16_t *sorted = reinterpret_cast<uint16_t *>(list);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = (int)a.n;
    const uint32_t range = blockIdx.x / a.chunks, rows = 1u << w.low;
    const int teams = 64 / a.lanes, of_wave = lane / a.lanes, team = wave * teams + of_wave;           // teams of a wave
    const int in_team = lane - of_wave * a.lanes, vector = (int)(blockIdx.x - range * a.chunks) * a.lanes + in_team;
    const int col = column<VW>(vector, a.dim);
    const bool works = of_wave < teams && vector * VW < a.dim;
    const G *g = (const G *)a.g + (works ? col : 0);
    // the tokens of the range, in order (items in order: wave, item, lane)
    const int items = (n + 1023) / 1024, per = items * 64;
    uint32_t key[ITEMS], m = 0;
    uint64_t hits[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (k < items) {
            const int i = wave * per + k * 64 + lane, at = i < n ? i : n - 1;
            const uint32_t v = key_of(wide ? ((const int64_t *)ids)[at] : (int64_t)((const int32_t *)ids)[at], a.n_rows, padding);
            key[k] = i < n ? v : a.n_rows;
        }
    if (tid == 0) heavy_count = 0;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (k < items) {
            hits[k] = __ballot(key[k] < a.n_rows && w.block_of(key[k]) == range);
            m += __popcll(hits[k]);
        }
    if (lane == 0) sums[wave] = m;
    __syncthreads();
    uint32_t at = 0;
    m = 0;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        if (v == wave) at = m;
        m += sums[v];
    }
    if (m == 0) {                                          // no token: the zeros
        Pack<T, VW> zero;
#pragma unroll
        for (int j = 0; j < VW; ++j) zero.e[j] = from_f32<T>(0.0f);
        if (works)
            for (uint32_t r = team; r < rows; r += 16 * teams) {
                const uint32_t row = w.row_of(range, r);
                if (row < a.n_rows) *reinterpret_cast<Pack<T, VW> *>((T *)a.grad + (int64_t)row * a.dim + col) = zero;
            }
        return;
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (k < items) {
            if ((hits[k] >> lane) & 1) list[at + lanes_below(hits[k])] = w.own_of(key[k]) << 14 | (wave * per + k * 64 + lane);
            at += __popcll(hits[k]);
        }
    for (uint32_t b = lane; b < (rows + 1) / 2; b += 64) reinterpret_cast<uint32_t *>(u.cnt[wave])[b] = 0;
    __syncthreads();
    // stable, by row
    const int mine = (m + 1023) / 1024;
    uint32_t entry[ITEMS], rank[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (k < mine) {
            const uint32_t e = wave * (mine * 64) + k * 64 + lane;
            const bool on = e < m;
            entry[k] = list[on ? e : 0];
            rank[k] = wave_rank(u.cnt[wave], on ? entry[k] >> 14 : 0, w.low, on);
        }
    __syncthreads();
    uint32_t total = 0;
    if (tid < (int)rows)
        for (int v = 0; v < 16; ++v) {
            const uint32_t c = u.cnt[v][tid];
            u.cnt[v][tid] = (uint16_t)total;
            total += c;
        }
    const uint32_t first = block_scan<16>(total, sums);
    if (tid < (int)rows) start[tid] = (uint16_t)first;
    if (tid == 0) start[rows] = (uint16_t)m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (k < mine && wave * (mine * 64) + k * 64 + lane < m)
            sorted[start[entry[k] >> 14] + u.cnt[wave][entry[k] >> 14] + rank[k]] = (uint16_t)(entry[k] & 0x3fff);
    __syncthreads();
    const auto load = [&](uint32_t q) { return *reinterpret_cast<const Pack<G, VW> *>(g + (int64_t)sorted[q] * a.g_stride); };
    // acc += the tokens q, q + step ... below hi
    const auto add = [&](float *acc, uint32_t q0, uint32_t hi, uint32_t step) {
        for (uint32_t q = q0; q < hi; q += kBatch * step) {
            Pack<G, VW> v[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) v[k] = load(q + k * step < hi ? q + k * step : q);
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
#pragma unroll
                for (int j = 0; j < VW; ++j) acc[j] += q + k * step < hi ? to_f32(v[k].e[j]) : 0.0f;
        }
    };
    if (works)
        for (uint32_t r0 = team; r0 < rows; r0 += 4 * 16 * teams) {         // four rows' first tokens in flight
            Pack<G, VW> v[4];
            uint32_t lo[4], c[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t r = r0 + k * 16 * teams < rows ? r0 + k * 16 * teams : r0;
                lo[k] = start[r], c[k] = start[r + 1] - lo[k];
            }
            if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = load(c[k] ? lo[k] : 0);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t r = r0 + k * 16 * teams, row = w.row_of(range, r);
                if (r >= rows || row >= a.n_rows) break;
                if (c[k] > kLight) {
                    if (in_team == 0) heavy[atomicAdd(&heavy_count, 1u)] = (uint16_t)r;
                    continue;
                }
                float acc[VW];
#pragma unroll
                for (int j = 0; j < VW; ++j) acc[j] = c[k] ? to_f32(v[k].e[j]) : 0.0f;
                if (c[k] > 1) add(acc, lo[k] + 1, lo[k] + c[k], 1);
                store_row<G, T, VW>(a, row, col, acc);
            }
        }
    __syncthreads();
    const auto add_teams = [&](float *acc) {               // the wave's sums, in its first team
        for (int t = teams; t > 1;) {
            const int half = (t + 1) / 2;
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float other = __shfl(acc[j], (lane + half * a.lanes) & 63);
                acc[j] += of_wave + half < t ? other : 0.0f;
            }
            t = half;
        }
    };
    const uint32_t heavies = heavy_count;
    for (uint32_t h = wave; h < heavies; h += 16) {
        const int r = heavy[h];
        const uint32_t lo = start[r], hi = start[r + 1];
        if ((int)(hi - lo) > kWaveTokens * teams) continue;
        float acc[VW] = {};
        if (works) add(acc, lo + of_wave, hi, teams);
        add_teams(acc);
        if (works && of_wave == 0) store_row<G, T, VW>(a, w.row_of(range, r), col, acc);
    }
    for (uint32_t h = 0; h < heavies; ++h) {
        const int r = heavy[h];
        const uint32_t lo = start[r], hi = start[r + 1];
        if ((int)(hi - lo) <= kWaveTokens * teams) continue;
        float acc[VW] = {};
        if (works) add(acc, lo + team, hi, 16 * teams);
        add_teams(acc);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VW; ++j) u.part[wave][lane * VW + j] = acc[j];
        __syncthreads();
        if (works && team == 0) {
            for (int v = 1; v < 16; ++v)
#pragma unroll
                for (int j = 0; j < VW; ++j) acc[j] += u.part[v][lane * VW + j];
            store_row<G, T, VW>(a, w.row_of(range, r), col, acc);
        }
    }
}

// ---------------------------------------------------------------------------------------------------- narrow rows
// Rows of g of up to 8 elements, more than a tile of tokens.  Gathering such rows by position fetches a cache line for each (44 us of
// 111 for 2^21 rows of two f32), and a second digit moves all pairs once more: here the rows travel with their ids through ONE
// pass, by the ids' high bits, into at most 1024 buckets of 2^low neighbouring table rows.  A block then takes up to `chunk` tokens
// of a bucket, ranks them by their low bits (stable), lays their rows out in that order in LDS, and a thread adds each element of the
// bucket's table rows, zeros included.  Buckets of more than a chunk leave their sums per chunk, added in order by a last launch.
// 2^21 rows of two f32 into 524288: 64 us (5 count, 7 scan, 31 scatter, 22 sums, 5 join) against 112 by sorted pairs.
struct NarrowArgs {
    const void *g;
    int64_t g_stride, n;
    void *grad;
    uint32_t *keys;            // [n] by bucket
    void *rows;                // [n][dim] in g's type, by bucket
    uint32_t *counts;          // [tiles][bins]
    uint32_t *totals;          // [bins]; behind them, where the bucket's tokens begin [bins], and the number of further chunks
    float *partial;            // [blocks][dim << low]: chunks of buckets that have more than one
    uint32_t n_rows;
    int dim, low, bins, chunk, tiles, blocks;
    float scale;
};
constexpr int kHeavy = 64;     // tokens of a table row beyond which a wave adds them

template <typename I, int ITEMS>
__global__ void __launch_bounds__(1024) narrow_count_kernel(const I *__restrict__ ids, int64_t padding, const NarrowArgs a) {
    __shared__ uint32_t cnt[1 << kMaxDigit];
    if ((int)threadIdx.x < a.bins) cnt[threadIdx.x] = 0;
    const int64_t i0 = (int64_t)blockIdx.x * (1024 * ITEMS) + threadIdx.x;
    uint32_t key[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) key[k] = key_of(ids[i0 + k * 1024 < a.n ? i0 + k * 1024 : a.n - 1], a.n_rows, padding);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (i0 + k * 1024 < a.n && key[k] < a.n_rows) atomicAdd(&cnt[key[k] >> a.low], 1u);
    __syncthreads();
    if ((int)threadIdx.x < a.bins) a.counts[(int64_t)blockIdx.x * a.bins + threadIdx.x] = cnt[threadIdx.x];
}

// U: unit that rows are moved in (their size and all addresses are multiples of it), `units` of them a row
template <typename I, int ITEMS, typename U>
__global__ void __launch_bounds__(1024) narrow_scatter_kernel(const I *__restrict__ ids, int64_t padding, const NarrowArgs a, int units,
                                                              int64_t unit_stride) {
    __shared__ uint32_t base[1 << kMaxDigit];
    __shared__ uint16_t cnt[16][1 << kMaxDigit], start[1 << kMaxDigit];
    __shared__ uint32_t key_of_place[1024 * ITEMS];
    __shared__ uint16_t item_of_place[1024 * ITEMS];
    __shared__ uint32_t sums[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = a.bins;
    const int64_t tile0 = (int64_t)blockIdx.x * (1024 * ITEMS);
    const int first_item = wave * (64 * ITEMS) + lane;
    uint32_t key[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = tile0 + first_item + k * 64;
        key[k] = i < a.n ? key_of(ids[i], a.n_rows, padding) : a.n_rows;
    }
    uint32_t total = 0, before = 0;
    if (tid < bins) {
        if (a.tiles <= kFewTiles) {                        // no scan launch: the blocks before, and all of them
#pragma unroll 8
            for (int t = 0; t < a.tiles; ++t) {
                const uint32_t c = a.counts[t * bins + tid];
                total += c;
                before += t < (int)blockIdx.x ? c : 0;
            }
        } else {
            total = a.totals[tid], before = a.counts[(int64_t)blockIdx.x * bins + tid];
        }
    }
    int bits = 1;
    while ((bins - 1) >> bits) ++bits;
    for (int b = tid; b < 16 << bits; b += 1024) cnt[b >> bits][b & ((1 << bits) - 1)] = 0;
    const uint32_t first = block_scan<16>(total, sums);
    if (blockIdx.x == 0) {                                 // for the launches behind this one
        const uint32_t further = total > (uint32_t)a.chunk ? (total - 1) / a.chunk : 0;
        const uint32_t f = block_scan<16>(further, sums);
        if (tid < bins) a.totals[tid] = total, a.totals[bins + tid] = first;
        if (tid == bins - 1) a.totals[2 * bins] = f + further;
    }
    uint32_t rank[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const bool on = key[k] < a.n_rows;
        rank[k] = wave_rank(cnt[wave], on ? key[k] >> a.low : 0, bits, on);
    }
    __syncthreads();
    uint32_t mine = 0;
    if (tid < bins) {
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const uint32_t c = cnt[w][tid];
            cnt[w][tid] = (uint16_t)mine;
            mine += c;
        }
    }
    const uint32_t local = block_scan<16>(mine, sums);
    if (tid < bins) {
        start[tid] = (uint16_t)local;
        base[tid] = first + before - local;
    }
    if (tid == bins - 1) sums[0] = local + mine;           // items of this block that take part
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (key[k] < a.n_rows) {
            const uint32_t d = key[k] >> a.low, place = start[d] + cnt[wave][d] + rank[k];
            key_of_place[place] = key[k];
            item_of_place[place] = (uint16_t)(first_item + k * 64);
        }
    __syncthreads();
    const int count = (int)sums[0];
    for (int q = tid; q < count; q += 1024) {
        const uint32_t k = key_of_place[q];
        const int64_t to = (int64_t)(base[k >> a.low] + q);
        a.keys[to] = k;
        const U *from = (const U *)a.g + (tile0 + item_of_place[q]) * unit_stride;
        U *row = (U *)a.rows + to * units;
        for (int w = 0; w < units; ++w) row[w] = from[w];
    }
}

// Which chunk of which bucket a block works on: block b < bins the first chunk of bucket b, the blocks behind them the further ones.
struct Piece {
    int bucket, chunks;
    int64_t begin;
    int count;
};

// Further chunks of the buckets before bucket `tid` (all threads call)
__device__ __forceinline__ uint32_t further_before(const NarrowArgs &a, uint32_t *own, uint32_t *sums) {
    const uint32_t total = (int)threadIdx.x < a.bins ? a.totals[threadIdx.x] : 0;
    *own = total > (uint32_t)a.chunk ? (total - 1) / a.chunk : 0;
    return block_scan<16>(*own, sums);
}

__device__ __forceinline__ Piece piece_of(const NarrowArgs &a, int block, uint32_t *sums, int *found) {
    Piece p;
    int chunk = 0;
    p.bucket = block;
    if (block >= a.bins) {
        const uint32_t x = block - a.bins;
        p.bucket = -1;
        if (x >= a.totals[2 * a.bins]) return p;
        uint32_t own;
        const uint32_t before = further_before(a, &own, sums);
        if (x - before < own) found[0] = threadIdx.x, found[1] = (int)(x - before) + 1;
        __syncthreads();
        p.bucket = found[0], chunk = found[1];
    }
    const uint32_t total = a.totals[p.bucket];
    p.begin = (int64_t)a.totals[a.bins + p.bucket] + (int64_t)chunk * a.chunk;
    p.chunks = total > (uint32_t)a.chunk ? (int)((total - 1) / a.chunk) + 1 : 1;
    const int64_t left = (int64_t)total - (int64_t)chunk * a.chunk;
    p.count = (int)(left < a.chunk ? left : a.chunk);
    return p;
}

// C: columns rounded up to a power of two; LDS holds chunk * dim <= 8192 values
template <typename G, typename T, int C>
__global__ void __launch_bounds__(1024) narrow_sum_kernel(const NarrowArgs a) {
    __shared__ float row_lds[8192];
    __shared__ uint16_t cnt[16][1 << kMaxDigit];
    __shared__ uint32_t start[(1 << kMaxDigit) + 1];
    __shared__ uint32_t sums[16], heavy_count;
    __shared__ uint16_t heavy[8192 / kHeavy];
    __shared__ int found[2];
    constexpr int kPer = 4;                                // chunk <= 4096
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Piece p = piece_of(a, blockIdx.x, sums, found);
    if (p.bucket < 0) return;
    const int per_bucket = 1 << a.low, dim = a.dim;
    const int64_t row0 = (int64_t)p.bucket << a.low;
    if (p.count == 0) {                                    // no token: the zeros
        const int64_t size = ((int64_t)a.n_rows - row0 < per_bucket ? (int64_t)a.n_rows - row0 : per_bucket) * dim;
        for (int64_t e = tid; e < size; e += 1024) ((T *)a.grad)[row0 * dim + e] = from_f32<T>(0.0f);
        return;
    }
    uint32_t low[kPer];
    float v[kPer][C];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = wave * (64 * kPer) + k * 64 + lane;
        const int64_t at = p.begin + (i < p.count ? i : 0);
        low[k] = a.keys[at] & (per_bucket - 1);
#pragma unroll
        for (int c = 0; c < C; ++c) v[k][c] = c < dim ? to_f32(((const G *)a.rows)[at * dim + c]) : 0.0f;
    }
    if (tid == 0) heavy_count = 0;
    for (int b = tid; b < 16 << a.low; b += 1024) cnt[b >> a.low][b & (per_bucket - 1)] = 0;
    __syncthreads();
    uint32_t rank[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const bool on = wave * (64 * kPer) + k * 64 + lane < p.count;
        rank[k] = wave_rank(cnt[wave], on ? low[k] : 0, a.low, on);
    }
    __syncthreads();
    uint32_t mine = 0;
    if (tid < per_bucket) {
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const uint32_t c = cnt[w][tid];
            cnt[w][tid] = (uint16_t)mine;
            mine += c;
        }
    }
    const uint32_t first = block_scan<16>(mine, sums);
    if (tid < per_bucket) start[tid] = first;
    if (tid == 0) start[per_bucket] = p.count;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k)
        if (wave * (64 * kPer) + k * 64 + lane < p.count) {
            const uint32_t place = start[low[k]] + cnt[wave][low[k]] + rank[k];
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (c < dim) row_lds[place * dim + c] = v[k][c];
        }
    __syncthreads();
    const auto store = [&](int r, int c, float sum) {
        if (p.chunks == 1) ((T *)a.grad)[(row0 + r) * dim + c] = from_f32<T>(sum * a.scale);
        else a.partial[(int64_t)blockIdx.x * (dim << a.low) + r * dim + c] = sum;
    };
    for (int e = tid; e < per_bucket * C; e += 1024) {
        const int r = e / C, c = e % C;
        if (c >= dim || row0 + r >= (int64_t)a.n_rows) continue;
        const uint32_t lo = start[r], hi = start[r + 1];
        if (hi - lo > kHeavy) {
            if (c == 0) heavy[atomicAdd(&heavy_count, 1u)] = (uint16_t)r;
            continue;
        }
        float sum = 0.0f;
#pragma unroll 8
        for (uint32_t q = lo; q < hi; ++q) sum += row_lds[q * dim + c];
        store(r, c, sum);
    }
    __syncthreads();
    // rows of many tokens: a wave each, its lanes a slice of the tokens and a column, the slices added by halves
    constexpr int kSlices = 64 / C;
    for (uint32_t h = wave; h < heavy_count; h += 16) {
        const int r = heavy[h], c = lane % C;
        const uint32_t lo = start[r], hi = start[r + 1], each = (hi - lo + kSlices - 1) / kSlices, q0 = lo + lane / C * each;
        const uint32_t q1 = q0 + each < hi ? q0 + each : hi;
        float sum = 0.0f;
        if (c < dim) {
#pragma unroll 8
            for (uint32_t q = q0; q < q1; ++q) sum += row_lds[q * dim + c];
        }
#pragma unroll
        for (int d = 32; d >= C; d >>= 1) sum += __shfl_xor(sum, d);
        if (lane < dim) store(r, lane, sum);
    }
}

// Buckets of several chunks, a block each: four threads an element, each a quarter of the chunks.
template <typename T>
__global__ void __launch_bounds__(1024) narrow_join_kernel(const NarrowArgs a) {
    __shared__ uint32_t sums[16];
    __shared__ int found;
    __shared__ float part[4][256];
    const int tid = threadIdx.x, bucket = blockIdx.x;
    const uint32_t own = a.totals[bucket];
    if (own <= (uint32_t)a.chunk) return;
    uint32_t further;
    const uint32_t before = further_before(a, &further, sums);
    if (tid == bucket) found = (int)before;
    __syncthreads();
    const int n = (int)((own + a.chunk - 1) / a.chunk), size = a.dim << a.low, quarter = tid >> 8;
    const int each = (n + 3) / 4, c0 = quarter * each, c1 = c0 + each < n ? c0 + each : n;
    for (int e0 = 0; e0 < size; e0 += 256) {
        const int e = e0 + (tid & 255);
        float sum = 0.0f;
        if (e < size) {
            // chunk 0 lies at the bucket's own block, the further ones behind all buckets
            const float *p = a.partial + ((int64_t)a.bins + found - 1) * size + e;
#pragma unroll 8
            for (int c = c0; c < c1; ++c) sum += c == 0 ? a.partial[(int64_t)bucket * size + e] : p[(int64_t)c * size];
        }
        part[quarter][tid & 255] = sum;
        __syncthreads();
        const int64_t at = (((int64_t)bucket << a.low) * a.dim) + e;
        if (quarter == 0 && e < size && at < (int64_t)a.n_rows * a.dim)
            ((T *)a.grad)[at] = from_f32<T>((((part[0][tid] + part[1][tid]) + part[2][tid]) + part[3][tid]) * a.scale);
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------------- host
struct BwdPlan {
    int passes, digit;         // of the sort
    int64_t sort_tiles;        // blocks of the many-block sort (0: one block)
    int sort_items;            // items of a thread in it
    int tile;                  // tokens of a sum tile
    int64_t sum_tiles;
    int low, bins, chunk, blocks;      // narrow rows: bits of a bucket, buckets, tokens of a block, blocks; bins 0: the other way
    int64_t off_a, off_b, off_counts, off_totals, off_head, off_tail, bytes;       // all zero: few tokens, no workspace
};

// Few rows, few tokens: without a sort (one or two launches against three or more).  The ids are read once a row or token, and a block may
// meet all of g: each of its teams then 256 tokens at most, about 20 us.
// Measured, us a call, against the sorted way: 4096 tokens x 32 over 100 rows 8.3 / 16.8, all on one row 10.1 / 17.4; 16384 x 8 over
// 256 rows 11.7 / 26.7; 64 x 1024 over 1024 rows 8.6 / 15.4.
enum Few { kNotFew, kFewRows, kFewTokens };
Few few_tokens(int64_t n, int64_t n_rows, int dim) {
    const int vw = dim >= 4 ? 4 : dim >= 2 ? 2 : 1, vectors = (dim + vw - 1) / vw, lanes = vectors < 256 ? vectors : 256;
    const int chunks = (vectors + 255) / 256;
    if (n > 256 * (256 / lanes)) return kNotFew;
    if (n_rows * chunks <= 4096 && n_rows * n <= 1 << 22) return kFewRows;
    return n <= 4096 ? kFewTokens : kNotFew;
}

// Ranges (what few rows leave): not for large gradients, whose zeros a launch of their own writes faster than blocks that wait for ids, nor
// where many blocks would read many ids.  Us a call by ranges / otherwise, for one token; 4096; 16384 (f32):
//   9298 rows x 544: 9.8 / 10.5, 16.3 / 24.3    50000 x 263: 15.0 / 13.0, 18.3 / 25.4, 43.3 / 35.3    100000 x 263: 23.4 / 18.9, 27.7 / 26.6,
//   61.3 / 42.3    1500000 x 10: 20.8 / 15.0, 42.0 / 25.3, 108 / 38.8    2^19 x 10: 16384 tokens 30.9 / 31.1
// The bound on the gradient's size is on the safe side: 4096 tokens x 263 over 27442 rows, just above it, take 14.8 by ranges, 24.4 otherwise.
bool in_ranges(int64_t n, int64_t n_rows, int dim) {
    return n <= kSmall && n_rows * dim <= 6 << 20 && n_rows * n <= (int64_t)1 << 33;
}

BwdPlan plan_bwd(int64_t n, int64_t n_rows, int dim) {
    BwdPlan p{};
    if (few_tokens(n, n_rows, dim) != kNotFew || in_ranges(n, n_rows, dim)) return p;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    if (dim <= 8 && n_rows > 0 && n_rows <= 1 << 20 && n > kTile) {
        // buckets no more than the digit has, and wide enough to keep half a block's threads in the sums
        while ((n_rows - 1) >> p.low >= 1 << kMaxDigit || (dim << p.low < 512 && 1 << p.low < n_rows)) ++p.low;
        p.bins = (int)(((n_rows - 1) >> p.low) + 1);
        p.chunk = 4096;
        while (p.chunk * dim > 8192) p.chunk >>= 1;
        p.blocks = p.bins + (int)(n / p.chunk);            // a first chunk each, and at most so many further ones
        p.sort_items = n <= (int64_t)kFewTiles * 1024 * kFewItems ? kFewItems : kTileItems;
        p.sort_tiles = (n + 1024 * p.sort_items - 1) / (1024 * p.sort_items);
        p.off_a = take(n * 4);
        p.off_b = take(n * dim * 4);
        p.off_counts = take(p.sort_tiles * p.bins * 4);
        p.off_totals = take((2 * p.bins + 1) * 4);
        p.off_head = take((int64_t)p.blocks * (dim << p.low) * 4);
        p.bytes = at;
        return p;
    }
    int bits = 1;
    while (bits < 32 && (n_rows >> bits) != 0) ++bits;     // keys go up to n_rows itself
    p.passes = (bits + kMaxDigit - 1) / kMaxDigit;
    p.digit = (bits + p.passes - 1) / p.passes;
    // one block sorts a tile's worth, and more while the zeros of a large gradient hide it (65 us for 16384 tokens)
    const bool one_block = n <= kTile || (n <= kSmall && n_rows * dim >= 1 << 28);
    p.sort_items = n <= (int64_t)kFewTiles * 1024 * kFewItems ? kFewItems : kTileItems;
    p.sort_tiles = one_block ? 0 : (n + 1024 * p.sort_items - 1) / (1024 * p.sort_items);
    // enough teams to fill the chip (8 waves on each of 256 CUs), yet tiles long enough that few runs cross them
    p.tile = 64;
    const int64_t vectors = (dim + 3) / 4;
    while (p.tile > kBatch && n * vectors / p.tile < 256 * 8 * 64) p.tile >>= 1;
    p.sum_tiles = (n + p.tile - 1) / p.tile;
    p.off_a = take(n * 8);
    p.off_b = p.passes > 1 && p.sort_tiles ? take(n * 8) : 0;
    p.off_counts = take(p.sort_tiles * (4 << p.digit));
    p.off_totals = take(p.sort_tiles ? (4 << p.digit) : 0);
    p.off_head = take(p.sum_tiles * dim * 4);
    p.off_tail = take(p.sum_tiles * dim * 4);
    p.bytes = at;
    return p;
}

template <typename I, int ITEMS>
const uint2 *sort_many(const BwdPlan &p, const I *ids, int64_t n, int64_t n_rows, int64_t padding, char *ws, void *grad,
                       int64_t grad_bytes, hipStream_t s) {
    const int fill = (int)((grad_bytes + kFill - 1) / kFill);
    uint2 *a = (uint2 *)(ws + p.off_a), *b = (uint2 *)(ws + p.off_b);
    uint32_t *counts = (uint32_t *)(ws + p.off_counts), *totals = (uint32_t *)(ws + p.off_totals);
    const int tiles = (int)p.sort_tiles, bins = 1 << p.digit;
    const uint2 *in = nullptr;
    uint2 *out = p.passes % 2 ? a : b;                          // the last pass ends in a
    for (int d = 0; d < p.passes; ++d) {
        const int shift = d * p.digit;
        if (d == 0)
            sort_count_kernel<I, true, ITEMS><<<tiles + fill, 1024, 0, s>>>(ids, nullptr, n, (uint32_t)n_rows, padding, 0, p.digit,
                                                                            tiles, counts, grad, grad_bytes);
        else
            sort_count_kernel<I, false, ITEMS><<<tiles, 1024, 0, s>>>(ids, in, n, (uint32_t)n_rows, padding, shift, p.digit, tiles,
                                                                      counts, nullptr, 0);
        if (tiles > kFewTiles) sort_scan_kernel<<<(bins + 63) / 64, 1024, 0, s>>>(counts, totals, bins, tiles);
        if (d == 0)
            sort_scatter_kernel<I, true, ITEMS><<<tiles, 1024, 0, s>>>(ids, nullptr, n, (uint32_t)n_rows, padding, 0, p.digit, tiles,
                                                                       counts, totals, out);
        else
            sort_scatter_kernel<I, false, ITEMS><<<tiles, 1024, 0, s>>>(ids, in, n, (uint32_t)n_rows, padding, shift, p.digit, tiles,
                                                                        counts, totals, out);
        in = out;
        out = out == a ? b : a;
    }
    return in;
}

template <typename I>
const uint2 *sort_pairs(const BwdPlan &p, const I *ids, int64_t n, int64_t n_rows, int64_t padding, char *ws, void *grad,
                        int64_t grad_bytes, hipStream_t s) {
    const int fill = (int)((grad_bytes + kFill - 1) / kFill);
    uint2 *a = (uint2 *)(ws + p.off_a), *b = (uint2 *)(ws + p.off_b);
    if (p.sort_tiles == 0) {
        sort_small_kernel<I><<<1 + fill, 1024, 0, s>>>(ids, (int)n, (uint32_t)n_rows, padding, p.passes, p.digit,
                                                                       a, grad, grad_bytes);
        return a;
    }
    return p.sort_items == kFewItems ? sort_many<I, kFewItems>(p, ids, n, n_rows, padding, ws, grad, grad_bytes, s)
                                     : sort_many<I, kTileItems>(p, ids, n, n_rows, padding, ws, grad, grad_bytes, s);
}

template <typename I, int ITEMS>
void narrow_scatter(const NarrowArgs &a, const I *ids, int64_t padding, int elem, hipStream_t s) {
    narrow_count_kernel<I, ITEMS><<<a.tiles, 1024, 0, s>>>(ids, padding, a);
    if (a.tiles > kFewTiles) sort_scan_kernel<<<(a.bins + 63) / 64, 1024, 0, s>>>(a.counts, a.totals, a.bins, a.tiles);
    // the largest unit that rows and their addresses are made of
    const int bytes = a.dim * elem;
    const uint64_t all = (uint64_t)(uintptr_t)a.g | (uint64_t)a.g_stride * elem | (uint64_t)bytes;
    const int unit = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
    const int units = bytes / unit;
    const int64_t stride = a.g_stride * elem / unit;
    if (unit == 16) narrow_scatter_kernel<I, ITEMS, uint4><<<a.tiles, 1024, 0, s>>>(ids, padding, a, units, stride);
    else if (unit == 8) narrow_scatter_kernel<I, ITEMS, uint2><<<a.tiles, 1024, 0, s>>>(ids, padding, a, units, stride);
    else if (unit == 4) narrow_scatter_kernel<I, ITEMS, uint32_t><<<a.tiles, 1024, 0, s>>>(ids, padding, a, units, stride);
    else narrow_scatter_kernel<I, ITEMS, uint16_t><<<a.tiles, 1024, 0, s>>>(ids, padding, a, units, stride);
}

template <typename G, typename T>
void launch_narrow(const SumArgs &sa, const BwdPlan &p, const void *ids, bool i64, int64_t padding, char *ws, hipStream_t s) {
    NarrowArgs a;
    a.g = sa.g, a.g_stride = sa.g_stride, a.n = sa.n, a.grad = sa.grad, a.n_rows = sa.n_rows, a.dim = sa.dim, a.scale = sa.scale;
    a.keys = (uint32_t *)(ws + p.off_a), a.rows = ws + p.off_b, a.counts = (uint32_t *)(ws + p.off_counts);
    a.totals = (uint32_t *)(ws + p.off_totals), a.partial = (float *)(ws + p.off_head);
    a.low = p.low, a.bins = p.bins, a.chunk = p.chunk, a.tiles = (int)p.sort_tiles, a.blocks = p.blocks;
    const int e = (int)sizeof(G);
    if (i64) p.sort_items == kFewItems ? narrow_scatter<int64_t, kFewItems>(a, (const int64_t *)ids, padding, e, s)
                                       : narrow_scatter<int64_t, kTileItems>(a, (const int64_t *)ids, padding, e, s);
    else p.sort_items == kFewItems ? narrow_scatter<int32_t, kFewItems>(a, (const int32_t *)ids, padding, e, s)
                                   : narrow_scatter<int32_t, kTileItems>(a, (const int32_t *)ids, padding, e, s);
    if (a.dim == 1) narrow_sum_kernel<G, T, 1><<<a.blocks, 1024, 0, s>>>(a);
    else if (a.dim == 2) narrow_sum_kernel<G, T, 2><<<a.blocks, 1024, 0, s>>>(a);
    else if (a.dim <= 4) narrow_sum_kernel<G, T, 4><<<a.blocks, 1024, 0, s>>>(a);
    else narrow_sum_kernel<G, T, 8><<<a.blocks, 1024, 0, s>>>(a);
    narrow_join_kernel<T><<<a.bins, 1024, 0, s>>>(a);
}

// A block for each of 256 CUs: as many ranges of rows as give that, then columns in pieces, which share a row of many tokens
template <typename G, typename T, int VW>
void launch_ranges(SumArgs a, const void *ids, bool i64, int64_t padding, hipStream_t s) {
    const int vectors = (a.dim + VW - 1) / VW;
    int most = 64, total = 0;                              // vectors: 4 MB of f32 in a block, should all tokens be its own
    while (most > 1 && (int64_t)most * VW * a.n > 1 << 20) most /= 2;
    while ((int64_t)1 << total < a.n_rows) ++total;
    a.chunks = (vectors + most - 1) / most;
    Ranges w{};
    while (w.bits < total && (2 << w.bits) * a.chunks <= 256) ++w.bits;
    const int pieces = a.dim * (int)sizeof(G) / 32;        // of 32 bytes or more
    const int split = pieces < 256 >> w.bits ? pieces : 256 >> w.bits;
    if (w.bits == total && split > a.chunks) a.chunks = split;
    while (total - w.bits > kMaxLow) ++w.bits;
    w.low = total - w.bits;
    while (w.group < w.low && a.dim * (int)sizeof(T) << w.group < 64) ++w.group;
    a.lanes = (vectors + a.chunks - 1) / a.chunks;
    const unsigned blocks = (1u << w.bits) * a.chunks;
    if (a.n <= kTile) sum_ranges_kernel<G, T, VW, kTileItems><<<blocks, 1024, 0, s>>>(a, ids, i64, padding, w);
    else sum_ranges_kernel<G, T, VW, kItems><<<blocks, 1024, 0, s>>>(a, ids, i64, padding, w);
}

template <typename G, typename T, int VW>
void launch_sums(SumArgs a, const BwdPlan &p, const void *ids, bool i64, int64_t padding, hipStream_t s) {
    const int vectors = (a.dim + VW - 1) / VW;
    a.chunks = (vectors + 255) / 256, a.lanes = (vectors + a.chunks - 1) / a.chunks, a.tiles = p.sum_tiles;
    if (p.bytes == 0) {
        if (few_tokens(a.n, a.n_rows, a.dim) == kFewRows) {
            const unsigned blocks = a.n_rows * a.chunks;
            if (i64) sum_rows_kernel<G, T, VW, int64_t, false><<<blocks, 256, 0, s>>>(a, (const int64_t *)ids, padding);
            else sum_rows_kernel<G, T, VW, int32_t, false><<<blocks, 256, 0, s>>>(a, (const int32_t *)ids, padding);
            return;
        }
        if (in_ranges(a.n, a.n_rows, a.dim)) return launch_ranges<G, T, VW>(a, ids, i64, padding, s);
        const int64_t bytes = (int64_t)a.n_rows * a.dim * (int64_t)sizeof(T);
        zero_kernel<<<(unsigned)((bytes + kFill - 1) / kFill), 1024, 0, s>>>((char *)a.grad, bytes);
        const unsigned blocks = (unsigned)a.n * a.chunks;
        if (blocks == 0) return;
        if (i64) sum_rows_kernel<G, T, VW, int64_t, true><<<blocks, 256, 0, s>>>(a, (const int64_t *)ids, padding);
        else sum_rows_kernel<G, T, VW, int32_t, true><<<blocks, 256, 0, s>>>(a, (const int32_t *)ids, padding);
        return;
    }
    const int teams = 256 / a.lanes;
    const unsigned blocks = (unsigned)((p.sum_tiles * a.chunks + teams - 1) / teams);
    sum_tiles_kernel<G, T, VW><<<blocks, 256, 0, s>>>(a);
    sum_join_kernel<G, T, VW><<<blocks, 256, 0, s>>>(a);
}

template <typename G, typename T>
void pick_sums(int vw, const SumArgs &a, const BwdPlan &p, const void *ids, bool i64, int64_t padding, char *ws, hipStream_t s) {
    if (p.bins) return launch_narrow<G, T>(a, p, ids, i64, padding, ws, s);
    if constexpr (sizeof(G) == 2 && sizeof(T) == 2)
        if (vw == 8) return launch_sums<G, T, 8>(a, p, ids, i64, padding, s);
    if (vw >= 4) return launch_sums<G, T, 4>(a, p, ids, i64, padding, s);
    if (vw == 2) return launch_sums<G, T, 2>(a, p, ids, i64, padding, s);
    launch_sums<G, T, 1>(a, p, ids, i64, padding, s);
}

// Elements of a vector: 16 bytes of f32, or of 16-bit types where that divides a row (gradient of 4096 x 420 bf16 over 4096: 8.7 us a call by 4, 14.1 by 8)
int width_of(int dim, int es_a, int es_b) {
    if (es_a == 2 && es_b == 2 && dim % 8 == 0) return 8;
    return dim >= 4 ? 4 : dim >= 2 ? 2 : 1;
}

bool pair_ok(int32_t narrow, int32_t wide) { return narrow == wide || (wide == NRF_F32 && dtype_size(narrow) == 2); }

}  // namespace

extern "C" int nrf_lookup_fwd(const void *table, int64_t table_stride, int32_t dtype, int64_t n_rows, int32_t dim,
                              const void *ids, int32_t ids_are_64, int64_t n, float scale, void *out, int32_t out_dtype,
                              void *stream) {
    NRF_REQUIRE(n >= 0 && n_rows >= 0 && dim >= 1, "nrf_lookup_fwd: n %lld, n_rows %lld, dim %d", (long long)n, (long long)n_rows, dim);
    NRF_REQUIRE(dtype_size(dtype) && dtype_size(out_dtype), "nrf_lookup_fwd: dtype %d, out_dtype %d", dtype, out_dtype);
    if (!pair_ok(dtype, out_dtype))
        return fail(NRF_ERR_UNSUPPORTED, "nrf_lookup_fwd: out must have the table's type or f32");
    if (dim > kMaxDim || n > INT32_MAX || n_rows >= INT32_MAX || (n * dim) >> 33)
        return fail(NRF_ERR_UNSUPPORTED, "nrf_lookup_fwd: dim at most %d, n and n_rows below 2^31, n * dim below 2^33", kMaxDim);
    if (n == 0) return NRF_OK;
    NRF_REQUIRE(ids && out && (table || n_rows == 0), "nrf_lookup_fwd: null pointer");
    NRF_REQUIRE(table_stride >= dim, "nrf_lookup_fwd: table_stride %lld below dim %d", (long long)table_stride, dim);
    const int vw = width_of(dim, dtype_size(dtype), dtype_size(out_dtype));
    hipStream_t s = as_stream(stream);
    const bool i64 = ids_are_64 != 0;
    if (dtype == NRF_F32) pick_fwd<float, float>(vw, table, table_stride, n_rows, ids, i64, n, dim, scale, out, s);
    else if (dtype == NRF_BF16 && out_dtype == NRF_BF16) pick_fwd<bf16_t, bf16_t>(vw, table, table_stride, n_rows, ids, i64, n, dim, scale, out, s);
    else if (dtype == NRF_BF16) pick_fwd<bf16_t, float>(vw, table, table_stride, n_rows, ids, i64, n, dim, scale, out, s);
    else if (out_dtype == NRF_F16) pick_fwd<f16_t, f16_t>(vw, table, table_stride, n_rows, ids, i64, n, dim, scale, out, s);
    else pick_fwd<f16_t, float>(vw, table, table_stride, n_rows, ids, i64, n, dim, scale, out, s);
    return check_launch("nrf_lookup_fwd");
}

static int bwd_shape(int64_t n, int64_t n_rows, int32_t dim) {
    NRF_REQUIRE(n >= 0 && n_rows >= 0 && dim >= 1, "nrf_lookup_bwd: n %lld, n_rows %lld, dim %d", (long long)n, (long long)n_rows, dim);
    if (dim > kMaxDim || n > INT32_MAX || n_rows >= INT32_MAX || (n * dim) >> 33 || (n_rows * dim) >> 33)
        return fail(NRF_ERR_UNSUPPORTED, "nrf_lookup_bwd: dim at most %d, n and n_rows below 2^31, n * dim and n_rows * dim below 2^33", kMaxDim);
    return NRF_OK;
}

extern "C" int64_t nrf_lookup_bwd_workspace_bytes(int64_t n, int64_t n_rows, int32_t dim) {
    return bwd_shape(n, n_rows, dim) == NRF_OK ? plan_bwd(n, n_rows, dim).bytes : -1;
}

extern "C" int nrf_lookup_bwd(const void *g_out, int64_t g_stride, int32_t g_dtype, const void *ids, int32_t ids_are_64, int64_t n,
                              int64_t n_rows, int32_t dim, float scale, int64_t padding_idx, void *grad, int32_t dtype,
                              void *workspace, void *stream) {
    if (int rc = bwd_shape(n, n_rows, dim)) return rc;
    NRF_REQUIRE(dtype_size(dtype) && dtype_size(g_dtype), "nrf_lookup_bwd: dtype %d, g_dtype %d", dtype, g_dtype);
    if (!pair_ok(dtype, g_dtype)) return fail(NRF_ERR_UNSUPPORTED, "nrf_lookup_bwd: g_out must have the table's type or f32");
    if (n_rows == 0) return NRF_OK;
    const BwdPlan p = plan_bwd(n, n_rows, dim);
    NRF_REQUIRE(grad && (n == 0 || (g_out && ids)) && (p.bytes == 0 || workspace), "nrf_lookup_bwd: null pointer");
    NRF_REQUIRE(n == 0 || g_stride >= dim, "nrf_lookup_bwd: g_stride %lld below dim %d", (long long)g_stride, dim);
    NRF_REQUIRE(((uintptr_t)workspace & 15) == 0, "nrf_lookup_bwd: workspace must be 16-byte aligned");
    const int64_t grad_bytes = n_rows * dim * dtype_size(dtype);
    hipStream_t s = as_stream(stream);
    const bool i64 = ids_are_64 != 0;
    char *ws = (char *)workspace;
    SumArgs a{};
    if (p.bytes && !p.bins)
        a.pairs = i64 ? sort_pairs(p, (const int64_t *)ids, n, n_rows, padding_idx, ws, grad, grad_bytes, s)
                      : sort_pairs(p, (const int32_t *)ids, n, n_rows, padding_idx, ws, grad, grad_bytes, s);
    if (p.bytes == 0 || n > 0) {
        a.g = g_out, a.g_stride = g_stride, a.grad = grad, a.head = (float *)(ws + p.off_head), a.tail = (float *)(ws + p.off_tail);
        a.n = n, a.n_rows = (uint32_t)n_rows, a.dim = dim, a.tile = p.tile, a.scale = scale;
        const int vw = width_of(dim, dtype_size(g_dtype), dtype_size(dtype));
        if (g_dtype == NRF_F32 && dtype == NRF_F32) pick_sums<float, float>(vw, a, p, ids, i64, padding_idx, ws, s);
        else if (g_dtype == NRF_F32 && dtype == NRF_BF16) pick_sums<float, bf16_t>(vw, a, p, ids, i64, padding_idx, ws, s);
        else if (g_dtype == NRF_F32) pick_sums<float, f16_t>(vw, a, p, ids, i64, padding_idx, ws, s);
        else if (g_dtype == NRF_BF16) pick_sums<bf16_t, bf16_t>(vw, a, p, ids, i64, padding_idx, ws, s);
        else pick_sums<f16_t, f16_t>(vw, a, p, ids, i64, padding_idx, ws, s);
    }
    return check_launch("nrf_lookup_bwd");
}
