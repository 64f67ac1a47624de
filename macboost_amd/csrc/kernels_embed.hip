// kernels_embed.hip — category vectors beside the forests' outputs (mbk_embed) and their
// gradient by sorted ids (mbk_embed_grad).  All of it moves data.
#include <algorithm>

#include "grid.hpp"
#include "mbk.h"
#include "ops.h"

namespace mbk {

namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

// E elements in a row, at any address that holds one.
template <typename T, int E>
using Run = T __attribute__((ext_vector_type(E), aligned(sizeof(T))));

// E elements at p as f32, of which the first n are read; the rest are 0.
template <typename T, int E>
__device__ __forceinline__ void load(const T *p, int n, float (&f)[E]) {
    if constexpr (E > 1)
        if (n >= E) {
            const Run<T, E> v = *reinterpret_cast<const Run<T, E> *>(p);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = to_f32(v[e]);
            return;
        }
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e < n ? to_f32(p[e]) : 0.0f;
}

template <typename T, int E>
__device__ __forceinline__ void store(T *p, int n, const float (&f)[E], bool streamed) {
    if constexpr (E > 1)
        if (n >= E) {
            Run<T, E> v;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = (T)f[e];
            put(p, v, streamed);
            return;
        }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e < n) p[e] = (T)f[e];
}

// ---------------------------------------------------------------------------
// The lookup: out[row] = base[row] + scale * table[ids[row]].  A row is `chunks` pieces of E
// elements; a workgroup takes 256 * LOOKUP pieces of all the rows' in their order, LOOKUP a
// thread, so that short rows leave no lane idle and each thread has LOOKUP rows on the way.
// Bound by memory: 65536 x 1024 bf16 with a base take 57 us, 380 MB at 6.7 TB/s with popular
// vectors out of the caches, and 73 in place; 64 x 37 f32 2.8, a launch and two reads one after the
// other.
// ---------------------------------------------------------------------------
constexpr int LOOKUP = 4;

template <typename T, int E>
__global__ __launch_bounds__(256) void k_embed(EmbedCall c, int32_t chunks) {
    const int64_t first = (int64_t)group_id() * (256 * LOOKUP);
    const int64_t row0 = first / chunks;
    const uint32_t rest = (uint32_t)(first - row0 * chunks);
    const T *table = static_cast<const T *>(c.table);
    const T *base = static_cast<const T *>(c.base);
    T *out = static_cast<T *>(c.out);
    // the last piece of a row is its last E columns, some of which the one before writes too, but
    // where it may have written them to the base
    const bool last_whole = E > 1 && base != out;
    int64_t row[LOOKUP];
    int col[LOOKUP];
    int32_t id[LOOKUP];
    bool here[LOOKUP];
#pragma unroll
    for (int q = 0; q < LOOKUP; ++q) {
        const uint32_t i = rest + q * 256 + threadIdx.x;
        const uint32_t r = i / (uint32_t)chunks;
        row[q] = row0 + r;
        col[q] = (int)(i - r * chunks) * E;
        if (last_whole) col[q] = min(col[q], c.dim - E);
        here[q] = row[q] < c.rows;
        id[q] = here[q] ? c.ids[row[q]] : -1;
    }
    float v[LOOKUP][E], b[LOOKUP][E];
#pragma unroll
    for (int q = 0; q < LOOKUP; ++q) {
        const bool kept = (int64_t)id[q] >= 0 && (int64_t)id[q] < c.entries;
        load<T, E>(table + (kept ? id[q] * c.table_stride : 0) + col[q],
                   kept ? c.dim - col[q] : 0, v[q]);
        load<T, E>(base + (here[q] && base ? row[q] * c.row_stride : 0) + col[q],
                   here[q] && base ? c.dim - col[q] : 0, b[q]);
    }
#pragma unroll
    for (int q = 0; q < LOOKUP; ++q) {
        if (!here[q]) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) v[q][e] = __builtin_fmaf(c.scale, v[q][e], b[q][e]);
        store<T, E>(out + row[q] * c.row_stride + col[q], c.dim - col[q], v[q], c.streamed);
    }
}

// ---------------------------------------------------------------------------
// The gradient.  The rows are sorted by id, stably, by radix; a row that is left out has the
// key `entries`, behind all others.
//
// A pass of the sort by up to 10 bits takes two launches: counts a workgroup, and the
// placement, in which each workgroup sums up the counts before its own (at most 256
// workgroups' of 1024, from L2, 16 bytes a lane) and writes runs of 2 to 16 pairs that it has
// ordered in LDS.
// ---------------------------------------------------------------------------
constexpr int SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64;
constexpr int MOST_UNITS = 256;
constexpr int MOST_BITS = 10;
template <int R> constexpr int CHUNK = SORT_THREADS * R;

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// For each of R keys of a lane: the lanes with its digit, among those whose key is here.  A bit of
// all R at a time, since a chain of one key's bits waits for itself.
template <int R>
__device__ __forceinline__ void same_digits(const uint32_t (&digit)[R], const bool (&here)[R],
                                            int bits, uint64_t (&same)[R]) {
#pragma unroll
    for (int q = 0; q < R; ++q) same[q] = __ballot(here[q]);
    for (int k = 0; k < bits; ++k)
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const uint32_t all = (uint32_t)((int32_t)(digit[q] << (31 - k)) >> 31);
            const uint64_t ones = __ballot(all != 0);
            const uint32_t lo = ~((uint32_t)ones ^ all), hi = ~((uint32_t)(ones >> 32) ^ all);
            same[q] &= (uint64_t)hi << 32 | lo;
        }
}

// The sum of v over the threads before, and over all, of a workgroup of W wavefronts.
template <int W>
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t *wave_sum, uint32_t &all) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) wave_sum[wave] = x;
    __syncthreads();
    uint32_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if (w < wave) before += wave_sum[w];
        all += wave_sum[w];
    }
    __syncthreads();
    return before + x - v;
}

// The first pass reads ids; an id outside [0, entries) is the key `entries`.
__device__ __forceinline__ uint32_t key_of(const int32_t *ids, uint32_t entries, int64_t i) {
    return min((uint32_t)ids[i], entries);
}

struct Pass {
    const int32_t *ids;              // the first pass's keys, else NULL
    uint32_t entries;
    const uint2 *in;                 // key and row
    uint2 *out;
    int64_t rows, per;               // rows a workgroup
    int32_t units, shift, bits;
    void *table;                     // [workgroup][digit], of the kernels' type of count
    uint32_t *zero;                  // a word that the placement clears
};

__device__ __forceinline__ uint32_t key_at(const Pass &p, int64_t i) {
    return p.ids ? key_of(p.ids, p.entries, i) : p.in[i].x;
}

// C: 16 bits where a workgroup has fewer than 2^13 rows.  Short of rows, not of bandwidth: 1M rows
// 6.4 us a pass (4 MB of ids), 16384 4.6.
template <int R, typename C>
__global__ __launch_bounds__(SORT_THREADS) void k_embed_count(Pass p) {
    __shared__ uint32_t count[1 << MOST_BITS];
    const int bins = 1 << p.bits;
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) count[d] = 0;
    __syncthreads();
    const int64_t a = blockIdx.x * p.per, b = min(p.rows, a + p.per);
    for (int64_t c = a; c < b; c += CHUNK<R>) {
        uint32_t key[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const int64_t i = c + q * SORT_THREADS + threadIdx.x;
            key[q] = i < b ? key_at(p, i) : 0;
        }
#pragma unroll
        for (int q = 0; q < R; ++q)
            if (c + q * SORT_THREADS + threadIdx.x < b)
                atomicAdd(&count[(key[q] >> p.shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    C *to = static_cast<C *>(p.table) + (int64_t)blockIdx.x * bins;
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) to[d] = (C)count[d];
}

// next[d]: the place of this workgroup's first row of digit d.
template <typename C>
__device__ __forceinline__ void first_places(const Pass &p, int bins, uint32_t *next,
                                             uint32_t *total, uint32_t *wave_sum) {
    constexpr int E = 16 / sizeof(C);
    typedef C V __attribute__((ext_vector_type(E)));
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) next[d] = total[d] = 0;
    __syncthreads();
    const int wide = bins / E, col = threadIdx.x & (wide - 1);
    const int group = threadIdx.x / wide, groups = SORT_THREADS / wide;
    const V *table = static_cast<const V *>(p.table) + col;
    uint32_t all[E];
#pragma unroll
    for (int e = 0; e < E; ++e) all[e] = 0;
    const auto add = [&](int u, int end) {
        for (; u < end; u += 8) {
            V c[8], sum = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                c[q] = 0;
                if (u + q < end) c[q] = table[(int64_t)(u + q) * wide];
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) sum += c[q];         // 8 counts of 2^13 fit 16 bits
#pragma unroll
            for (int e = 0; e < E; ++e) all[e] += sum[e];
        }
    };
    // a run of the workgroups a group of threads: those before this one, and the others
    const int run = (p.units + groups - 1) / groups, from = group * run;
    const int to = min(from + run, p.units), mid = max(from, min(to, (int)blockIdx.x));
    add(from, mid);
#pragma unroll
    for (int e = 0; e < E; ++e) atomicAdd(&next[col * E + e], all[e]);
    add(mid, to);
#pragma unroll
    for (int e = 0; e < E; ++e) atomicAdd(&total[col * E + e], all[e]);
    __syncthreads();
    uint32_t sum, below = 0;
    for (int d0 = 0; d0 < bins; d0 += SORT_THREADS) {
        const int d = d0 + threadIdx.x;
        const uint32_t at =
            below + sum_before<SORT_WAVES>(d < bins ? total[d] : 0, wave_sum, sum);
        if (d < bins) next[d] += at;
        below += sum;
    }
    __syncthreads();
}

// Bound by the latency of its chain: the counts before its own out of L2, ranks in LDS, and stores
// to as many places as there are digits: 1M rows 14.6 us a pass, 16384 7.7.
template <int R, typename C>
__global__ __launch_bounds__(SORT_THREADS) void k_embed_place(Pass p) {
    extern __shared__ uint32_t lds[];
    const int bins = 1 << p.bits;
    uint32_t *wave_sum = lds;                        // SORT_WAVES
    uint32_t *next = wave_sum + SORT_WAVES;          // [digit] its next place
    uint32_t *first = next + bins;                   // [digit] its first place in the chunk
    uint2 *staged = reinterpret_cast<uint2 *>(first + bins);        // [place in the chunk]
    uint32_t *count = reinterpret_cast<uint32_t *>(staged + CHUNK<R>);      // [wave][digit]
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.zero = 0;
    const int64_t a = blockIdx.x * p.per, b = min(p.rows, a + p.per);
    uint2 pair[R];
    // wavefront by wavefront, so that equal digits keep their order
    const auto load_chunk = [&](int64_t c) {
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const int64_t i = c + wave * (64 * R) + q * 64 + lane;
            pair[q] = uint2{0, 0};
            if (i < b) pair[q] = p.ids ? uint2{key_of(p.ids, p.entries, i), (uint32_t)i} : p.in[i];
        }
    };
    load_chunk(a);                                   // on the way while the counts are
    uint32_t all;
    first_places<C>(p, bins, next, first, wave_sum);
    for (int64_t c = a; c < b; c += CHUNK<R>) {
        const int64_t w = c + wave * (64 * R);
        uint32_t rank[R];
        if (c > a) load_chunk(c);
        for (int d = threadIdx.x; d < SORT_WAVES * bins; d += SORT_THREADS) count[d] = 0;
        __syncthreads();
        uint32_t *mine = count + wave * bins;
        uint32_t digit[R];
        bool here[R];
        uint64_t same[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            digit[q] = (pair[q].x >> p.shift) & (bins - 1);
            here[q] = w + q * 64 + lane < b;
        }
        same_digits(digit, here, p.bits, same);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const uint32_t r = lanes_below(same[q]);
            rank[q] = here[q] ? mine[digit[q]] + r : 0;
            __builtin_amdgcn_wave_barrier();
            if (here[q] && r == 0) mine[digit[q]] = rank[q] + (uint32_t)__popcll(same[q]);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        uint32_t taken = 0;
        for (int d0 = 0; d0 < bins; d0 += SORT_THREADS) {
            const int d = d0 + threadIdx.x;
            uint32_t sum = 0;
            if (d < bins)
#pragma unroll
                for (int v = 0; v < SORT_WAVES; ++v) {
                    const uint32_t n = count[v * bins + d];
                    count[v * bins + d] = sum;
                    sum += n;
                }
            const uint32_t at = taken + sum_before<SORT_WAVES>(sum, wave_sum, all);
            if (d < bins) {
                first[d] = at;
                next[d] -= at;
            }
            taken += all;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < R; ++q) {
            if (here[q]) staged[first[digit[q]] + mine[digit[q]] + rank[q]] = pair[q];
        }
        __syncthreads();
        for (uint32_t l = threadIdx.x; l < taken; l += SORT_THREADS) {
            const uint2 v = staged[l];
            p.out[next[(v.x >> p.shift) & (bins - 1)] + l] = v;
        }
        __syncthreads();
        for (int d = threadIdx.x; d < bins; d += SORT_THREADS)       // the chunk is behind
            next[d] += d + 1 < bins ? first[d + 1] : taken;
        __syncthreads();
    }
}

// Few rows: the whole sort by one workgroup.  Up to 64 * EACH rows a wavefront, p.per of them;
// keys and order hold the sorted list in the end, key and row a lane's places of it.
template <int WAVES, int EACH>
__device__ __forceinline__ void sort_in_lds(const Pass &p, int passes, uint32_t *wave_sum,
                                            uint32_t *count, uint32_t *keys, uint16_t *order,
                                            uint32_t (&key)[EACH], uint16_t (&row)[EACH]) {
    constexpr int N = 64 * WAVES;
    const int bins = 1 << p.bits, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int a = min((int)p.rows, wave * (int)p.per), b = min((int)p.rows, a + (int)p.per);
    uint32_t rank[EACH];
#pragma unroll
    for (int q = 0; q < EACH; ++q) {
        const int i = a + q * 64 + lane;
        key[q] = i < b ? key_of(p.ids, p.entries, i) : 0;
        row[q] = (uint16_t)i;
    }
    for (int s = 0; s < passes; ++s) {
        const int shift = s * p.bits;
        for (int d = threadIdx.x * 4; d < WAVES * bins; d += N * 4)
            *reinterpret_cast<uint4 *>(count + d) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        uint32_t *mine = count + wave * bins;
        uint32_t digit[EACH];
        bool here[EACH];
        uint64_t same[EACH];
#pragma unroll
        for (int q = 0; q < EACH; ++q) {
            digit[q] = (key[q] >> shift) & (bins - 1);
            here[q] = a + q * 64 + lane < b;
        }
        same_digits(digit, here, p.bits, same);
#pragma unroll
        for (int q = 0; q < EACH; ++q) {
            if (a + q * 64 >= b) continue;
            const uint32_t r = lanes_below(same[q]);
            rank[q] = here[q] ? mine[digit[q]] + r : 0;
            __builtin_amdgcn_wave_barrier();
            if (here[q] && r == 0) mine[digit[q]] = rank[q] + (uint32_t)__popcll(same[q]);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        // a thread the digits DIGITS t and on
        constexpr int DIGITS = (1 << MOST_BITS) / N > 1 ? (1 << MOST_BITS) / N : 1;
        typedef uint32_t D __attribute__((ext_vector_type(DIGITS)));
        D *counts = reinterpret_cast<D *>(count) + threadIdx.x;
        D sum = 0;
        if ((int)threadIdx.x * DIGITS < bins)
#pragma unroll
            for (int v = 0; v < WAVES; ++v) sum += counts[v * bins / DIGITS];
        uint32_t total = 0, all;
#pragma unroll
        for (int e = 0; e < DIGITS; ++e) total += sum[e];
        total = sum_before<WAVES>(total, wave_sum, all);
        if ((int)threadIdx.x * DIGITS < bins) {
            D at;
#pragma unroll
            for (int e = 0; e < DIGITS; ++e) {
                at[e] = total;
                total += sum[e];
            }
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                const D n = counts[v * bins / DIGITS];
                counts[v * bins / DIGITS] = at;
                at += n;
            }
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < EACH; ++q) {
            if (!here[q]) continue;
            const uint32_t to = mine[digit[q]] + rank[q];
            keys[to] = key[q];
            order[to] = row[q];
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < EACH; ++q) {
            const int i = a + q * 64 + lane;
            if (i >= b) continue;
            key[q] = keys[i];
            row[q] = order[i];
        }
        __syncthreads();
    }
}

// (16384 rows of 17 bits take 46 us so, 20 by the kernels above.)
constexpr int SMALL_WAVES = 16, SMALL_THREADS = 64 * SMALL_WAVES, SMALL_EACH = 4;
constexpr int64_t SMALL_ROWS = SMALL_THREADS * SMALL_EACH;
__global__ __launch_bounds__(SMALL_THREADS) void k_embed_sort_small(Pass p, int32_t passes) {
    extern __shared__ uint32_t lds[];
    uint32_t *wave_sum = lds;                            // SMALL_WAVES
    uint32_t *count = wave_sum + SMALL_WAVES;            // [wave][digit]
    uint32_t *keys = count + (SMALL_WAVES << p.bits);    // [rows]
    uint16_t *order = reinterpret_cast<uint16_t *>(keys + p.rows);
    if (threadIdx.x == 0) *p.zero = 0;
    uint32_t key[SMALL_EACH];
    uint16_t row[SMALL_EACH];
    sort_in_lds<SMALL_WAVES>(p, passes, wave_sum, count, keys, order, key, row);
    const int a = (threadIdx.x >> 6) * (int)p.per;
    const int b = min((int)p.rows, a + (int)p.per);
#pragma unroll
    for (int q = 0; q < SMALL_EACH; ++q) {
        const int i = a + q * 64 + (threadIdx.x & 63);
        if (i < b) p.out[i] = uint2{key[q], row[q]};
    }
}

// ---------------------------------------------------------------------------
// The sums.  The sorted rows and the table's entries are merged: entry e comes behind the
// rows of key e, so that row i of key k lies at i + k.  A worker, `lanes` lanes that hold E columns
// each, takes `per` items of that list: it adds the rows and writes the entries, zeros for those
// without rows, so that rows and entries weigh the same whatever the ids, and what both read
// (an entry its base) is on the way AHEAD items at a time.  Where dtable is its own base, entries
// without rows are not on the list, and a worker takes `per` rows.
//
// A worker's end that falls into an entry's rows is put behind them if they are at most `whole`;
// else the entry is longer than a worker: each of its workers leaves its sum in parts, and the
// one in which it ends puts it on the list that k_embed_join works off.  Where all of a workgroup's
// workers are inside one entry, they leave one sum, as their first one's.  Sums of a worker are in
// the rows' order, those of parts in a fixed order too: the same bits in every run.
// ---------------------------------------------------------------------------
constexpr int SUM_WAVES = 4, SUM_THREADS = 64 * SUM_WAVES;
constexpr int MOST_ITEMS = 4096;     // of a workgroup
constexpr int AHEAD = 8;             // items on the way
constexpr uint32_t ENTRY = 0x80000000u;      // an item that is an entry: which, if not all are there
constexpr uint32_t NOTHING = 0xFFFFFFFFu;
constexpr uint32_t PASSED = 0xFFFFFFFEu;     // an entry that is summed elsewhere

struct Sums {
    int64_t rows, workers;
    uint32_t entries;
    int32_t dim, chunks;             // pieces of E columns
    int32_t lanes, groups;           // of a worker; workers a wavefront
    int32_t per;
    int32_t whole;                   // rows of an entry that are not parted: per, or all rows
    bool dense;                      // entries without rows are on the list
    bool streamed;                   // dtable is stored past the caches
    int64_t row_stride, table_stride;
    float scale;
    const uint2 *sorted;             // key and row
    const void *dout, *base;
    void *dtable;
    int32_t part_stride;             // dim in whole fours
    float *parts;                    // [worker][head, tail][part_stride]
    uint32_t *open;                  // [worker] the entry that it leaves open, or NOTHING
    uint32_t *found;                 // [0]: how many; then (worker, entry)
};
// Rows that a workgroup of `items` items may look at.
__host__ __device__ constexpr int held_rows(int items, int whole) { return items + 2 * whole + 2; }
// Bytes of LDS of a workgroup that holds `most` rows: key, item and, of lists of rows only, place
// (16 bits, since there are at most 2 * most items).  With the kernel's static ones they are at most
// the 64 KB that a launch may ask for without more ado.
constexpr size_t sum_lds(bool dense, size_t most) {
    return dense ? 4 * (2 * most + AHEAD + 1) : 4 * (3 * most + AHEAD) + 2 * (most + 2);
}
static_assert(sum_lds(false, held_rows(MOST_ITEMS, 64)) <= (63 << 10) &&
                  2 * held_rows(MOST_ITEMS, 64) < (1 << 16),
              "the largest lists' LDS");

// Rows and entries before an item.  i counts from the first row that the workgroup holds in LDS.
struct Cut {
    int i;
    uint32_t e;
    bool open;                       // e's rows begin before i, and there are more than `whole`
};

// The first of [lo, hi) for which under() does not hold, which does for all before.
template <class Under>
__device__ __forceinline__ int first_not(int lo, int hi, Under under) {
    while (lo < hi) {
        const int m = (lo + hi) >> 1;
        if (under(m)) lo = m + 1;
        else hi = m;
    }
    return lo;
}

// key[i]: row begin + i's, of `held` rows; the cut is in [lo, hi].
__device__ __forceinline__ Cut cut_at(const Sums &s, const uint32_t *key, int64_t begin, int held,
                                      int lo, int hi, int64_t d) {
    Cut c;
    if (s.dense) {
        d = min(d, s.rows + (int64_t)s.entries) - begin;
        c.i = first_not(lo, hi, [&](int m) { return m + (int64_t)key[m] < d; });
        c.e = (uint32_t)min(d - c.i, (int64_t)s.entries);
        c.open = begin + c.i > 0 && c.e < s.entries && key[c.i - 1] == c.e;
    } else {
        d = min(d, s.rows);
        c.i = (int)(d - begin);
        c.e = d > 0 ? key[c.i - 1] : 0;
        c.open = d > 0 && d < s.rows && c.e < s.entries && key[c.i] == c.e;
    }
    if (!c.open) return c;
    const int a = first_not(max(0, c.i - s.whole - 1), c.i, [&](int m) { return key[m] < c.e; });
    const int b = first_not(c.i, min(held, c.i + s.whole + 1),
                            [&](int m) { return key[m] <= c.e; });
    if (b - a <= s.whole) {
        c.i = b;
        c.e += 1;
        c.open = false;
    }
    return c;
}

// 256-ary search: the number of rows i with i + key[i] below d[0] and d[1], of [lo, hi] both.
__device__ __forceinline__ void both_ends(const Sums &s, const int64_t (&d)[2], int64_t *found) {
    int64_t lo[2], hi[2];
    for (int x = 0; x < 2; ++x) {
        lo[x] = max((int64_t)0, d[x] - (int64_t)s.entries);
        hi[x] = min(s.rows, d[x]);
    }
    while (hi[0] > lo[0] || hi[1] > lo[1]) {
        uint32_t k[2];
        int64_t m[2], step[2];
        bool in[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            step[x] = (hi[x] - lo[x] + SUM_THREADS - 1) / SUM_THREADS;
            m[x] = lo[x] + threadIdx.x * step[x];
            in[x] = m[x] < hi[x];
            k[x] = in[x] ? s.sorted[m[x]].x : 0;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int n = __syncthreads_count(in[x] && m[x] + (int64_t)k[x] < d[x]);
            if (n == 0) {
                hi[x] = lo[x];
                continue;
            }
            const int64_t last = lo[x] + (n - 1) * step[x];
            hi[x] = min(hi[x], last + step[x]);
            lo[x] = last + 1;
        }
    }
    found[0] = lo[0];
    found[1] = lo[1];
}

// The items [p, end): rows are added to acc, at_entry(entry, its base) takes it.  next: the next
// entry, where all are on the list.  SOME: some entries are passed.
template <typename T, int E, bool BASE, bool ONE, bool SOME, class AtEntry>
__device__ __forceinline__ void walk(const Sums &s, const uint32_t *item, int p, int end,
                                     uint32_t next, const T *dout, const T *base, const T *dtable,
                                     float (&acc)[E], AtEntry at_entry) {
    const T *some_row = s.rows ? dout : dtable;
    for (; p < end; p += AHEAD) {
        uint32_t what[AHEAD];
        Run<T, E> v[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            what[q] = item[p + q];
            if constexpr (ONE) what[q] = __builtin_amdgcn_readfirstlane(what[q]);
            if (s.dense) {
                const bool entry = what[q] == ENTRY, passed = SOME && what[q] == PASSED;
                what[q] |= entry ? next : passed ? NOTHING : 0;
                next += entry || passed;
            }
            if (p + q >= end) what[q] = NOTHING;
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const bool is_row = what[q] < ENTRY;
            // without branches: what has nothing to read takes row 0, or entry 0 where there are no
            // rows, which is never in place
            if constexpr (BASE) {
                const T *at = is_row ? dout : what[q] == NOTHING ? some_row : base;
                const uint32_t which = what[q] == NOTHING ? 0 : what[q] & ~ENTRY;
                v[q] = *reinterpret_cast<const Run<T, E> *>(
                    at + which * (is_row ? s.row_stride : s.table_stride));
            } else {
                v[q] = *reinterpret_cast<const Run<T, E> *>(
                    some_row + (is_row ? what[q] : 0) * s.row_stride);
            }
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const bool is_row = what[q] < ENTRY;
            if constexpr (ONE) {
                if (is_row)
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] += to_f32(v[q][e]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = is_row ? acc[e] + to_f32(v[q][e]) : acc[e];
            }
            if (is_row || what[q] == NOTHING) continue;
            at_entry(what[q] & ~ENTRY, v[q]);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = 0.0f;
        }
    }
}

// E > 1: the last piece of a row that is no multiple of E long is its last E columns, some of which
// the piece before has too: both lanes write the same.
// BASE: dtable has a base.  ONE: one worker a wavefront, whose items are the same in all lanes.
// Bound by memory: 1M x 64 f32 rows in any order to 100000 entries take 69 us, 282 MB at 4.1 TB/s
// in pieces of 256 bytes; 16384 x 1024 bf16 on top of 65536 entries 56.  In place 78 and 21, and 60
// where 1030 columns leave 2 bytes a lane.
template <typename T, int E, bool BASE, bool ONE>
__global__ __launch_bounds__(SUM_THREADS) void k_embed_sum(Sums s) {
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t wave_sum[SUM_WAVES];
    const int items = SUM_WAVES * s.groups * s.per, most = held_rows(items, s.whole);
    uint32_t *key = lds;                             // [row]
    uint32_t *item = key + most;                     // [item]: a row, or an entry
    // [row]: its item, where that is not i + key
    uint16_t *place = reinterpret_cast<uint16_t *>(item + 2 * most + AHEAD);
    const int64_t first = (int64_t)group_id() * (SUM_WAVES * s.groups);
    if (first >= s.workers) return;
    const int64_t d[2] = {first * s.per, min(min(first + SUM_WAVES * s.groups, s.workers) * s.per,
                                             s.rows + (s.dense ? (int64_t)s.entries : 0))};
    int64_t ends[2] = {d[0], d[1]};
    if (s.dense) both_ends(s, d, ends);
    const int64_t begin = max((int64_t)0, ends[0] - s.whole - 1);
    const int held = (int)(min(s.rows, ends[1] + s.whole + 1) - begin);
    const int lo = (int)(ends[0] - begin), hi = (int)(ends[1] - begin);
    if (s.dense) {
        for (int i = threadIdx.x; i < items + s.whole + 2; i += SUM_THREADS) item[i] = ENTRY;
        __syncthreads();
        for (int i = threadIdx.x; i < held; i += SUM_THREADS) {
            const uint2 x = s.sorted[begin + i];
            key[i] = x.x;
            const int64_t at = begin + i + (int64_t)x.x - d[0];
            if (at >= 0 && at < items + s.whole + 2 && x.x < s.entries) item[at] = x.y;
        }
    } else {
        for (int i = threadIdx.x; i < held; i += SUM_THREADS) key[i] = s.sorted[begin + i].x;
        __syncthreads();
        // a row's item lies behind as many entries as end before it
        uint32_t before = 0, all;
        for (int i0 = 0; i0 < held; i0 += SUM_THREADS) {
            const int i = i0 + threadIdx.x;
            const uint32_t k = i < held ? key[i] : NOTHING;
            const bool ends_here = k < s.entries && (begin + i + 1 >= s.rows ||
                                                     (i + 1 < held && key[i + 1] != k));
            const uint32_t at = i + before + sum_before<SUM_WAVES>(ends_here, wave_sum, all);
            if (i < held) {
                place[i] = (uint16_t)at;
                item[at] = s.sorted[begin + i].y;
                if (ends_here) item[at + 1] = ENTRY | k;
            }
            before += all;
        }
        if (threadIdx.x == 0) place[held] = (uint16_t)(held + before);
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, group = lane / s.lanes;
    const int mine = (threadIdx.x >> 6) * s.groups + min(group, s.groups - 1);
    const int64_t worker = min(first + mine, s.workers - 1);
    const int32_t chunk = min(blockIdx.y * 64 + lane - group * s.lanes, s.chunks - 1);
    // lanes without a worker or columns of their own do another's work and write none of it
    const bool idle = group >= s.groups || first + mine >= s.workers ||
                      (int)(blockIdx.y * 64) + lane - group * s.lanes >= s.chunks;
    const Cut from = cut_at(s, key, begin, held, lo, hi, worker * s.per);
    Cut to = cut_at(s, key, begin, held, lo, hi, (worker + 1) * s.per);
    if (to.i > from.i && key[to.i - 1] >= s.entries)         // rows that are left out, behind all
        to.i = first_not(from.i, to.i, [&](int m) { return key[m] < s.entries; });
    uint32_t next = from.e;          // the next entry, where all are on the list
    int p = s.dense ? (int)(begin + from.i + (int64_t)from.e - d[0]) : (int)place[from.i];
    int end = s.dense ? (int)(begin + to.i + (int64_t)to.e - d[0]) : (int)place[to.i];
    if constexpr (ONE) {
        next = __builtin_amdgcn_readfirstlane(next);
        p = __builtin_amdgcn_readfirstlane(p);
        end = __builtin_amdgcn_readfirstlane(end);
    }
    const int col = min(chunk * E, s.dim - E);
    const T *dout = static_cast<const T *>(s.dout) + col;
    const T *base = BASE ? static_cast<const T *>(s.base) + col : nullptr;
    T *dtable = static_cast<T *>(s.dtable) + col;
    float *parts = s.parts + worker * 2 * s.part_stride + col;

    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    bool head = from.open;
    const auto leave = [&](int side) {
        if (idle) return;
#pragma unroll
        for (int e = 0; e < E; ++e) parts[side * s.part_stride + e] = acc[e];
    };
    walk<T, E, BASE, ONE, false>(s, item, p, end, next, dout, base, dtable, acc,
                          [&](uint32_t entry, const Run<T, E> &v) {
        if (head) {
            leave(0);
            if (!idle && chunk == 0) {
                const uint32_t at = atomicAdd(&s.found[0], 1u);
                s.found[2 + 2 * at] = (uint32_t)worker;
                s.found[3 + 2 * at] = entry;
            }
            head = false;
        } else {
            Run<T, E> out;
#pragma unroll
            for (int e = 0; e < E; ++e)
                out[e] = (T)__builtin_fmaf(s.scale, acc[e], BASE ? to_f32(v[e]) : 0.0f);
            if (!idle)
                put(dtable + entry * s.table_stride, out, s.streamed);
        }
    });
    if (!idle && chunk == 0) s.open[worker] = to.open ? to.e : NOTHING;
    const bool inside = from.open && to.open && from.e == to.e;
    const int here = (int)min((int64_t)SUM_WAVES * s.groups, s.workers - first);
    if (!__syncthreads_and(inside) || here == 1) {
        if (to.open) leave(1);
        return;
    }
    float *meet = reinterpret_cast<float *>(lds) + threadIdx.x * E;
    const int stride = s.lanes * E;                  // between the workers of a wavefront
#pragma unroll
    for (int e = 0; e < E; ++e) meet[e] = acc[e];
    for (int o = 128; o > 0; o >>= 1) {              // at most 256 workers
        __syncthreads();
        const int other = mine + o;
        if (!idle && mine < o && other < here) {
            const float *from_other =
                meet + ((other / s.groups - (int)(threadIdx.x >> 6)) * 64 * E) +
                (other % s.groups - group) * stride;
#pragma unroll
            for (int e = 0; e < E; ++e) meet[e] += from_other[e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = meet[e];
    if (mine == 0) leave(1);
}

// The entries on the list: heads and tails of their workers, from the first that left the entry
// open to the one in which it ends; of workgroups all inside it, one tail.  A wavefront an entry,
// or all of a workgroup's an entry of more than WAVE_PARTS parts: slices of the parts are summed
// side by side, and the slices' sums by halves.
constexpr int JOIN_WAVES = 4, JOIN_THREADS = 64 * JOIN_WAVES;
constexpr int WAVE_PARTS = 64;
constexpr int PARTS = 8;             // parts on the way
struct Span {
    int32_t start, last;             // workers
    int32_t blocks, behind;          // the first worker of the workgroups all inside, and behind them
    int32_t inside, each;            // how many workgroups, of how many workers
    uint32_t entry;
    __device__ __forceinline__ int32_t parts() const {
        return last + 1 - start - (behind - blocks) + inside;
    }
    // The place in parts of the i-th part.
    __device__ __forceinline__ int64_t at(int32_t i) const {
        const int32_t before = blocks - start;
        const int32_t w = i < before ? start + i
                          : i < before + inside ? blocks + (i - before) * each
                                                : behind + (i - before - inside);
        return (int64_t)w * 2 + (w < last);
    }
};
// A launch and a chain of three reads for most: 16384 x 1024 to 65536 entries 6.0 us, 1M x 64 to
// 100000 8.2.
template <typename T>
__global__ __launch_bounds__(JOIN_THREADS) void k_embed_join(Sums s) {
    typedef float V __attribute__((ext_vector_type(4)));
    __shared__ V sums[JOIN_THREADS];
    __shared__ Span spans[JOIN_WAVES];
    const uint32_t count = s.found[0];
    const int fours = s.part_stride / 4, wide = min(fours, 64), groups = 64 / wide;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, group = lane / wide;
    const int col0 = lane - group * wide;
    // Slice `slice` of `slices` of a span's parts, four columns.
    const auto part_sum = [&](const Span &x, int slice, int slices, int four) {
        const int32_t n = x.parts(), each = (n + slices - 1) / slices;
        const int32_t a = slice * each, b = min(a + each, n);
        V sum = {0, 0, 0, 0};
        if (group < groups && four < fours)
            for (int32_t i = a; i < b; i += PARTS) {
                V v[PARTS];
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
                    v[q] = *reinterpret_cast<const V *>(
                        s.parts + x.at(min(i + q, b - 1)) * s.part_stride + four * 4);
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] += i + q < b ? v[q][e] : 0.0f;
            }
        sums[threadIdx.x] = sum;
    };
    // The sum of slice v and the one o behind.
    const auto halve = [&](int v, int o, int slices, int first_wave) {
        if (group >= groups || v >= o || v + o >= slices) return;
        const V other = sums[(first_wave + (v + o) / groups) * 64 + (v + o) % groups * wide + col0];
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[threadIdx.x][e] += other[e];
    };
    const auto write = [&](uint32_t entry, int four) {
        if (group != 0 || four >= fours) return;
        const V total = sums[threadIdx.x];
        const int col = four * 4;
        const int64_t at = (int64_t)entry * s.table_stride + col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < s.dim) {
                const float b0 = s.base ? to_f32(static_cast<const T *>(s.base)[at + e]) : 0.0f;
                static_cast<T *>(s.dtable)[at + e] = (T)__builtin_fmaf(s.scale, total[e], b0);
            }
    };
    // few entries: one a workgroup
    const uint32_t turn = count > gridDim.x ? JOIN_WAVES : 1;
    for (uint32_t f0 = blockIdx.x * turn; f0 < count; f0 += gridDim.x * turn) {
        const uint32_t f = f0 + wave;
        Span x{};
        x.each = SUM_WAVES * s.groups;
        x.last = -1;
        const bool has = (uint32_t)wave < turn && f < count;
        if (has) {
            x.last = x.start = (int32_t)s.found[2 + 2 * f];
            x.entry = s.found[3 + 2 * f];
            // the entry's workers lie side by side: the 64 before, or 64-ary search
            const int w = x.start - 1 - lane;
            const int n = __popcll(__ballot(w >= 0 && s.open[max(w, 0)] == x.entry));
            x.start -= n;
            int lo = 0;
            while (n == 64 && x.start > lo) {        // the first one is in [lo, start]
                const int step = (x.start - lo + 63) / 64;
                const int64_t m = x.start - (int64_t)step * (lane + 1);
                const int more =
                    __popcll(__ballot(m >= lo && s.open[max(m, (int64_t)lo)] == x.entry));
                lo = (int)max((int64_t)lo, x.start - (int64_t)step * (more + 1) + 1);
                x.start -= step * more;
            }
            x.blocks = (x.start / x.each + 1) * x.each;
            x.behind = x.last / x.each * x.each;
            if (x.blocks >= x.behind) x.blocks = x.behind = x.last;
            x.inside = (x.behind - x.blocks) / x.each;
        }
        if (lane == 0) spans[wave] = x;
        __syncthreads();
        for (int four0 = blockIdx.y * wide; four0 < fours; four0 += gridDim.y * wide) {
            const int four = four0 + col0;
            if (has && x.parts() <= WAVE_PARTS) {
                part_sum(x, group, groups, four);
                for (int o = 32; o > 0; o >>= 1) {
                    __builtin_amdgcn_wave_barrier();
                    halve(group, o, groups, wave);
                }
                __builtin_amdgcn_wave_barrier();
                write(x.entry, four);
                __builtin_amdgcn_wave_barrier();
            }
            for (uint32_t y = 0; y < turn && f0 + y < count; ++y) {
                if (spans[y].parts() <= WAVE_PARTS) continue;
                const int slice = wave * groups + group, slices = JOIN_WAVES * groups;
                __syncthreads();
                part_sum(spans[y], slice, slices, four);
                for (int o = 32 * JOIN_WAVES; o > 0; o >>= 1) {
                    __syncthreads();
                    halve(slice, o, slices, 0);
                }
                __syncthreads();
                if (wave == 0) write(spans[y].entry, four);
                __syncthreads();
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Up to FEW_ROWS rows to many entries: one launch, bound by the chain of the sort (6 us) and the reads behind it
// (1000 x 64 f32 to 60000 entries 19.8 us with the host's call).  Every workgroup sorts all of them for
// itself; the first `lists` take the merged list as above, without the entries of more than `whole`
// rows, and each of the others one of those.
// ---------------------------------------------------------------------------
constexpr int FEW_EACH = 4;
constexpr int64_t FEW_ROWS = 64 * SUM_WAVES * FEW_EACH;
struct FewLayout {                   // words of LDS, at most 28 KB
    int count, keys, order, place, item, all;
};
__host__ __device__ inline FewLayout few_layout(const Sums &s, int bits, int elements) {
    FewLayout l{};
    const int items = SUM_WAVES * s.groups * s.per + s.whole + 2 + AHEAD;
    const int rows = ((int)s.rows + 63) / 64 * 64;
    l.keys = SUM_WAVES;              // behind the wavefronts' sums
    l.order = l.keys + rows;
    l.place = l.order + rows / 2;
    l.count = l.item = (l.place + rows + 4) / 4 * 4;     // one behind the other in time
    int most = SUM_WAVES << bits;
    most = most > items ? most : items;
    most = most > 2 * rows + 2 + AHEAD ? most : 2 * rows + 2 + AHEAD;
    most = most > SUM_THREADS * elements ? most : SUM_THREADS * elements;
    l.all = l.item + most;
    return l;
}

template <typename T, int E, bool BASE>
__global__ __launch_bounds__(SUM_THREADS) void k_embed_few(Sums s, Pass p, int32_t passes,
                                                           int32_t lists) {
    extern __shared__ uint32_t lds[];
    const FewLayout l = few_layout(s, p.bits, E);
    uint32_t *wave_sum = lds, *key = lds + l.keys, *item = lds + l.item, *place = lds + l.place;
    uint16_t *order = reinterpret_cast<uint16_t *>(lds + l.order);
    {
        uint32_t k[FEW_EACH];
        uint16_t r[FEW_EACH];
        sort_in_lds<SUM_WAVES>(p, passes, wave_sum, lds + l.count, key, order, k, r);
    }
    const int rows = (int)s.rows, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int group = lane / s.lanes, chunk0 = blockIdx.y * 64 + lane - group * s.lanes;
    const int32_t chunk = min(chunk0, s.chunks - 1);
    const int col = min(chunk * E, s.dim - E);
    const T *dout = static_cast<const T *>(s.dout) + col;
    const T *base = BASE ? static_cast<const T *>(s.base) + col : nullptr;
    T *dtable = static_cast<T *>(s.dtable) + col;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    const auto write = [&](uint32_t entry, const Run<T, E> &b) {
        Run<T, E> out;
#pragma unroll
        for (int e = 0; e < E; ++e)
            out[e] = (T)__builtin_fmaf(s.scale, acc[e], BASE ? to_f32(b[e]) : 0.0f);
        put(dtable + entry * s.table_stride, out, s.streamed);
    };

    if ((int)blockIdx.x >= lists) {
        // the rows [a, b) of the entry: slices of them side by side, and their sums by halves
        __shared__ int found;
        uint32_t before = 0, all;
        for (int i0 = 0; i0 < rows; i0 += SUM_THREADS) {
            const int i = i0 + threadIdx.x;
            const bool starts = i + s.whole < rows && key[i] < s.entries &&
                                (i == 0 || key[i - 1] != key[i]) && key[i + s.whole] == key[i];
            const uint32_t at = before + sum_before<SUM_WAVES>(starts, wave_sum, all);
            if (starts && at == blockIdx.x - lists) found = i;
            before += all;
        }
        __syncthreads();
        if (blockIdx.x - lists >= before) return;
        const int a = found;
        const uint32_t entry = key[a];
        const int b = first_not(a, rows, [&](int m) { return key[m] == entry; });
        const int groups = 64 / s.lanes, slices = SUM_WAVES * groups;
        const int slice = wave * groups + min(group, groups - 1);
        const bool idle = group >= groups || chunk0 >= s.chunks;
        const int each = (b - a + slices - 1) / slices;
        const int to = min(b, a + (slice + 1) * each);
        for (int i = a + slice * each; i < to; i += AHEAD) {
            Run<T, E> v[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                v[q] = *reinterpret_cast<const Run<T, E> *>(dout + order[min(i + q, to - 1)] *
                                                                       s.row_stride);
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += i + q < to ? to_f32(v[q][e]) : 0.0f;
        }
        float *meet = reinterpret_cast<float *>(item) + threadIdx.x * E;
#pragma unroll
        for (int e = 0; e < E; ++e) meet[e] = acc[e];
        for (int o = 128; o > 0; o >>= 1) {
            __syncthreads();
            const int other = slice + o;
            if (!idle && slice < o && other < slices) {
                const float *from = meet + ((other / groups - wave) * 64 +
                                            (other % groups - group) * s.lanes) * E;
#pragma unroll
                for (int e = 0; e < E; ++e) meet[e] += from[e];
            }
        }
        if (idle || slice != 0) return;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = meet[e];
        Run<T, E> b0{};
        if constexpr (BASE) b0 = *reinterpret_cast<const Run<T, E> *>(base + entry * s.table_stride);
        write(entry, b0);
        return;
    }

    const int64_t first = (int64_t)blockIdx.x * (SUM_WAVES * s.groups), d0 = first * s.per;
    const int items = SUM_WAVES * s.groups * s.per + s.whole + 2;
    // whether the entry of row i has more than `whole` rows
    const auto is_long = [&](int i) {
        const uint32_t k = key[i];
        const int a = first_not(max(0, i - s.whole), i, [&](int m) { return key[m] < k; });
        return a + s.whole < rows && key[a + s.whole] == k;
    };
    if (s.dense) {
        for (int i = threadIdx.x; i < items; i += SUM_THREADS) item[i] = ENTRY;
        __syncthreads();
        for (int i = threadIdx.x; i < rows; i += SUM_THREADS) {
            const uint32_t k = key[i];
            const int64_t at = i + (int64_t)k - d0;
            if (k >= s.entries || at < -1 || at >= items) continue;
            const bool elsewhere = is_long(i);
            if (at >= 0) item[at] = elsewhere ? NOTHING : order[i];
            if (elsewhere && at + 1 < items && (i + 1 == rows || key[i + 1] != k))
                item[at + 1] = PASSED;
        }
    } else {
        uint32_t before = 0, all;
        for (int i0 = 0; i0 < rows; i0 += SUM_THREADS) {
            const int i = i0 + threadIdx.x;
            const uint32_t k = i < rows ? key[i] : NOTHING;
            const bool ends_here = k < s.entries && (i + 1 == rows || key[i + 1] != k);
            const uint32_t at = i + before + sum_before<SUM_WAVES>(ends_here, wave_sum, all);
            if (i < rows) {
                const bool elsewhere = k < s.entries && is_long(i);
                place[i] = at;
                item[at] = elsewhere ? NOTHING : order[i];
                if (ends_here) item[at + 1] = elsewhere ? NOTHING : ENTRY | k;
            }
            before += all;
        }
        if (threadIdx.x == 0) place[rows] = rows + before;
    }
    __syncthreads();
    const int mine = wave * s.groups + group;
    const int64_t worker = first + mine;
    if (group >= s.groups || worker >= s.workers || chunk0 >= s.chunks) return;
    const Cut from = cut_at(s, key, 0, rows, 0, rows, worker * s.per);
    Cut to = cut_at(s, key, 0, rows, 0, rows, (worker + 1) * s.per);
    if (to.i > from.i && key[to.i - 1] >= s.entries)         // rows that are left out, behind all
        to.i = first_not(from.i, to.i, [&](int m) { return key[m] < s.entries; });
    const int at = s.dense ? (int)(from.i + (int64_t)from.e - d0) : (int)place[from.i];
    const int end = s.dense ? (int)(to.i + (int64_t)to.e - d0) : (int)place[to.i];
    walk<T, E, BASE, false, true>(s, item, at, end, from.e, dout, base, dtable, acc, write);
}

// ---------------------------------------------------------------------------
// Few entries: slices of up to FEW_ROWS rows, each sorted and summed by a workgroup, which writes the
// sums of the entries that it has and a bit for each of them; and those of all slices summed up.
// Two launches instead of four or more.  The first is bound by its sort (7 us) and then by reading
// dout: 99991 x 37 to 300 entries 13.4 us and 6.0 for the sums' sums, 1M x 64 to 5 43.5 (5.9 TB/s)
// and 8.5.
// ---------------------------------------------------------------------------
constexpr int SLICE_WORDS = (1 << MOST_BITS) / 32;   // bits of a slice's entries

template <typename T, int E>
__global__ __launch_bounds__(SUM_THREADS) void k_embed_slice(Sums s, Pass p) {
    extern __shared__ uint32_t lds[];
    uint32_t *wave_sum = lds, *bits = lds + SUM_WAVES, *key = bits + SLICE_WORDS;
    uint16_t *order = reinterpret_cast<uint16_t *>(key + FEW_ROWS);
    uint32_t *rest = key + FEW_ROWS + FEW_ROWS / 2;
    const int64_t row0 = (int64_t)blockIdx.x * s.whole;
    p.ids += row0;
    p.rows = min(p.rows - row0, (int64_t)s.whole);
    if (threadIdx.x < SLICE_WORDS) bits[threadIdx.x] = 0;
    {
        uint32_t k[FEW_EACH];
        uint16_t r[FEW_EACH];
        sort_in_lds<SUM_WAVES>(p, 1, wave_sum, rest, key, order, k, r);
    }
    const int kept = first_not(0, (int)p.rows, [&](int m) { return key[m] < s.entries; });
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int group = lane / s.lanes, chunk0 = blockIdx.y * 64 + lane - group * s.lanes;
    const int32_t chunk = min(chunk0, s.chunks - 1);
    const int col = min(chunk * E, s.dim - E);
    const T *dout = static_cast<const T *>(s.dout) + row0 * s.row_stride + col;
    float *sums = s.parts + (int64_t)blockIdx.x * s.entries * s.part_stride + col;
    for (int i = threadIdx.x; i < kept; i += SUM_THREADS)
        if (i == 0 || key[i - 1] != key[i]) atomicOr(&bits[key[i] >> 5], 1u << (key[i] & 31));
    // a worker takes `each` rows of the sorted list.  What it has of an entry that a worker before
    // began goes to the LDS, where the worker that began it finds it.
    const int mine = wave * s.groups + group, workers = SUM_WAVES * s.groups;
    const bool idle = group >= s.groups || chunk0 >= s.chunks;
    const int each = (kept + workers - 1) / workers;
    const int a = idle ? kept : min(kept, mine * each), b = min(kept, a + each);
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    float *head = reinterpret_cast<float *>(rest);
    const auto write = [&](uint32_t entry) {
        Run<float, E> out;
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = acc[e];
        *reinterpret_cast<Run<float, E> *>(sums + (int64_t)entry * s.part_stride) = out;
    };
    const auto leave = [&]() {
#pragma unroll
        for (int e = 0; e < E; ++e) head[threadIdx.x * E + e] = acc[e];
    };
    bool begun = a > 0 && a < b && key[a - 1] == key[a];     // by a worker before
    for (int i = a; i < b; i += AHEAD) {
        Run<T, E> v[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
            v[q] = *reinterpret_cast<const Run<T, E> *>(dout + order[min(i + q, b - 1)] *
                                                                   s.row_stride);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            if (i + q >= b) break;
            if (i + q > a && key[i + q - 1] != key[i + q]) {
                if (begun) leave();
                else write(key[i + q - 1]);
                begun = false;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += to_f32(v[q][e]);
        }
    }
    if (a < b && begun) leave();
    __syncthreads();
    if (blockIdx.y == 0 && threadIdx.x < SLICE_WORDS)
        s.open[(int64_t)blockIdx.x * SLICE_WORDS + threadIdx.x] = bits[threadIdx.x];
    if (a >= b || begun) return;
    const uint32_t entry = key[b - 1];
    for (int w = mine + 1, at = b; at < kept && key[at] == entry; ++w, at += each) {
        const int from = (w / s.groups * 64 + w % s.groups * s.lanes + lane - group * s.lanes) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += head[from + e];
    }
    write(entry);
}

// A workgroup an entry and 256 columns, four a lane; the lanes share the slices.
template <typename T>
__global__ __launch_bounds__(SUM_THREADS) void k_embed_total(Sums s, int32_t slices) {
    typedef float V __attribute__((ext_vector_type(4)));
    __shared__ V meet[SUM_THREADS];
    const uint32_t entry = blockIdx.x;
    const int chunks = s.part_stride / 4 - blockIdx.y * 64, lanes = min(chunks, 64);
    const int sub = threadIdx.x / lanes, subs = SUM_THREADS / lanes;
    const int64_t col = (blockIdx.y * 64 + threadIdx.x - sub * lanes) * 4;
    V acc = {0, 0, 0, 0};
    bool any = false;
    if (sub < subs)
        for (int p0 = sub; p0 < slices; p0 += AHEAD * subs) {
            uint32_t word[AHEAD];
            V v[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int64_t p = min(p0 + q * subs, slices - 1);
                word[q] = s.open[p * SLICE_WORDS + (entry >> 5)];
                v[q] = *reinterpret_cast<const V *>(s.parts + (p * s.entries + entry) *
                                                                  s.part_stride + col);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {            // what is not there was not written
                const bool there = p0 + q * subs < slices && ((word[q] >> (entry & 31)) & 1u);
                any |= there;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = there ? acc[e] + v[q][e] : acc[e];
            }
        }
    meet[threadIdx.x] = acc;
    if (!__syncthreads_or(any) && s.base == s.dtable) return;
    for (int o = SUM_THREADS / 2; o > 0; o >>= 1) {
        if (sub < o && sub + o < subs) {
            const V other = meet[threadIdx.x + o * lanes];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += other[e];
            meet[threadIdx.x] = acc;
        }
        __syncthreads();
    }
    if (sub != 0) return;
    const int n = (int)min((int64_t)4, s.dim - col);
    const int64_t at = (int64_t)entry * s.table_stride + col;
    float b[4] = {0, 0, 0, 0}, out[4];
    if (s.base) load<T, 4>(static_cast<const T *>(s.base) + at, n, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = __builtin_fmaf(s.scale, acc[e], b[e]);
    store<T, 4>(static_cast<T *>(s.dtable) + at, n, out, false);
}

int bits_of(int64_t most) {          // of keys 0..most
    int bits = 1;
    while (bits < 32 && (most >> bits)) ++bits;
    return bits;
}

struct GradShape {
    int units, passes, bits;
    bool small;
    int64_t per;                     // rows a workgroup of the sort, or a wavefront
    int each;                        // R
    bool narrow;                     // counts of 16 bits
    int lanes, groups, cols, items, whole, chunks;
    int elements;                    // E
    bool dense;
    int64_t workers;
    bool few;                        // one launch
    int64_t lists;                   // its workgroups of the list
    int64_t slices;                  // of few entries, g.whole rows each; 0: none
};

// Slices: as many as CUs, down to 128 rows (10000 x 64 to 1000: 14.3 us, 18.2 by 64 rows and 17.4 by
// 512), while their sums do not outweigh the longer sort (with the host's call, 50000 x 64 to 1000,
// 50 MB of sums: 21.0 us, 36.8 without slices; 1M x 16 to 1000, 63 MB: 49.2 and 63.7; 300000 x 256 to
// 300, 90 MB: 113 and 93).
constexpr int64_t SLICE_LEAST = 128, SLICE_BYTES = (int64_t)64 << 20;
constexpr int64_t SLICED_FEW = 48, SLICED_FEW_ELEMENTS = (int64_t)1 << 18;

int32_t part_stride(const EmbedCall &c) { return (c.dim + 3) / 4 * 4; }

GradShape grad_shape(const EmbedCall &c) {
    GradShape g{};
    const int bits = bits_of(c.entries);
    g.small = c.rows <= SMALL_ROWS;
    g.passes = (bits + MOST_BITS - 1) / MOST_BITS;
    g.bits = std::max(3, (bits + g.passes - 1) / g.passes);      // 16 bytes of counts
    if (g.small) {
        g.per = ((c.rows + SMALL_WAVES - 1) / SMALL_WAVES + 63) / 64 * 64;
        g.units = 1;
    } else {
        g.each = c.rows <= (int64_t)MOST_UNITS * CHUNK<4> ? 4 : 8;
        const int64_t chunk = (int64_t)SORT_THREADS * g.each;
        const int64_t chunks = (c.rows + chunk - 1) / chunk;
        g.per = (chunks + MOST_UNITS - 1) / MOST_UNITS * chunk;
        g.units = (int)((c.rows + g.per - 1) / g.per);
        g.narrow = g.per < (1 << 13);
    }
    // 16 bytes a lane, unless the last piece of a row shares columns with one of another
    // wavefront that may have written them to the base
    const int elements = c.bf16 ? 8 : 4;
    const bool apart = c.dim % elements == 0 || c.dim <= 64 * elements || c.base != c.dtable;
    g.elements = c.dim >= elements && apart ? elements : 1;
    g.chunks = (c.dim + g.elements - 1) / g.elements;
    g.lanes = std::min(g.chunks, 64);
    g.groups = 64 / g.lanes;
    g.cols = (g.chunks + 63) / 64;
    g.dense = c.base != c.dtable;
    const int64_t items = c.rows + (g.dense ? c.entries : 0);
    // 16 to 64 items a worker, as many as leave every CU 16 wavefronts
    const int64_t workers = (int64_t)16 * c.num_cus * g.groups / g.cols + 1;
    int64_t per = std::min<int64_t>(64, std::max<int64_t>(16, items / workers));
    per = std::min<int64_t>(per, MOST_ITEMS / (SUM_WAVES * g.groups));
    // a workgroup each CU rather than full wavefronts: short lists are bound by what a workgroup
    // does before its first row (10532 x 1 to 291457 16.3 us by 256 workers a workgroup, 12.8 so)
    g.groups = (int)std::max<int64_t>(
        1, std::min<int64_t>(g.groups, items / per / (SUM_WAVES * (int64_t)c.num_cus)));
    g.items = (int)per;
    g.whole = c.rows <= 64 ? 64 : g.items;           // few rows: nothing to join
    g.workers = (items + per - 1) / per;
    // few rows: sorted again by each workgroup, which pays up to where there are very many of them
    // (1000 x 64 f32 to 60,000 entries 19.8 us, 27.3 by three launches; to 1M 70.5 and 73.2)
    g.lists = (g.workers + (int64_t)SUM_WAVES * g.groups - 1) / ((int64_t)SUM_WAVES * g.groups);
    g.few = c.rows >= 1 && c.rows <= FEW_ROWS && g.lists * g.cols <= 64 * (int64_t)c.num_cus;
    if (g.few) {
        g.whole = 64;
        g.per = ((c.rows + SUM_WAVES - 1) / SUM_WAVES + 63) / 64 * 64;
    }
    const int64_t slice = std::min<int64_t>(
        FEW_ROWS, std::max<int64_t>(SLICE_LEAST, (c.rows * g.cols / c.num_cus + 63) / 64 * 64));
    const int64_t slices = (c.rows + slice - 1) / slice;
    // of up to FEW_ROWS rows where one launch takes longer than two: not of the least, nor where many
    // entries are written twice (300 x 37 to 300 entries 12.0 us, 16.0 by one; 1000 x 1000 to one 12.5
    // and 25.0; 32 x 1024 to 20 10.9 and 9.3; 200 x 512 to 1000 16.4 and 13.6)
    const bool sliced =
        !g.few || (c.rows >= SLICED_FEW && c.entries * c.dim <= SLICED_FEW_ELEMENTS);
    if (sliced && c.rows >= 1 && c.entries < (1 << MOST_BITS) && g.cols <= 4 &&
        slices * c.entries * part_stride(c) * 4 <= SLICE_BYTES) {
        g.few = false;
        g.slices = slices;
        g.whole = (int)slice;
        g.bits = std::max(3, bits);
        g.per = ((slice + SUM_WAVES - 1) / SUM_WAVES + 63) / 64 * 64;
        // 16 rows a worker at least
        g.groups = (int)std::min<int64_t>(64 / g.lanes, (slice + 16 * SUM_WAVES - 1) / (16 * SUM_WAVES));
    }
    return g;
}

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t table_bytes(const GradShape &g) {
    return rounded(g.small ? 0 : ((size_t)g.units << g.bits) * (g.narrow ? 2 : 4));
}

template <int R, typename C>
hipError_t sort_pass(hipStream_t st, const Pass &p) {
    const hipError_t e = allow_all_lds(reinterpret_cast<const void *>(k_embed_place<R, C>));
    if (e != hipSuccess) return e;
    const dim3 grid((uint32_t)p.units), block(SORT_THREADS);
    const size_t lds = 4 * (SORT_WAVES + ((size_t)(2 + SORT_WAVES) << p.bits) + 2 * CHUNK<R>);
    hipLaunchKernelGGL((k_embed_count<R, C>), grid, block, 0, st, p);
    hipLaunchKernelGGL((k_embed_place<R, C>), grid, block, lds, st, p);
    return hipGetLastError();
}

template <typename T, int E, bool BASE, bool ONE>
void sums(hipStream_t st, const Sums &s, int cols) {
    const int64_t each = SUM_WAVES * s.groups;
    const size_t most = (size_t)held_rows((int)each * s.per, s.whole);
    const size_t lds = std::max(sum_lds(s.dense, most), sizeof(float) * SUM_THREADS * E);
    hipLaunchKernelGGL((k_embed_sum<T, E, BASE, ONE>),
                       grid_of((s.workers + each - 1) / each, (uint32_t)cols), dim3(SUM_THREADS), lds,
                       st, s);
}
template <typename T, int E> void sums(hipStream_t st, const Sums &s, int cols) {
    if (s.groups == 1)
        s.base ? sums<T, E, true, true>(st, s, cols) : sums<T, E, false, true>(st, s, cols);
    else
        s.base ? sums<T, E, true, false>(st, s, cols) : sums<T, E, false, false>(st, s, cols);
}
template <typename T>
hipError_t sums(hipStream_t st, const Sums &s, const GradShape &g, int num_cus) {
    constexpr int E = 16 / sizeof(T);
    g.elements > 1 ? sums<T, E>(st, s, g.cols) : sums<T, 1>(st, s, g.cols);
    if (s.rows <= s.whole) return hipGetLastError();     // no entry is parted
    const int turns = (s.part_stride / 4 + 63) / 64;
    hipLaunchKernelGGL((k_embed_join<T>),
                       dim3((uint32_t)(4 * num_cus), (uint32_t)std::min(turns, 16)),
                       dim3(JOIN_THREADS), 0, st, s);
    return hipGetLastError();
}

template <typename T, int E, bool BASE>
hipError_t few(hipStream_t st, const Sums &s, const Pass &p, const GradShape &g) {
    const int64_t longs = s.rows / (s.whole + 1);
    hipLaunchKernelGGL((k_embed_few<T, E, BASE>),
                       dim3((uint32_t)(g.lists + longs), (uint32_t)g.cols), dim3(SUM_THREADS),
                       4 * (size_t)few_layout(s, p.bits, E).all, st, s, p, g.passes,
                       (int32_t)g.lists);
    return hipGetLastError();
}
template <typename T>
hipError_t few(hipStream_t st, const Sums &s, const Pass &p, const GradShape &g) {
    constexpr int E = 16 / sizeof(T);
    if (g.elements > 1) return s.base ? few<T, E, true>(st, s, p, g) : few<T, E, false>(st, s, p, g);
    return s.base ? few<T, 1, true>(st, s, p, g) : few<T, 1, false>(st, s, p, g);
}

template <typename T>
hipError_t slices(hipStream_t st, const Sums &s, const Pass &p, const GradShape &g) {
    constexpr int E = 16 / sizeof(T);
    const dim3 grid((uint32_t)g.slices, (uint32_t)g.cols), block(SUM_THREADS);
    const size_t lds = 4 * (SUM_WAVES + SLICE_WORDS + (size_t)FEW_ROWS / 2 * 3 +
                            std::max((size_t)SUM_WAVES << p.bits, (size_t)SUM_THREADS * g.elements));
    if (g.elements > 1) hipLaunchKernelGGL((k_embed_slice<T, E>), grid, block, lds, st, s, p);
    else hipLaunchKernelGGL((k_embed_slice<T, 1>), grid, block, lds, st, s, p);
    hipLaunchKernelGGL((k_embed_total<T>),
                       dim3(s.entries, (uint32_t)((s.part_stride / 4 + 63) / 64)), block, 0, st, s,
                       (int32_t)g.slices);
    return hipGetLastError();
}

template <typename T>
hipError_t lookup(hipStream_t st, const EmbedCall &c) {
    constexpr int E = 16 / sizeof(T);
    const int32_t chunks = c.dim >= E ? (c.dim + E - 1) / E : c.dim;
    const dim3 g = grid_of((c.rows * chunks + 256 * LOOKUP - 1) / (256 * LOOKUP));
    if (c.dim >= E) hipLaunchKernelGGL((k_embed<T, E>), g, dim3(256), 0, st, c, chunks);
    else hipLaunchKernelGGL((k_embed<T, 1>), g, dim3(256), 0, st, c, chunks);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_embed(hipStream_t s, const EmbedCall &call) {
    EmbedCall c = call;
    c.streamed = c.rows * c.dim * (c.bf16 ? 2 : 4) > STREAMED;
    return c.bf16 ? lookup<__bf16>(s, c) : lookup<float>(s, c);
}

size_t embed_grad_scratch(const EmbedCall &c) {
    const GradShape g = grad_shape(c);
    if (g.few) return 0;
    if (g.slices)
        return rounded(4 * SLICE_WORDS * (size_t)g.slices) +
               4 * (size_t)(g.slices * c.entries) * part_stride(c);
    const size_t rows = rounded((size_t)c.rows * sizeof(uint2));
    return (g.small || g.passes < 2 ? 1 : 2) * rows + table_bytes(g) +
           rounded(4 * (size_t)g.workers) + rounded(8 + 8 * (size_t)g.workers) +
           rounded(8 * (size_t)g.workers * part_stride(c));
}

hipError_t launch_embed_grad(hipStream_t st, const EmbedCall &c, char *scratch) {
    const GradShape g = grad_shape(c);
    char *const scratch0 = scratch;
    const size_t rows = rounded((size_t)c.rows * sizeof(uint2));
    uint2 *pairs[2];
    for (int i = 0; i < (g.small || g.passes < 2 ? 1 : 2); ++i) {
        pairs[i] = reinterpret_cast<uint2 *>(scratch);
        scratch += rows;
    }
    void *table = scratch;
    scratch += table_bytes(g);
    Sums s{};
    s.open = reinterpret_cast<uint32_t *>(scratch);
    scratch += rounded(4 * (size_t)g.workers);
    s.found = reinterpret_cast<uint32_t *>(scratch);
    s.parts = reinterpret_cast<float *>(scratch + rounded(8 + 8 * (size_t)g.workers));
    s.part_stride = part_stride(c);
    Pass p{};
    p.entries = (uint32_t)c.entries;
    p.rows = c.rows;
    p.per = g.per;
    p.units = g.units;
    p.bits = g.bits;
    p.table = table;
    p.zero = s.found;
    s.rows = c.rows;
    s.workers = g.workers;
    s.entries = (uint32_t)c.entries;
    s.dim = c.dim;
    s.chunks = g.chunks;
    s.lanes = g.lanes;
    s.groups = g.groups;
    s.per = g.items;
    s.whole = g.whole;
    s.dense = g.dense;
    // whole lines only: narrower rows' are made whole by the caches (1000 rows to 16M entries of 4 f32
    // 697 us past them, 184 so; 100000 to 2M of 32, lines of 128 bytes, 104 past them and 120)
    s.streamed = g.dense && g.lanes * g.elements * (c.bf16 ? 2 : 4) >= 128 &&
                 c.entries * c.dim * (c.bf16 ? 2 : 4) > STREAMED;
    s.row_stride = c.row_stride;
    s.table_stride = c.table_stride;
    s.scale = c.scale;
    s.dout = c.dout;
    s.base = c.base;
    s.dtable = c.dtable;
    if (g.few) {
        p.ids = c.ids;
        return c.bf16 ? few<__bf16>(st, s, p, g) : few<float>(st, s, p, g);
    }
    if (g.slices) {
        p.ids = c.ids;
        s.open = reinterpret_cast<uint32_t *>(scratch0);
        s.parts = reinterpret_cast<float *>(scratch0 + rounded(4 * SLICE_WORDS * (size_t)g.slices));
        return c.bf16 ? slices<__bf16>(st, s, p, g) : slices<float>(st, s, p, g);
    }
    int to = 0;
    if (g.small) {
        const hipError_t e = allow_all_lds(reinterpret_cast<const void *>(k_embed_sort_small));
        if (e != hipSuccess) return e;
        p.ids = c.ids;
        p.out = pairs[0];
        const size_t lds = 4 * (SMALL_WAVES + ((size_t)SMALL_WAVES << g.bits) + c.rows) + 2 * c.rows;
        hipLaunchKernelGGL(k_embed_sort_small, dim3(1), dim3(SMALL_THREADS), lds, st, p, g.passes);
    } else {
        for (int i = 0; i < g.passes; ++i) {
            to = i & 1;
            p.ids = i == 0 ? c.ids : nullptr;
            if (i > 0) p.in = pairs[to ^ 1];
            p.out = pairs[to];
            p.shift = i * g.bits;
            const hipError_t e = g.each == 4 ? sort_pass<4, uint16_t>(st, p)
                                 : g.narrow  ? sort_pass<8, uint16_t>(st, p)
                                             : sort_pass<8, uint32_t>(st, p);
            if (e != hipSuccess) return e;
        }
    }
    s.sorted = pairs[to];
    return c.bf16 ? sums<__bf16>(st, s, g, c.num_cus) : sums<float>(st, s, g, c.num_cus);
}

}  // namespace mbk
