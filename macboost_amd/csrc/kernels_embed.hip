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

// E elements at p as f32, of which the first n are read; the rest are 0.  E > 1: 16 bytes at an
// address that is a multiple of 16.
template <typename T, int E>
__device__ __forceinline__ void load(const T *p, int n, float (&f)[E]) {
    if constexpr (E > 1) {
        typedef T V __attribute__((ext_vector_type(E)));
        if (n >= E) {
            const V v = *reinterpret_cast<const V *>(p);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = to_f32(v[e]);
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e < n ? to_f32(p[e]) : 0.0f;
}

template <typename T, int E>
__device__ __forceinline__ void store(T *p, int n, const float (&f)[E]) {
    if constexpr (E > 1) {
        typedef T V __attribute__((ext_vector_type(E)));
        if (n >= E) {
            V v;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = (T)f[e];
            *reinterpret_cast<V *>(p) = v;
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e < n) p[e] = (T)f[e];
}

// ---------------------------------------------------------------------------
// The lookup: out[row] = base[row] + scale * table[ids[row]].  A row is `chunks` pieces of E
// elements; a workgroup takes 256 * LOOKUP pieces of all the rows' in their order, LOOKUP a
// thread, so that short rows leave no lane idle and each thread has LOOKUP rows on the way.
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
        store<T, E>(out + row[q] * c.row_stride + col[q], c.dim - col[q], v[q]);
    }
}

// ---------------------------------------------------------------------------
// The gradient.  The rows are sorted by id, stably, by radix; a row that is left out has the
// key `entries`, behind all others.
//
// A pass of the sort by up to 10 bits takes two launches: counts a workgroup, and the
// placement, in which each workgroup sums up the counts before its own (at most 256
// workgroups' of 1024, from L2) and writes runs of 2 to 16 pairs that it has ordered in LDS.
// ---------------------------------------------------------------------------
constexpr int SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64;
constexpr int MOST_UNITS = 256;
constexpr int MOST_BITS = 10;
template <int R> constexpr int CHUNK = SORT_THREADS * R;

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Lanes with this lane's digit, among those that are here.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool here, int bits) {
    uint64_t same = __ballot(here);
    for (int k = 0; k < bits; ++k) {
        const uint64_t ones = __ballot((digit >> k) & 1u);
        same &= (digit >> k) & 1u ? ones : ~ones;
    }
    return same;
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
    const uint32_t *key_in, *row_in;
    uint32_t *key_out, *row_out;
    int64_t rows, per;               // rows a workgroup
    int32_t units, shift, bits;
    uint32_t *table;                 // [workgroup][digit]
    uint32_t *zero;                  // a word that the placement clears
};

__device__ __forceinline__ uint32_t key_at(const Pass &p, int64_t i) {
    return p.ids ? key_of(p.ids, p.entries, i) : p.key_in[i];
}

template <int R>
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
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS)
        p.table[(int64_t)blockIdx.x * bins + d] = count[d];
}

template <int R>
__global__ __launch_bounds__(SORT_THREADS) void k_embed_place(Pass p) {
    extern __shared__ uint32_t lds[];
    const int bins = 1 << p.bits;
    uint32_t *wave_sum = lds;                        // SORT_WAVES
    uint32_t *next = wave_sum + SORT_WAVES;          // [digit] its next place
    uint32_t *first = next + bins;                   // [digit] its first place in the chunk
    uint32_t *key_staged = first + bins;             // [place in the chunk]
    uint32_t *row_staged = key_staged + CHUNK<R>;
    uint32_t *count = row_staged + CHUNK<R>;         // [wave][digit]
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.zero = 0;
    uint32_t all, below = 0;
    for (int d0 = 0; d0 < bins; d0 += SORT_THREADS) {
        const int d = d0 + threadIdx.x;
        uint32_t before = 0, total = 0;
        if (d < bins)
            for (int u0 = 0; u0 < p.units; u0 += 8) {
                uint32_t c[8];
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    c[q] = u0 + q < p.units ? p.table[(int64_t)(u0 + q) * bins + d] : 0;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    total += c[q];
                    if (u0 + q < (int)blockIdx.x) before += c[q];
                }
            }
        const uint32_t at = below + sum_before<SORT_WAVES>(total, wave_sum, all);
        if (d < bins) next[d] = at + before;
        below += all;
    }
    const int64_t a = blockIdx.x * p.per, b = min(p.rows, a + p.per);
    for (int64_t c = a; c < b; c += CHUNK<R>) {
        // wavefront by wavefront, so that equal digits keep their order
        const int64_t w = c + wave * (64 * R);
        uint32_t key[R], row[R], rank[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const int64_t i = w + q * 64 + lane;
            key[q] = i < b ? key_at(p, i) : 0;
            row[q] = i < b ? (p.ids ? (uint32_t)i : p.row_in[i]) : 0;
        }
        for (int d = threadIdx.x; d < SORT_WAVES * bins; d += SORT_THREADS) count[d] = 0;
        __syncthreads();
        uint32_t *mine = count + wave * bins;
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const uint32_t d = (key[q] >> p.shift) & (bins - 1);
            const bool here = w + q * 64 + lane < b;
            const uint64_t same = same_digit(d, here, p.bits);
            const uint32_t r = lanes_below(same);
            rank[q] = here ? mine[d] + r : 0;
            __builtin_amdgcn_wave_barrier();
            if (here && r == 0) mine[d] = rank[q] + (uint32_t)__popcll(same);
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
            if (w + q * 64 + lane >= b) continue;
            const uint32_t d = (key[q] >> p.shift) & (bins - 1);
            const uint32_t at = first[d] + mine[d] + rank[q];
            key_staged[at] = key[q];
            row_staged[at] = row[q];
        }
        __syncthreads();
        for (uint32_t l = threadIdx.x; l < taken; l += SORT_THREADS) {
            const uint32_t k = key_staged[l];
            const uint32_t to = next[(k >> p.shift) & (bins - 1)] + l;
            p.key_out[to] = k;
            p.row_out[to] = row_staged[l];
        }
        __syncthreads();
        for (int d = threadIdx.x; d < bins; d += SORT_THREADS)       // the chunk is behind
            next[d] += d + 1 < bins ? first[d + 1] : taken;
        __syncthreads();
    }
}

// Few rows: the whole sort by one workgroup in one launch.
constexpr int SMALL_WAVES = 16, SMALL_THREADS = 64 * SMALL_WAVES, SMALL_EACH = 16;
constexpr int64_t SMALL_ROWS = SMALL_THREADS * SMALL_EACH;
constexpr int SMALL_BITS = 8;
__global__ __launch_bounds__(SMALL_THREADS) void k_embed_sort_small(Pass p, int32_t passes) {
    extern __shared__ uint32_t lds[];
    const int bins = 1 << p.bits;
    uint32_t *wave_sum = lds;                            // SMALL_WAVES
    uint32_t *count = wave_sum + SMALL_WAVES;            // [wave][digit]
    uint32_t *keys = count + SMALL_WAVES * bins;         // [rows]
    uint16_t *order = reinterpret_cast<uint16_t *>(keys + p.rows);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (threadIdx.x == 0) *p.zero = 0;
    const int a = min((int)p.rows, wave * (int)p.per), b = min((int)p.rows, a + (int)p.per);
    uint32_t key[SMALL_EACH], rank[SMALL_EACH];
    uint16_t row[SMALL_EACH];
#pragma unroll
    for (int q = 0; q < SMALL_EACH; ++q) {
        const int i = a + q * 64 + lane;
        key[q] = i < b ? key_of(p.ids, p.entries, i) : 0;
        row[q] = (uint16_t)i;
    }
    for (int s = 0; s < passes; ++s) {
        const int shift = s * p.bits;
        for (int d = threadIdx.x; d < SMALL_WAVES * bins; d += SMALL_THREADS) count[d] = 0;
        __syncthreads();
        uint32_t *mine = count + wave * bins;
#pragma unroll
        for (int q = 0; q < SMALL_EACH; ++q) {
            if (a + q * 64 >= b) continue;
            const uint32_t d = (key[q] >> shift) & (bins - 1);
            const bool here = a + q * 64 + lane < b;
            const uint64_t same = same_digit(d, here, p.bits);
            const uint32_t r = lanes_below(same);
            rank[q] = here ? mine[d] + r : 0;
            __builtin_amdgcn_wave_barrier();
            if (here && r == 0) mine[d] = rank[q] + (uint32_t)__popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        uint32_t sum = 0, all;                           // bins <= SMALL_THREADS
        const int d = threadIdx.x;
        if (d < bins)
            for (int v = 0; v < SMALL_WAVES; ++v) sum += count[v * bins + d];
        uint32_t at = sum_before<SMALL_WAVES>(sum, wave_sum, all);
        if (d < bins)
            for (int v = 0; v < SMALL_WAVES; ++v) {
                const uint32_t n = count[v * bins + d];
                count[v * bins + d] = at;
                at += n;
            }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < SMALL_EACH; ++q) {
            if (a + q * 64 + lane >= b) continue;
            const uint32_t to = mine[(key[q] >> shift) & (bins - 1)] + rank[q];
            keys[to] = key[q];
            order[to] = row[q];
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < SMALL_EACH; ++q) {
            const int i = a + q * 64 + lane;
            if (i >= b) continue;
            key[q] = keys[i];
            row[q] = order[i];
        }
        __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < SMALL_EACH; ++q) {
        const int i = a + q * 64 + lane;
        if (i >= b) continue;
        p.key_out[i] = key[q];
        p.row_out[i] = row[q];
    }
}

// ---------------------------------------------------------------------------
// The sums.  The sorted rows and the table's entries are merged: entry e comes behind the
// rows of key e.  A worker, `lanes` lanes that hold E columns each, takes `per` items of that
// list: it adds the rows and writes the entries, zeros for those without rows, so that rows and
// entries weigh the same whatever the ids.  (Without entries, where dtable is its own base, the
// list is the rows.)
//
// A worker's end that falls into an entry's rows is put behind them if they are at most SHORT;
// else the entry is longer than a worker: each of its workers leaves its sum in parts, and the
// one in which it ends puts it on the list that k_embed_join works off.  Sums of a worker are
// in the rows' order, those of parts in a fixed order too: the same bits in every run.
// ---------------------------------------------------------------------------
constexpr int SUM_WAVES = 4, SUM_THREADS = 64 * SUM_WAVES;
constexpr int SHORT = 64;            // rows
constexpr int MOST_ITEMS = 4096;     // of a workgroup
constexpr int AHEAD = 8;             // rows on the way

struct Sums {
    int64_t rows, workers;
    uint32_t entries;
    int32_t dim, chunks;             // pieces of E columns
    int32_t lanes, groups;           // of a worker; workers a wavefront
    int32_t per;
    bool dense;                      // entries without rows are written
    int64_t row_stride, table_stride;
    float scale;
    const uint32_t *key, *row;
    const void *dout, *base;
    void *dtable;
    float *parts;                    // [worker][head, tail][dim]
    uint32_t *found;                 // [0]: how many; then (worker, entry)
};

// Rows of the sorted list and entries before an item of the merged one, in which row i of key
// k lies at i + k.  i counts from the first row that the workgroup holds in LDS.
struct Cut {
    int i;
    uint32_t e;
    bool open;                       // e's rows begin before i, and there are more than SHORT
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
    const int a = first_not(max(0, c.i - SHORT - 1), c.i, [&](int m) { return key[m] < c.e; });
    const int b = first_not(c.i, min(held, c.i + SHORT + 1),
                            [&](int m) { return key[m] <= c.e; });
    if (b - a <= SHORT) {
        c.i = b;
        c.e += 1;
        c.open = false;
    }
    return c;
}

template <typename T, int E>
__global__ __launch_bounds__(SUM_THREADS) void k_embed_sum(Sums s) {
    extern __shared__ uint32_t lds[];
    __shared__ int64_t ends[2];
    const int64_t first = (int64_t)group_id() * (SUM_WAVES * s.groups);
    if (first >= s.workers) return;
    // the rows of the workgroup's items: 256-ary search for both ends
    const int64_t d0 = first * s.per;
    const int64_t d1 = min(min(first + SUM_WAVES * s.groups, s.workers) * s.per,
                           s.rows + (s.dense ? (int64_t)s.entries : 0));
    if (!s.dense) {
        if (threadIdx.x < 2) ends[threadIdx.x] = threadIdx.x ? d1 : d0;
    } else {
        for (int side = 0; side < 2; ++side) {
            const int64_t d = side ? d1 : d0;
            int64_t lo = max((int64_t)0, d - (int64_t)s.entries), hi = min(s.rows, d);
            while (hi > lo) {                            // the answer is in [lo, hi]
                const int64_t step = (hi - lo + SUM_THREADS - 1) / SUM_THREADS;
                const int64_t m = lo + threadIdx.x * step;
                const bool under = m < hi && m + (int64_t)s.key[m] < d;
                const int n = __syncthreads_count(under);
                if (n == 0) {
                    hi = lo;
                    break;
                }
                const int64_t last = lo + (n - 1) * step;
                lo = last + 1;
                hi = min(hi, last + step);
            }
            if (threadIdx.x == 0) ends[side] = lo;
        }
    }
    __syncthreads();
    const int64_t lo = ends[0], hi = ends[1];
    const int64_t begin = max((int64_t)0, lo - SHORT - 1), end = min(s.rows, hi + SHORT + 1);
    uint32_t *key = lds;
    uint32_t *row = lds + (SUM_WAVES * s.groups * s.per + 2 * SHORT + 2);
    for (int64_t i = begin + threadIdx.x; i < end; i += SUM_THREADS) {
        key[i - begin] = s.key[i];
        row[i - begin] = s.row[i];
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, group = lane / s.lanes;
    const int64_t worker = first + (threadIdx.x >> 6) * s.groups + group;
    const int32_t chunk = blockIdx.y * 64 + lane - group * s.lanes;
    if (group >= s.groups || worker >= s.workers || chunk >= s.chunks) return;
    const int held = (int)(end - begin), from_lo = (int)(lo - begin), to_hi = (int)(hi - begin);
    const Cut from = cut_at(s, key, begin, held, from_lo, to_hi, worker * s.per);
    const Cut to = cut_at(s, key, begin, held, from_lo, to_hi, (worker + 1) * s.per);
    const int col = chunk * E, n = s.dim - col;
    const T *dout = static_cast<const T *>(s.dout) + col;
    const T *base = static_cast<const T *>(s.base);
    T *dtable = static_cast<T *>(s.dtable) + col;
    if (base) base += col;

    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    uint32_t next = from.e;          // the next entry to write
    bool has = from.open, head = from.open;
    // Writes entry e = base + scale * acc.
    const auto write = [&](uint32_t e) {
        float v[E], b[E];
#pragma unroll
        for (int x = 0; x < E; ++x) b[x] = 0.0f;
        if (base) load<T, E>(base + (int64_t)e * s.table_stride, n, b);
#pragma unroll
        for (int x = 0; x < E; ++x) v[x] = __builtin_fmaf(s.scale, acc[x], b[x]);
        store<T, E>(dtable + (int64_t)e * s.table_stride, n, v);
    };
    const auto leave = [&](int side) {
        float *p = s.parts + (worker * 2 + side) * s.dim + col;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < n) p[e] = acc[e];
    };
    // The entry `next`, whose rows are all added.
    const auto finish = [&]() {
        if (head) {
            leave(0);
            if (chunk == 0) {
                const uint32_t at = atomicAdd(&s.found[0], 1u);
                s.found[2 + 2 * at] = (uint32_t)worker;
                s.found[3 + 2 * at] = next;
            }
            head = false;
        } else {
            write(next);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.0f;
        has = false;
        ++next;
    };
    for (int i = from.i; i < to.i; i += AHEAD) {
        float v[AHEAD][E];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const bool here = i + q < to.i && key[i + q] < s.entries;
            load<T, E>(dout + (here ? row[i + q] * s.row_stride : 0), here ? n : 0, v[q]);
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            if (i + q >= to.i) break;
            const uint32_t k = key[i + q];
            if (k >= s.entries) break;                   // left out, as are all behind
            if (k != next || !has) {
                if (has) finish();
                if (s.dense)
                    while (next < k) finish();
                next = k;
                has = true;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += v[q][e];
        }
    }
    if (to.open && (has ? next : from.e) == to.e) {
        leave(1);
        return;
    }
    if (has) finish();
    if (s.dense)
        while (next < to.e) finish();
}

// The entries on the list: heads and tails of their workers.  A workgroup an entry; slices of
// its workers are summed side by side, and the slices' sums in their order.
constexpr int JOIN_WAVES = 8, JOIN_THREADS = 64 * JOIN_WAVES;
template <typename T>
__global__ __launch_bounds__(JOIN_THREADS) void k_embed_join(Sums s) {
    __shared__ float sums[JOIN_THREADS];
    const uint32_t count = s.found[0];
    const int wide = min(s.dim, 64), groups = 64 / wide, slices = JOIN_WAVES * groups;
    const int lane = threadIdx.x & 63, group = lane / wide;
    const int slice = (threadIdx.x >> 6) * groups + group, col0 = lane - group * wide;
    for (uint32_t f = blockIdx.x; f < count; f += gridDim.x) {
        const int64_t last = s.found[2 + 2 * f];
        const uint32_t entry = s.found[3 + 2 * f];
        int64_t lo = 0, hi = s.rows;                     // the entry's first row
        while (hi > lo) {
            const int64_t step = (hi - lo + JOIN_THREADS - 1) / JOIN_THREADS;
            const int64_t m = lo + threadIdx.x * step;
            const int n = __syncthreads_count(m < hi && s.key[m] < entry);
            if (n == 0) break;
            const int64_t at = lo + (n - 1) * step;
            lo = at + 1;
            hi = min(hi, at + step);
        }
        const int64_t start = (lo + (s.dense ? (int64_t)entry : 0)) / s.per;
        const int64_t each = (last - start + slices) / slices;      // of last - start + 1 parts
        const int64_t a = start + slice * each, b = min(a + each, last + 1);
        for (int c0 = 0; c0 < s.dim; c0 += wide) {
            const int col = c0 + col0;
            float sum = 0.0f;
            if (group < groups && col < s.dim)
                for (int64_t w = a; w < b; w += AHEAD) {
                    float v[AHEAD];
#pragma unroll
                    for (int q = 0; q < AHEAD; ++q)
                        v[q] = w + q < b
                                   ? s.parts[((w + q) * 2 + (w + q < last)) * s.dim + col] : 0.0f;
#pragma unroll
                    for (int q = 0; q < AHEAD; ++q) sum += v[q];
                }
            sums[threadIdx.x] = sum;
            __syncthreads();
            if (threadIdx.x < (unsigned)wide && col < s.dim) {
                float total = 0.0f;
                for (int v = 0; v < slices; ++v)
                    total += sums[(v / groups) * 64 + (v % groups) * wide + col0];
                T *to = static_cast<T *>(s.dtable) + (int64_t)entry * s.table_stride + col;
                const float b0 = s.base ? to_f32(static_cast<const T *>(
                                              s.base)[(int64_t)entry * s.table_stride + col])
                                        : 0.0f;
                *to = (T)__builtin_fmaf(s.scale, total, b0);
            }
            __syncthreads();
        }
    }
}

bool aligned(const void *p, int64_t stride, size_t size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * (int64_t)size % 16 == 0;
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
    int lanes, groups, cols, items, chunks;
    int elements;                    // E
    bool dense;
    int64_t workers;
};

GradShape grad_shape(const EmbedCall &c) {
    GradShape g{};
    const int bits = bits_of(c.entries);
    g.small = c.rows <= SMALL_ROWS;
    const int most = g.small ? SMALL_BITS : MOST_BITS;
    g.passes = (bits + most - 1) / most;
    g.bits = (bits + g.passes - 1) / g.passes;
    if (g.small) {
        g.per = ((c.rows + SMALL_WAVES - 1) / SMALL_WAVES + 63) / 64 * 64;
        g.units = 1;
    } else {
        g.each = c.rows <= (int64_t)MOST_UNITS * CHUNK<4> ? 4 : 8;
        const int64_t chunk = (int64_t)SORT_THREADS * g.each;
        const int64_t chunks = (c.rows + chunk - 1) / chunk;
        g.per = (chunks + MOST_UNITS - 1) / MOST_UNITS * chunk;
        g.units = (int)((c.rows + g.per - 1) / g.per);
    }
    const size_t size = c.bf16 ? 2 : 4;
    const bool wide = aligned(c.dout, c.row_stride, size) && aligned(c.dtable, c.table_stride, size) &&
                      (!c.base || aligned(c.base, c.table_stride, size));
    g.elements = wide ? (c.bf16 ? 8 : 4) : 1;
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
    g.items = (int)per;
    g.workers = (items + per - 1) / per;
    return g;
}

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

template <typename T, int E>
hipError_t sums(hipStream_t st, const Sums &s, int cols, int num_cus) {
    const int64_t each = SUM_WAVES * s.groups;
    dim3 g = grid_of((s.workers + each - 1) / each, (uint32_t)cols);
    const size_t lds = 2 * sizeof(uint32_t) * (each * s.per + 2 * SHORT + 2);
    hipLaunchKernelGGL((k_embed_sum<T, E>), g, dim3(SUM_THREADS), lds, st, s);
    hipLaunchKernelGGL((k_embed_join<T>), dim3((uint32_t)(2 * num_cus)), dim3(JOIN_THREADS), 0, st,
                       s);
    return hipGetLastError();
}

template <typename T>
hipError_t lookup(hipStream_t st, const EmbedCall &c) {
    constexpr int E = 16 / sizeof(T);
    const bool wide = aligned(c.table, c.table_stride, sizeof(T)) &&
                      aligned(c.out, c.row_stride, sizeof(T)) &&
                      (!c.base || aligned(c.base, c.row_stride, sizeof(T)));
    const int32_t chunks = wide ? (c.dim + E - 1) / E : c.dim;
    const dim3 g = grid_of((c.rows * chunks + 256 * LOOKUP - 1) / (256 * LOOKUP));
    if (wide) hipLaunchKernelGGL((k_embed<T, E>), g, dim3(256), 0, st, c, chunks);
    else hipLaunchKernelGGL((k_embed<T, 1>), g, dim3(256), 0, st, c, chunks);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_embed(hipStream_t s, const EmbedCall &c) {
    return c.bf16 ? lookup<__bf16>(s, c) : lookup<float>(s, c);
}

size_t embed_grad_scratch(const EmbedCall &c) {
    const GradShape g = grad_shape(c);
    const size_t rows = rounded((size_t)c.rows * 4);
    return (g.small || g.passes < 2 ? 2 : 4) * rows +
           rounded(g.small ? 0 : ((size_t)g.units << g.bits) * 4) + rounded(8 + 8 * (size_t)g.workers) +
           rounded(8 * (size_t)g.workers * c.dim);
}

hipError_t launch_embed_grad(hipStream_t st, const EmbedCall &c, char *scratch) {
    const GradShape g = grad_shape(c);
    const size_t rows = rounded((size_t)c.rows * 4);
    uint32_t *key[2], *row[2];
    const int sides = g.small || g.passes < 2 ? 1 : 2;
    for (int i = 0; i < sides; ++i) {
        key[i] = reinterpret_cast<uint32_t *>(scratch);
        row[i] = reinterpret_cast<uint32_t *>(scratch + rows);
        scratch += 2 * rows;
    }
    uint32_t *table = reinterpret_cast<uint32_t *>(scratch);
    scratch += rounded(g.small ? 0 : ((size_t)g.units << g.bits) * 4);
    Sums s{};
    s.found = reinterpret_cast<uint32_t *>(scratch);
    s.parts = reinterpret_cast<float *>(scratch + rounded(8 + 8 * (size_t)g.workers));
    Pass p{};
    p.entries = (uint32_t)c.entries;
    p.rows = c.rows;
    p.per = g.per;
    p.units = g.units;
    p.bits = g.bits;
    p.table = table;
    p.zero = s.found;
    int to = 0;
    if (g.small) {
        const hipError_t e = allow_all_lds(reinterpret_cast<const void *>(k_embed_sort_small));
        if (e != hipSuccess) return e;
        p.ids = c.ids;
        p.key_out = key[0];
        p.row_out = row[0];
        const size_t lds = 4 * (SMALL_WAVES + ((size_t)SMALL_WAVES << g.bits) + c.rows) + 2 * c.rows;
        hipLaunchKernelGGL(k_embed_sort_small, dim3(1), dim3(SMALL_THREADS), lds, st, p, g.passes);
    } else {
        for (const void *f : {reinterpret_cast<const void *>(k_embed_place<4>),
                              reinterpret_cast<const void *>(k_embed_place<8>)}) {
            const hipError_t e = allow_all_lds(f);
            if (e != hipSuccess) return e;
        }
        const dim3 grid((uint32_t)g.units), block(SORT_THREADS);
        const size_t lds = 4 * (SORT_WAVES + ((size_t)(2 + SORT_WAVES) << g.bits) +
                                2 * (size_t)SORT_THREADS * g.each);
        for (int i = 0; i < g.passes; ++i) {
            to = i & 1;
            p.ids = i == 0 ? c.ids : nullptr;
            if (i > 0) {
                p.key_in = key[to ^ 1];
                p.row_in = row[to ^ 1];
            }
            p.key_out = key[to];
            p.row_out = row[to];
            p.shift = i * g.bits;
            if (g.each == 4) {
                hipLaunchKernelGGL(k_embed_count<4>, grid, block, 0, st, p);
                hipLaunchKernelGGL(k_embed_place<4>, grid, block, lds, st, p);
            } else {
                hipLaunchKernelGGL(k_embed_count<8>, grid, block, 0, st, p);
                hipLaunchKernelGGL(k_embed_place<8>, grid, block, lds, st, p);
            }
        }
    }
    s.rows = c.rows;
    s.workers = g.workers;
    s.entries = (uint32_t)c.entries;
    s.dim = c.dim;
    s.chunks = g.chunks;
    s.lanes = g.lanes;
    s.groups = g.groups;
    s.per = g.items;
    s.dense = g.dense;
    s.row_stride = c.row_stride;
    s.table_stride = c.table_stride;
    s.scale = c.scale;
    s.key = key[to];
    s.row = row[to];
    s.dout = c.dout;
    s.base = c.base;
    s.dtable = c.dtable;
    if (c.bf16)
        return g.elements > 1 ? sums<__bf16, 8>(st, s, g.cols, c.num_cus)
                              : sums<__bf16, 1>(st, s, g.cols, c.num_cus);
    return g.elements > 1 ? sums<float, 4>(st, s, g.cols, c.num_cus)
                          : sums<float, 1>(st, s, g.cols, c.num_cus);
}

}  // namespace mbk
