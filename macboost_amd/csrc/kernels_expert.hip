// kernels_expert.hip — rows sorted by expert and back (mbk_expert_*): a stable
// counting sort of the assignments by expert, the rows' features in that order,
// the experts' outputs summed back for each row, and the gradient of that sum.
// All of them move data; none has work worth counting.
#include <algorithm>

#include "grid.hpp"
#include "mbk.h"
#include "ops.h"

namespace mbk {

namespace {

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

// ---------------------------------------------------------------------------
// The sort.  Wavefront u owns the assignments [u * per, (u + 1) * per): it
// counts them by expert, the counts are summed over the wavefronts before it
// and the experts below, and it then hands out slots in ascending order: every
// step is ordered, so the sort is stable and needs no atomic on global memory.
// Counters of one wavefront lie in LDS.  Keys are loaded AHEAD at a time, since one at a
// time waits for memory.
// ---------------------------------------------------------------------------
constexpr int SORT_WAVES = 4;
constexpr int AHEAD = 8;

// Workgroups go to the 8 XCDs in turn; each XCD gets a run of them, so that neighbours'
// writes to one list meet in one L2.
__device__ __forceinline__ uint32_t run_of(uint32_t id, uint32_t total) {
    const uint32_t xcd = id & 7, per = total >> 3, more = total & 7;
    return xcd * per + min(xcd, more) + (id >> 3);
}

// Keys [a, b) in their order, 64 at a time: take(first index, key), -1 behind the end.
template <class Take>
__device__ __forceinline__ void each_key(const int32_t *__restrict__ expert, int64_t a, int64_t b,
                                         Take take) {
    const int lane = threadIdx.x & 63;
    int32_t ahead[AHEAD];
    const auto load = [&](int64_t i0) {
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const int64_t i = i0 + q * 64 + lane;
            ahead[q] = i < b ? expert[i] : -1;
        }
    };
    if (a < b) load(a);
    for (int64_t i0 = a; i0 < b; i0 += 64 * AHEAD) {
        int32_t now[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) now[q] = ahead[q];
        if (i0 + 64 * AHEAD < b) load(i0 + 64 * AHEAD);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
            if (i0 + q * 64 < b) take(i0 + q * 64, (uint32_t)now[q]);
    }
}

__device__ __forceinline__ void count_keys(const int32_t *__restrict__ expert, int64_t a, int64_t b,
                                           int32_t experts, uint32_t *count) {
    each_key(expert, a, b, [&](int64_t, uint32_t e) {
        if (e < (uint32_t)experts) atomicAdd(&count[e], 1u);
    });
}

// next[e]: the slot that the wavefront's next assignment to e gets.  Lanes with nothing to
// write write to trash: with stores under a branch the loads ahead would wait for all
// of them to be done.
__device__ __forceinline__ void place_keys(const int32_t *__restrict__ expert, int64_t a, int64_t b,
                                           int32_t experts, int32_t key_bits, uint32_t *next,
                                           int32_t *__restrict__ source,
                                           int32_t *__restrict__ slot, int32_t *trash) {
    const int lane = threadIdx.x & 63;
    each_key(expert, a, b, [&](int64_t i0, uint32_t e) {
        const int64_t i = i0 + lane;
        const bool kept = e < (uint32_t)experts;
        uint64_t same = __ballot(kept);         // lanes with this lane's expert
        for (int k = 0; k < key_bits; ++k) {
            const uint64_t ones = __ballot((e >> k) & 1u);
            same &= (e >> k) & 1u ? ones : ~ones;
        }
        const uint32_t rank = lanes_below(same);
        uint32_t at = 0;
        if (kept) at = next[e] + rank;
        __builtin_amdgcn_wave_barrier();
        if (kept && rank == 0) next[e] = at + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        *(kept ? source + at : trash) = (int32_t)i;
        *(i < b ? slot + i : trash) = kept ? (int32_t)at : -1;
    });
}
// source of [a, b) behind the last slot taken.
__device__ __forceinline__ void no_source(int64_t a, int64_t b, int64_t kept,
                                          int32_t *__restrict__ source) {
    for (int64_t i = max(a, kept) + (threadIdx.x & 63); i < b; i += 64) source[i] = -1;
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

// table[e * units + u]: assignments of wavefront u to expert e.
__global__ __launch_bounds__(64 * SORT_WAVES) void k_expert_count(
    const int32_t *__restrict__ expert, int64_t slots, int32_t experts, int64_t per, int32_t units,
    uint32_t *__restrict__ table) {
    extern __shared__ uint32_t lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t *count = lds + (size_t)wave * experts;
    const int32_t u = run_of(blockIdx.x, gridDim.x) * SORT_WAVES + wave;
    for (int e = lane; e < experts; e += 64) count[e] = 0;
    __syncthreads();
    if (u < units) count_keys(expert, u * per, min(slots, (u + 1) * per), experts, count);
    __syncthreads();
    if (u < units)
        for (int e = lane; e < experts; e += 64) table[(int64_t)e * units + u] = count[e];
}

// A workgroup an expert: its counts become sums over the wavefronts before, total[e] their
// sum.  Up to 8 wavefronts' counts a thread.
constexpr int SCAN = 256, SCAN_EACH = 8;
__global__ __launch_bounds__(SCAN) void k_expert_scan(uint32_t *__restrict__ table, int32_t units,
                                                      uint32_t *__restrict__ total) {
    __shared__ uint32_t wave_sum[SCAN / 64];
    uint32_t *row = table + (int64_t)blockIdx.x * units;
    const int u0 = threadIdx.x * SCAN_EACH;
    uint32_t c[SCAN_EACH], sum = 0, all;
#pragma unroll
    for (int q = 0; q < SCAN_EACH; ++q) c[q] = u0 + q < units ? row[u0 + q] : 0;
#pragma unroll
    for (int q = 0; q < SCAN_EACH; ++q) sum += c[q];
    uint32_t before = sum_before<SCAN / 64>(sum, wave_sum, all);
#pragma unroll
    for (int q = 0; q < SCAN_EACH; ++q) {
        if (u0 + q < units) row[u0 + q] = before;
        before += c[q];
    }
    if (threadIdx.x == 0) total[blockIdx.x] = all;
}

// offsets[e] = assignments to experts below e, by one workgroup.
__global__ __launch_bounds__(1024) void k_expert_offsets(const uint32_t *__restrict__ total,
                                                         int32_t experts,
                                                         int32_t *__restrict__ offsets) {
    __shared__ uint32_t wave_sum[16];
    uint32_t before = 0, all;
    for (int e0 = 0; e0 < experts; e0 += 1024) {
        const int e = e0 + threadIdx.x;
        const uint32_t below = sum_before<16>(e < experts ? total[e] : 0, wave_sum, all);
        if (e < experts) offsets[e] = (int32_t)(before + below);
        before += all;
    }
    if (threadIdx.x == 0) offsets[experts] = (int32_t)before;
}

__global__ __launch_bounds__(64 * SORT_WAVES) void k_expert_place(
    const int32_t *__restrict__ expert, int64_t slots, int32_t experts, int32_t key_bits,
    int64_t per, int32_t units, const uint32_t *__restrict__ table,
    const int32_t *__restrict__ offsets, int32_t *__restrict__ source,
    int32_t *__restrict__ slot, int32_t *trash) {
    extern __shared__ uint32_t lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t *next = lds + (size_t)wave * experts;
    const int32_t u = run_of(blockIdx.x, gridDim.x) * SORT_WAVES + wave;
    if (u >= units) return;                     // no barrier below
    for (int e = lane; e < experts; e += 64)
        next[e] = (uint32_t)offsets[e] + table[(int64_t)e * units + u];
    const int64_t a = u * per, b = min(slots, a + per);
    place_keys(expert, a, b, experts, key_bits, next, source, slot, trash);
    no_source(a, b, offsets[experts], source);
}

// Up to CHUNK_EXPERTS experts (their counters of eight wavefronts fit LDS beside the chunk;
// 10M assignments to 2048 145 us, 188 by wavefronts; to 1024 83 and 164): a workgroup takes
// chunks of assignments, orders each in LDS by (expert, assignment) and writes source from
// there, in runs.  (10M assignments to
// 1000 experts: with a wavefront a unit and single writes 88 us, 304 MB written for 80:
// the part of source that an XCD writes at once does not fit its L2.)
// R times 64 assignments a wavefront: 16, or 4 where that would leave most CUs idle (131k
// assignments to 64 experts: 18 us by 16 workgroups, 10 by 64).
constexpr int CHUNK_WAVES = 8;
template <int R> constexpr int CHUNK = R * CHUNK_WAVES * 64;
// (1M assignments to 64 experts: 24 us by 16, 18 by 4; 4M to 1000: 41 and 61.)
constexpr int64_t FEW_SLOTS = (int64_t)1 << 20;
constexpr int32_t CHUNK_EXPERTS = 2048;
// Counters a place kernel sums up by itself, without the two kernels that scan them, and the
// experts whose sums its wavefronts can take one after another (131k assignments: 4 experts
// 14 us, 20 with the scan, 128 18 and 20; 256 27 and 20; 20k to 512 46 and 20).
constexpr int64_t DIRECT_COUNTERS = 8192;
constexpr int32_t DIRECT_EXPERTS = 128;

// table[e * units + u]: assignments of workgroup u to expert e.
template <int R>
__global__ __launch_bounds__(64 * CHUNK_WAVES) void k_expert_count_chunks(
    const int32_t *__restrict__ expert, int64_t slots, int32_t experts, int64_t per, int32_t units,
    uint32_t *__restrict__ table) {
    extern __shared__ uint32_t count[];
    const int32_t u = run_of(blockIdx.x, gridDim.x);
    for (int e = threadIdx.x; e < experts; e += 64 * CHUNK_WAVES) count[e] = 0;
    __syncthreads();
    const int64_t b = min(slots, (u + 1) * per);
    for (int64_t a = u * per; a < b; a += CHUNK<R>) {
        const int64_t w = a + (threadIdx.x >> 6) * (64 * R);
        int32_t key[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const int64_t i = w + q * 64 + (threadIdx.x & 63);
            key[q] = i < b ? expert[i] : -1;
        }
#pragma unroll
        for (int q = 0; q < R; ++q)
            if ((uint32_t)key[q] < (uint32_t)experts) atomicAdd(&count[key[q]], 1u);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += 64 * CHUNK_WAVES)
        table[(int64_t)e * units + u] = count[e];
}

// DIRECT: the table holds counts, and workgroup 0 writes the offsets; else sums over the
// workgroups before, and the offsets are there.
template <int R, bool DIRECT>
__global__ __launch_bounds__(64 * CHUNK_WAVES) void k_expert_place_chunks(
    const int32_t *__restrict__ expert, int64_t slots, int32_t experts, int32_t key_bits,
    int64_t per, int32_t units, const uint32_t *__restrict__ table,
    int32_t *__restrict__ offsets, int32_t *__restrict__ source, int32_t *__restrict__ slot) {
    extern __shared__ uint32_t lds[];
    constexpr int THREADS = 64 * CHUNK_WAVES;
    uint32_t *wave_sum = lds;                        // CHUNK_WAVES
    uint32_t *next = wave_sum + CHUNK_WAVES;         // [expert] its next slot
    uint32_t *first = next + experts;                // [expert] its first place in the chunk
    uint32_t *staged = first + experts;              // [place] expert << 13 | assignment
    uint32_t *count = staged + CHUNK<R>;                // [wave][expert]
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int32_t u = run_of(blockIdx.x, gridDim.x);
    uint32_t kept_all, all;
    if constexpr (DIRECT) {
        // first: all of an expert's assignments; next: those before this workgroup's
        for (int e = wave; e < experts; e += CHUNK_WAVES) {
            uint32_t before = 0, sum = 0;
            for (int v = lane; v < units; v += 64) {
                const uint32_t c = table[(int64_t)e * units + v];
                sum += c;
                if (v < u) before += c;
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                sum += __shfl_xor(sum, o, 64);
                before += __shfl_xor(before, o, 64);
            }
            if (lane == 0) {
                first[e] = sum;
                next[e] = before;
            }
        }
        __syncthreads();
        uint32_t below = 0;
        for (int e0 = 0; e0 < experts; e0 += THREADS) {
            const int e = e0 + threadIdx.x;
            const uint32_t at =
                below + sum_before<CHUNK_WAVES>(e < experts ? first[e] : 0, wave_sum, all);
            if (e < experts) {
                next[e] += at;
                if (u == 0) offsets[e] = (int32_t)at;
            }
            below += all;
        }
        if (u == 0 && threadIdx.x == 0) offsets[experts] = (int32_t)below;
        kept_all = below;
    } else {
        for (int e = threadIdx.x; e < experts; e += THREADS)
            next[e] = (uint32_t)offsets[e] + table[(int64_t)e * units + u];
        kept_all = (uint32_t)offsets[experts];
    }
    const int64_t b = min(slots, (u + 1) * per);
    for (int64_t a = u * per; a < b; a += CHUNK<R>) {
        const int64_t w = a + wave * (64 * R);
        int32_t key[R];
        uint32_t rank[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const int64_t i = w + q * 64 + lane;
            key[q] = i < b ? expert[i] : -1;
        }
        for (int e = threadIdx.x; e < CHUNK_WAVES * experts; e += THREADS) count[e] = 0;
        __syncthreads();
        uint32_t *mine = count + wave * experts;
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const uint32_t e = (uint32_t)key[q];
            const bool kept = e < (uint32_t)experts;
            uint64_t same = __ballot(kept);          // lanes with this lane's expert
            for (int k = 0; k < key_bits; ++k) {
                const uint64_t ones = __ballot((e >> k) & 1u);
                same &= (e >> k) & 1u ? ones : ~ones;
            }
            const uint32_t r = lanes_below(same);
            rank[q] = kept ? mine[e] + r : 0;
            __builtin_amdgcn_wave_barrier();
            if (kept && r == 0) mine[e] = rank[q] + (uint32_t)__popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        // counts become sums over the wavefronts before, first the place of each expert,
        // next the slot that goes with place 0
        uint32_t taken = 0;
        for (int e0 = 0; e0 < experts; e0 += THREADS) {
            const int e = e0 + threadIdx.x;
            uint32_t sum = 0;
            if (e < experts)
#pragma unroll
                for (int v = 0; v < CHUNK_WAVES; ++v) {
                    const uint32_t c = count[v * experts + e];
                    count[v * experts + e] = sum;
                    sum += c;
                }
            const uint32_t at = taken + sum_before<CHUNK_WAVES>(sum, wave_sum, all);
            if (e < experts) {
                first[e] = at;
                next[e] -= at;
            }
            taken += all;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const int64_t i = w + q * 64 + lane;
            if (i >= b) continue;
            const uint32_t e = (uint32_t)key[q];
            int32_t s = -1;
            if (e < (uint32_t)experts) {
                const uint32_t at = first[e] + mine[e] + rank[q];
                staged[at] = e << 13 | (uint32_t)(i - a);
                s = (int32_t)(next[e] + at);
            }
            slot[i] = s;
        }
        __syncthreads();
        for (uint32_t l = threadIdx.x; l < taken; l += THREADS) {
            const uint32_t v = staged[l];
            source[next[v >> 13] + l] = (int32_t)(a + (v & (CHUNK<R> - 1)));
        }
        __syncthreads();
        // the chunk's assignments are behind
        for (int e0 = 0; e0 < experts; e0 += THREADS) {
            const int e = e0 + threadIdx.x;
            if (e < experts) next[e] += e + 1 < experts ? first[e + 1] : taken;
        }
        __syncthreads();
    }
    for (int64_t i = max(u * per, (int64_t)kept_all) + threadIdx.x; i < b; i += THREADS)
        source[i] = -1;                              // behind the last slot taken
}

// Few assignments: the whole sort by one workgroup, in one launch (4096 to 1000 experts 10
// us, 19 by the kernels above; at 16384 to 4 15 and 16, at 32768 26 and 14).  Counters of its
// wavefronts fit LDS up to 2048 experts.
constexpr int SMALL_WAVES = 16;
constexpr int64_t SMALL_SLOTS = 16384;
constexpr int32_t SMALL_EXPERTS = 2048;
__global__ __launch_bounds__(64 * SMALL_WAVES) void k_expert_sort_small(
    const int32_t *__restrict__ expert, int64_t slots, int32_t experts, int32_t key_bits,
    int64_t per, int32_t *__restrict__ offsets, int32_t *__restrict__ source,
    int32_t *__restrict__ slot, int32_t *trash) {
    extern __shared__ uint32_t lds[];
    uint32_t *wave_sum = lds, *count = lds + SMALL_WAVES;        // [wave][expert]
    const int wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < SMALL_WAVES * experts; e += 64 * SMALL_WAVES) count[e] = 0;
    __syncthreads();
    const int64_t a = min(slots, wave * per), b = min(slots, a + per);
    count_keys(expert, a, b, experts, count + wave * experts);
    __syncthreads();
    uint32_t before = 0, all;
    for (int e0 = 0; e0 < experts; e0 += 64 * SMALL_WAVES) {
        const int e = e0 + threadIdx.x;
        uint32_t sum = 0;
        if (e < experts)
            for (int w = 0; w < SMALL_WAVES; ++w) sum += count[w * experts + e];
        uint32_t at = before + sum_before<SMALL_WAVES>(sum, wave_sum, all);
        if (e < experts) {
            offsets[e] = (int32_t)at;
            for (int w = 0; w < SMALL_WAVES; ++w) {
                const uint32_t c = count[w * experts + e];
                count[w * experts + e] = at;
                at += c;
            }
        }
        before += all;
    }
    if (threadIdx.x == 0) offsets[experts] = (int32_t)before;
    __syncthreads();
    place_keys(expert, a, b, experts, key_bits, count + wave * experts, source, slot, trash);
    no_source(a, b, before, source);
}

struct SortShape {
    int64_t per;
    int32_t units;
};
// At least 1024 assignments a wavefront, at most 8 wavefronts a CU (a thread of the scan
// takes eight) and 4M counters.
SortShape sort_shape(const ExpertPlan &p, int num_cus) {
    const int64_t slots = p.rows * p.k;
    int64_t units = std::min<int64_t>((slots + 1023) / 1024,
                                      std::min<int64_t>(8 * (int64_t)num_cus, SCAN * SCAN_EACH));
    units = std::max<int64_t>(1, std::min<int64_t>(units, ((int64_t)4 << 20) / p.experts));
    const int64_t per = std::max<int64_t>(64, ((slots + units - 1) / units + 63) / 64 * 64);
    return {per, (int32_t)std::max<int64_t>(1, (slots + per - 1) / per)};
}

// ---------------------------------------------------------------------------
// Moving rows.  Assignment a of slot s lies in the sorted matrix at
// base + f * step: [slots][cols] has base s * cols and step 1, blocks (the
// expert's [cols][n_e] at cols * offsets[e]) have base cols * offsets[e] + s -
// offsets[e] and step n_e.
// ---------------------------------------------------------------------------
struct Place {
    int64_t base;                // -1: dropped
    int64_t step;
};
__device__ __forceinline__ Place place_of(const ExpertPlan &p, int64_t a, int32_t cols,
                                          bool blocked) {
    const int32_t s = p.slot[a];
    if (s < 0) return {-1, 0};
    if (!blocked) return {(int64_t)s * cols, 1};
    const int32_t e = p.expert[a];
    const int32_t first = p.offsets[e];
    return {(int64_t)first * cols + (s - first), p.offsets[e + 1] - first};
}

// ---- both matrices by rows: L lanes a row, B bytes a lane ----
template <int B> struct Bytes;
template <> struct Bytes<16> { typedef __attribute__((ext_vector_type(4))) uint32_t type; };
template <> struct Bytes<4> { typedef uint32_t type; };
template <> struct Bytes<2> { typedef uint16_t type; };

// Row and chunks of a lane: rows_of(256 / lanes a workgroup).
struct RowLanes {
    int64_t row;
    int lane, lanes;
};
__device__ __forceinline__ RowLanes row_lanes(int log2_lanes) {
    const int lanes = 1 << log2_lanes;
    return {((int64_t)group_id() << (8 - log2_lanes)) + (threadIdx.x >> log2_lanes),
            (int)threadIdx.x & (lanes - 1), lanes};
}

// A row is read once and written to each of its slots.  65536 rows of 1024 bf16 to two
// experts each: 77 us, 5.2 TB/s.
template <typename T, int B>
__global__ __launch_bounds__(256) void k_expert_gather_rows(ExpertPlan p, ExpertMatrix x,
                                                            int32_t chunks, int log2_lanes,
                                                            T *__restrict__ sorted) {
    typedef typename Bytes<B>::type V;
    const RowLanes r = row_lanes(log2_lanes);
    if (r.row >= p.rows) return;
    const V *from = reinterpret_cast<const V *>(static_cast<const T *>(x.data) +
                                                r.row * x.row_stride);
    const int32_t *slots = p.slot + r.row * p.k;
    for (int c = r.lane; c < chunks; c += 4 * r.lanes) {
        V v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (c + q * r.lanes < chunks) v[q] = from[c + q * r.lanes];
        for (int j = 0; j < p.k; ++j) {
            const int32_t s = slots[j];
            if (s < 0) continue;
            V *to = reinterpret_cast<V *>(sorted + (int64_t)s * x.cols);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c + q * r.lanes < chunks) to[c + q * r.lanes] = v[q];
        }
    }
}

template <typename T, int B>
__global__ __launch_bounds__(256) void k_expert_combine_rows(ExpertPlan p,
                                                             const T *__restrict__ sorted,
                                                             const float *__restrict__ weights,
                                                             ExpertMatrix out, int32_t chunks,
                                                             int log2_lanes) {
    typedef typename Bytes<B>::type V;
    constexpr int E = B / sizeof(T);
    const RowLanes r = row_lanes(log2_lanes);
    if (r.row >= p.rows) return;
    V *to = reinterpret_cast<V *>(static_cast<T *>(out.data) + r.row * out.row_stride);
    for (int c = r.lane; c < chunks; c += 2 * r.lanes) {
        float sum[2][E];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < E; ++e) sum[q][e] = 0.0f;
        for (int j = 0; j < p.k; ++j) {
            const int64_t a = r.row * p.k + j;
            const int32_t s = p.slot[a];
            if (s < 0) continue;
            const float w = weights ? weights[a] : 1.0f;
            const V *from = reinterpret_cast<const V *>(sorted + (int64_t)s * out.cols);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (c + q * r.lanes >= chunks) break;
                const V v = from[c + q * r.lanes];
                T x[E];
                __builtin_memcpy(x, &v, B);
#pragma unroll
                for (int e = 0; e < E; ++e) sum[q][e] += w * to_f32(x[e]);
            }
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (c + q * r.lanes >= chunks) break;
            T x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = (T)sum[q][e];
            V v;
            __builtin_memcpy(&v, x, B);
            to[c + q * r.lanes] = v;
        }
    }
}

// A row's dot products are summed by its lanes, each over its own columns, and the lanes
// added in a fixed order.  65536 rows of 1024 bf16 from two experts each: 134 us, 5.0 TB/s.
template <typename T, int B>
__global__ __launch_bounds__(256) void k_expert_combine_grad_rows(
    ExpertPlan p, ExpertMatrix dout, const T *__restrict__ sorted,
    const float *__restrict__ weights, T *__restrict__ d_sorted, float *__restrict__ d_weights,
    int32_t chunks, int log2_lanes) {
    typedef typename Bytes<B>::type V;
    constexpr int E = B / sizeof(T);
    const RowLanes r = row_lanes(log2_lanes);
    if (r.row >= p.rows) return;
    const V *from = reinterpret_cast<const V *>(static_cast<const T *>(dout.data) +
                                                r.row * dout.row_stride);
    for (int j = 0; j < p.k; ++j) {
        const int64_t a = r.row * p.k + j;
        const int32_t s = p.slot[a];
        float dot = 0.0f;
        if (s >= 0) {
            const float w = weights ? weights[a] : 1.0f;
            const V *y = reinterpret_cast<const V *>(sorted + (int64_t)s * dout.cols);
            V *dy = reinterpret_cast<V *>(d_sorted + (int64_t)s * dout.cols);
#pragma unroll 2
            for (int c = r.lane; c < chunks; c += r.lanes) {
                const V gv = from[c], yv = y[c];
                T g[E], x[E];
                __builtin_memcpy(g, &gv, B);
                __builtin_memcpy(x, &yv, B);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float f = to_f32(g[e]);
                    dot += f * to_f32(x[e]);
                    x[e] = (T)(w * f);
                }
                V v;
                __builtin_memcpy(&v, x, B);
                dy[c] = v;
            }
        }
        for (int o = r.lanes / 2; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
        if (r.lane == 0) d_weights[a] = s < 0 ? 0.0f : dot;
    }
}

// ---- feature-major to blocks: the assignments of a run of rows, in LDS in their order ----
// An expert's assignments of consecutive rows have consecutive slots: with the run's values
// of a column ordered by (expert, slot) in LDS, both sides of the copy are runs of
// addresses.  Up to RUN_EXPERTS experts, whose places LDS holds, and 16 assignments a row,
// which leave a run of 64 rows; there they win (100k x 100 f32 in us, and by the tiles below: 4
// experts 27 and 32, 64 32 and 55, 512 48 and 83, 64 with k = 16 385 and 1660, 512 752 and 2020).
// 1M x 100 f32: 211 us, 3.8 TB/s.
constexpr int RUN = 1024, RUN_COLS = 4, RUN_EXPERTS = 512;
template <typename T>
__global__ __launch_bounds__(256) void k_expert_gather_runs(ExpertPlan p, ExpertMatrix x,
                                                            int32_t run_rows,
                                                            T *__restrict__ sorted) {
    __shared__ uint32_t first[RUN_EXPERTS], begin[RUN_EXPERTS], wave_sum[4];
    __shared__ int64_t base[RUN];
    __shared__ int32_t step[RUN];
    __shared__ T tile[RUN_COLS][RUN];
    const int64_t i0 = (int64_t)run_of(blockIdx.x, gridDim.x) * run_rows;
    const int32_t rows = (int32_t)min((int64_t)run_rows, p.rows - i0), n = rows * p.k;
    for (int e = threadIdx.x; e < RUN_EXPERTS; e += 256) {
        first[e] = 0xFFFFFFFFu;
        begin[e] = 0;
    }
    __syncthreads();
    int32_t slot[RUN / 256], expert[RUN / 256];
#pragma unroll
    for (int q = 0; q < RUN / 256; ++q) {
        const int a = threadIdx.x + 256 * q;
        slot[q] = a < n ? p.slot[i0 * p.k + a] : -1;
        expert[q] = slot[q] >= 0 ? p.expert[i0 * p.k + a] : 0;
        if (slot[q] >= 0) {
            atomicMin(&first[expert[q]], (uint32_t)slot[q]);
            atomicAdd(&begin[expert[q]], 1u);
        }
    }
    __syncthreads();
    uint32_t taken;
    {
        const int e = threadIdx.x * 2;               // RUN_EXPERTS / 256 experts a thread
        const uint32_t c0 = begin[e], c1 = begin[e + 1];
        const uint32_t before = sum_before<4>(c0 + c1, wave_sum, taken);
        begin[e] = before;
        begin[e + 1] = before + c0;
    }
    __syncthreads();
    int at[RUN / 256], row[RUN / 256];
#pragma unroll
    for (int q = 0; q < RUN / 256; ++q) {
        at[q] = -1;
        row[q] = (threadIdx.x + 256 * q) / p.k;
        if (slot[q] < 0) continue;
        const int32_t e = expert[q], o = p.offsets[e];
        at[q] = (int)(begin[e] + ((uint32_t)slot[q] - first[e]));
        base[at[q]] = (int64_t)o * x.cols + (slot[q] - o);
        step[at[q]] = p.offsets[e + 1] - o;
    }
    const T *from[RUN / 256];
#pragma unroll
    for (int q = 0; q < RUN / 256; ++q)
        from[q] = static_cast<const T *>(x.data) + (i0 + (at[q] >= 0 ? row[q] : 0)) * x.row_stride;
    T v[RUN / 256][RUN_COLS];
    // the next columns are asked for before the last ones are stored: a load waits for
    // every access before it
    const auto load = [&](int32_t f0) {
#pragma unroll
        for (int c = 0; c < RUN_COLS; ++c) {
            const int64_t f = (int64_t)min(f0 + c, x.cols - 1) * x.col_stride;
#pragma unroll
            for (int q = 0; q < RUN / 256; ++q) v[q][c] = from[q][f];
        }
    };
    int32_t f0 = blockIdx.y * RUN_COLS;
    if (f0 < x.cols) load(f0);
    for (; f0 < x.cols; f0 += gridDim.y * RUN_COLS) {
        __syncthreads();                             // base and step, the last columns' reads
#pragma unroll
        for (int q = 0; q < RUN / 256; ++q)
            if (at[q] >= 0)
#pragma unroll
                for (int c = 0; c < RUN_COLS; ++c) tile[c][at[q]] = v[q][c];
        __syncthreads();
        const int32_t next = f0 + gridDim.y * RUN_COLS;
        if (next < x.cols) load(next);
        const int cols = min(RUN_COLS, x.cols - f0);
#pragma unroll
        for (int q = 0; q < RUN / 256; ++q) {
            const int l = threadIdx.x + 256 * q;
            if (l >= (int)taken) break;
            T *to = sorted + base[l] + (int64_t)f0 * step[l];
#pragma unroll
            for (int c = 0; c < RUN_COLS; ++c)
                if (c < cols) to[(int64_t)c * step[l]] = tile[c][l];
        }
    }
}

// ---- other layouts: a tile of 64 rows x 64 columns at a time, 256 threads ----
// XCOLS / SCOLS: the lanes of a wavefront run along the columns of the rows' matrix / of
// the sorted matrix, else along the rows; LDS turns the tile where the two differ.  Sums of
// 99991 x 2 blocks' rows of 37 f32: 14.4 us, 3.0 TB/s of its 43 MB, much of them in the L2s.
constexpr int TILE = 64;
template <typename T, bool XCOLS, bool SCOLS>
__global__ __launch_bounds__(256) void k_expert_gather(ExpertPlan p, ExpertMatrix x,
                                                       T *__restrict__ sorted) {
    __shared__ T tile[TILE][TILE + 1];
    const int64_t i0 = (int64_t)run_of(group_id(), group_count()) * TILE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T *data = static_cast<const T *>(x.data);
    for (int32_t f0 = blockIdx.y * TILE; f0 < x.cols; f0 += gridDim.y * TILE) {
#pragma unroll 4
        for (int q = wave; q < TILE; q += 4) {
            const int64_t i = i0 + (XCOLS ? q : lane);
            const int32_t f = f0 + (XCOLS ? lane : q);
            if (i < p.rows && f < x.cols)
                tile[XCOLS ? q : lane][XCOLS ? lane : q] =
                    data[i * x.row_stride + f * x.col_stride];
        }
        __syncthreads();
        if (SCOLS) {
            constexpr int Q = TILE / 4;
            for (int j = 0; j < p.k; ++j) {
                int32_t s[Q];
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    const int64_t i = i0 + wave + 4 * q;
                    s[q] = i < p.rows && f0 + lane < x.cols ? p.slot[i * p.k + j] : -1;
                }
#pragma unroll
                for (int q = 0; q < Q; ++q)
                    if (s[q] >= 0)
                        sorted[(int64_t)s[q] * x.cols + f0 + lane] = tile[wave + 4 * q][lane];
            }
        } else if (i0 + lane < p.rows) {
            for (int j = 0; j < p.k; ++j) {
                const Place at = place_of(p, (i0 + lane) * p.k + j, x.cols, x.blocked);
                if (at.base < 0) continue;
                for (int q = wave; q < TILE && f0 + q < x.cols; q += 4)
                    sorted[at.base + (f0 + q) * at.step] = tile[lane][q];
            }
        }
        __syncthreads();
    }
}

// out[i] = sum over j, ascending, of weight[i][j] * sorted[slot[i][j]], in f32.
template <typename T, bool XCOLS, bool SCOLS>
__global__ __launch_bounds__(256) void k_expert_combine(ExpertPlan p, const T *__restrict__ sorted,
                                                        const float *__restrict__ weights,
                                                        ExpertMatrix out) {
    constexpr int Q = TILE / 4;
    __shared__ float tile[TILE][TILE + 1];
    const int64_t i0 = (int64_t)run_of(group_id(), group_count()) * TILE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T *data = static_cast<T *>(out.data);
    for (int32_t f0 = blockIdx.y * TILE; f0 < out.cols; f0 += gridDim.y * TILE) {
        if (SCOLS) {
            // eight of the wavefront's rows at once, so that their loads are on the way together
            constexpr int H = Q / 2;
#pragma unroll 1
            for (int q0 = wave; q0 < TILE; q0 += 4 * H) {
                float sum[H];
#pragma unroll
                for (int q = 0; q < H; ++q) sum[q] = 0.0f;
                for (int j = 0; j < p.k; ++j) {
                    int32_t s[H];
                    float v[H], w[H];
#pragma unroll
                    for (int q = 0; q < H; ++q) {
                        const int64_t i = i0 + q0 + 4 * q, a = i * p.k + j;
                        s[q] = i < p.rows ? p.slot[a] : -1;
                        w[q] = weights && i < p.rows ? weights[a] : 1.0f;
                    }
#pragma unroll
                    for (int q = 0; q < H; ++q)
                        v[q] = s[q] >= 0 && f0 + lane < out.cols
                                   ? to_f32(sorted[(int64_t)s[q] * out.cols + f0 + lane]) : 0.0f;
#pragma unroll
                    for (int q = 0; q < H; ++q)
                        if (s[q] >= 0) sum[q] += w[q] * v[q];
                }
#pragma unroll
                for (int q = 0; q < H; ++q) tile[q0 + 4 * q][lane] = sum[q];
            }
        } else if (i0 + lane < p.rows) {
            float sum[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) sum[q] = 0.0f;
            // two assignments' values are asked for at once
            for (int j = 0; j < p.k; j += 2) {
                float v[2][Q], w[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t a = (i0 + lane) * p.k + min(j + h, p.k - 1);
                    const Place at = place_of(p, a, out.cols, out.blocked);
                    const bool take = at.base >= 0 && j + h < p.k;
                    w[h] = take && weights ? weights[a] : 1.0f;
                    const T *from = sorted + at.base + (f0 + wave) * at.step;
#pragma unroll
                    for (int q = 0; q < Q; ++q)
                        v[h][q] = take && f0 + wave + 4 * q < out.cols
                                      ? to_f32(from[4 * q * at.step]) : 0.0f;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < Q; ++q) sum[q] += w[h] * v[h][q];
            }
#pragma unroll
            for (int q = 0; q < Q; ++q) tile[lane][wave + 4 * q] = sum[q];
        }
        __syncthreads();
        for (int q = wave; q < TILE; q += 4) {
            const int r = XCOLS ? q : lane, c = XCOLS ? lane : q;
            if (i0 + r < p.rows && f0 + c < out.cols)
                data[(i0 + r) * out.row_stride + (f0 + c) * out.col_stride] = (T)tile[r][c];
        }
        __syncthreads();
    }
}

// d_sorted[slot[i][j]] = weight[i][j] * dout[i] and d_weights[i][j] = dout[i] .
// sorted[slot[i][j]].  A workgroup has all columns of its rows: each thread sums its
// own columns in f32, and the threads of a row are added in a fixed order.  With few rows their
// k go to workgroups of their own (1775 x 8 rows of 2 bf16 77 us by 28 workgroups).
template <typename T, bool XCOLS, bool SCOLS>
__global__ __launch_bounds__(256, 4) void k_expert_combine_grad(
    ExpertPlan p, ExpertMatrix dout, const T *__restrict__ sorted,
    const float *__restrict__ weights, T *__restrict__ d_sorted, float *__restrict__ d_weights) {
    __shared__ T tile[TILE][TILE + 1];
    __shared__ float sums[TILE][5];
    const int64_t i0 = (int64_t)run_of(group_id(), group_count()) * TILE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T *data = static_cast<const T *>(dout.data);
    for (int j = blockIdx.y; j < p.k; j += gridDim.y) {
        // SCOLS: the sums of rows wave + 4 q over this lane's columns; else of row lane
        float dot[SCOLS ? TILE / 4 : 1];
#pragma unroll
        for (int q = 0; q < (SCOLS ? TILE / 4 : 1); ++q) dot[q] = 0.0f;
        int32_t s[SCOLS ? TILE / 4 : 1];
        float wt[SCOLS ? TILE / 4 : 1];
        if constexpr (SCOLS)
#pragma unroll
            for (int q = 0; q < TILE / 4; ++q) {
                const int64_t i = i0 + wave + 4 * q, a = i * p.k + j;
                s[q] = i < p.rows ? p.slot[a] : -1;
                wt[q] = weights && i < p.rows ? weights[a] : 1.0f;
            }
        Place mine{-1, 0};
        float w = 1.0f;
        if (!SCOLS && i0 + lane < p.rows) {
            mine = place_of(p, (i0 + lane) * p.k + j, dout.cols, dout.blocked);
            if (weights) w = weights[(i0 + lane) * p.k + j];
        }
        for (int32_t f0 = 0; f0 < dout.cols; f0 += TILE) {
            __syncthreads();
#pragma unroll 4
            for (int q = wave; q < TILE; q += 4) {
                const int r = XCOLS ? q : lane, c = XCOLS ? lane : q;
                if (i0 + r < p.rows && f0 + c < dout.cols)
                    tile[r][c] = data[(i0 + r) * dout.row_stride + (f0 + c) * dout.col_stride];
            }
            __syncthreads();
            if constexpr (SCOLS) {
                // eight rows at once, so that their loads are on the way together
                constexpr int H = TILE / 8;
#pragma unroll
                for (int q0 = 0; q0 < TILE / 4; q0 += H) {
                    int64_t at[H];
                    float v[H];
#pragma unroll
                    for (int q = 0; q < H; ++q) {
                        int32_t slot = f0 + lane < dout.cols ? s[q0 + q] : -1;
                        asm volatile("" : "+v"(slot));   // places are not kept over f0: registers
                        at[q] = slot < 0 ? -1 : (int64_t)slot * dout.cols + f0 + lane;
                        v[q] = slot < 0 ? 0.0f : to_f32(sorted[at[q]]);
                    }
#pragma unroll
                    for (int q = 0; q < H; ++q) {
                        if (at[q] < 0) continue;
                        const float g = to_f32(tile[wave + 4 * (q0 + q)][lane]);
                        dot[q0 + q] += g * v[q];
                        d_sorted[at[q]] = (T)(wt[q0 + q] * g);
                    }
                }
            } else if (mine.base >= 0) {
#pragma unroll 4
                for (int q = wave; q < TILE; q += 4) {
                    if (f0 + q >= dout.cols) break;
                    const float g = to_f32(tile[lane][q]);
                    const int64_t k = mine.base + (f0 + q) * mine.step;
                    dot[0] += g * to_f32(sorted[k]);
                    d_sorted[k] = (T)(w * g);
                }
            }
        }
        if constexpr (SCOLS) {
            // each exchange halves the rows a lane holds
#pragma unroll
            for (int n = TILE / 8, o = 32; n > 0; n >>= 1, o >>= 1)
#pragma unroll
                for (int q = 0; q < n; ++q) {
                    const bool upper = lane & o;
                    const float keep = upper ? dot[q + n] : dot[q], give = upper ? dot[q] : dot[q + n];
                    dot[q] = keep + __shfl_xor(give, o, 64);
                }
            dot[0] += __shfl_xor(dot[0], 2, 64);
            dot[0] += __shfl_xor(dot[0], 1, 64);
            const int64_t i = i0 + wave + 4 * ((lane >> 5 & 1) * 8 + (lane >> 4 & 1) * 4 +
                                               (lane >> 3 & 1) * 2 + (lane >> 2 & 1));
            if ((lane & 3) == 0 && i < p.rows) d_weights[i * p.k + j] = dot[0];
        } else {
            sums[lane][wave] = dot[0];
            __syncthreads();
            if (threadIdx.x < TILE && i0 + lane < p.rows)
                d_weights[(i0 + lane) * p.k + j] =
                    (sums[lane][0] + sums[lane][1]) + (sums[lane][2] + sums[lane][3]);
        }
    }
}

bool along_columns(const ExpertMatrix &x) { return x.col_stride <= x.row_stride; }

dim3 tile_grid(int64_t rows, int32_t cols) {
    return grid_of((rows + TILE - 1) / TILE,
                   (uint32_t)std::min<int32_t>((cols + TILE - 1) / TILE, 1024));
}

// Bytes a lane moves where both matrices lie by rows: 16 where everything is aligned to
// it, else 4 or an element (sums of 65536 x 2 rows of 1024 bf16 77 us by 16 bytes, 112 by 4; of
// 100k x 2 rows of 100 f32 23 and 30, their gradient 37 and 51).
int lane_bytes(const ExpertMatrix &x, int size, const void *a, const void *b) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(x.data) | reinterpret_cast<uintptr_t>(a) |
                          reinterpret_cast<uintptr_t>(b) | (uintptr_t)(x.row_stride * size) |
                          (uintptr_t)((int64_t)x.cols * size);
    return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : size;
}
struct RowShape {
    int bytes, log2_lanes;
    int32_t chunks;
    uint32_t groups;
};
RowShape row_shape(const ExpertMatrix &x, int64_t rows, int size, const void *a, const void *b) {
    RowShape r{lane_bytes(x, size, a, b), 0, 0, 0};
    r.chunks = (int32_t)((int64_t)x.cols * size / r.bytes);
    while (r.log2_lanes < 6 && (1 << r.log2_lanes) < r.chunks) ++r.log2_lanes;
    const int64_t per = 256 >> r.log2_lanes;
    r.groups = (uint32_t)((rows + per - 1) / per);
    return r;
}
// By rows on both sides.
bool by_rows(const ExpertMatrix &x) { return x.col_stride == 1 && !x.blocked; }

#define BY_BYTES(kernel, ...)                                                                    \
    do {                                                                                         \
        if (r.bytes == 16)                                                                       \
            hipLaunchKernelGGL((kernel<T, 16>), grid_of(r.groups), dim3(256), 0, s, __VA_ARGS__);   \
        else if (r.bytes == 4)                                                                   \
            hipLaunchKernelGGL((kernel<T, 4>), grid_of(r.groups), dim3(256), 0, s, __VA_ARGS__);    \
        else if constexpr (sizeof(T) == 2)                                                       \
            hipLaunchKernelGGL((kernel<T, 2>), grid_of(r.groups), dim3(256), 0, s, __VA_ARGS__);    \
    } while (0)
#define BY_LAYOUT(kernel, grid, ...)                                                             \
    do {                                                                                         \
        const bool xc = along_columns(x), sc = !x.blocked;                                       \
        if (xc && sc) hipLaunchKernelGGL((kernel<T, true, true>), grid, dim3(256), 0, s, __VA_ARGS__);  \
        else if (xc) hipLaunchKernelGGL((kernel<T, true, false>), grid, dim3(256), 0, s, __VA_ARGS__);  \
        else if (sc) hipLaunchKernelGGL((kernel<T, false, true>), grid, dim3(256), 0, s, __VA_ARGS__);  \
        else hipLaunchKernelGGL((kernel<T, false, false>), grid, dim3(256), 0, s, __VA_ARGS__);  \
    } while (0)

template <typename T>
hipError_t gather(hipStream_t s, const ExpertPlan &p, const ExpertMatrix &x, void *sorted) {
    T *out = static_cast<T *>(sorted);
    if (by_rows(x)) {
        const RowShape r = row_shape(x, p.rows, sizeof(T), sorted, nullptr);
        BY_BYTES(k_expert_gather_rows, p, x, r.chunks, r.log2_lanes, out);
    } else if (x.blocked && !along_columns(x) && p.experts <= RUN_EXPERTS && p.k <= 16) {
        const int32_t rows = RUN / p.k;
        const uint32_t runs = (uint32_t)((p.rows + rows - 1) / rows);
        const uint32_t cols = (uint32_t)((x.cols + RUN_COLS - 1) / RUN_COLS);
        // few runs: their columns go to several workgroups
        const uint32_t parts = std::max(1u, std::min({cols, 1024 / std::max(1u, runs), 65535u}));
        hipLaunchKernelGGL((k_expert_gather_runs<T>), dim3(runs, parts), dim3(256), 0, s, p, x, rows,
                           out);
    } else {
        BY_LAYOUT(k_expert_gather, tile_grid(p.rows, x.cols), p, x, out);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t combine(hipStream_t s, const ExpertPlan &p, const void *sorted, const float *w,
                   const ExpertMatrix &x) {
    const T *y = static_cast<const T *>(sorted);
    if (by_rows(x)) {
        const RowShape r = row_shape(x, p.rows, sizeof(T), sorted, nullptr);
        BY_BYTES(k_expert_combine_rows, p, y, w, x, r.chunks, r.log2_lanes);
    } else {
        BY_LAYOUT(k_expert_combine, tile_grid(p.rows, x.cols), p, y, w, x);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t combine_grad(hipStream_t s, const ExpertPlan &p, const ExpertMatrix &x,
                        const void *sorted, const float *w, void *d_sorted, float *d_weights) {
    const T *y = static_cast<const T *>(sorted);
    T *dy = static_cast<T *>(d_sorted);
    if (by_rows(x)) {
        const RowShape r = row_shape(x, p.rows, sizeof(T), sorted, d_sorted);
        BY_BYTES(k_expert_combine_grad_rows, p, x, y, w, dy, d_weights, r.chunks, r.log2_lanes);
    } else {
        const int64_t groups = (p.rows + TILE - 1) / TILE;
        const int64_t each = std::max<int64_t>(1, std::min<int64_t>({p.k, 1024 / groups, 65535}));
        BY_LAYOUT(k_expert_combine_grad, grid_of(groups, (uint32_t)each), p, x, y, w, dy, d_weights);
    }
    return hipGetLastError();
}
#undef BY_BYTES
#undef BY_LAYOUT

// Chunks of up to 2048 workgroups (a thread of the scan takes eight).
SortShape chunk_shape(const ExpertPlan &p, int64_t chunk) {
    const int64_t slots = p.rows * p.k, chunks = (slots + chunk - 1) / chunk;
    const int64_t per = std::max<int64_t>(1, (chunks + SCAN * SCAN_EACH - 1) / (SCAN * SCAN_EACH));
    return {per * chunk, (int32_t)std::max<int64_t>(1, (chunks + per - 1) / per)};
}
bool by_chunks(const ExpertPlan &p) { return p.experts <= CHUNK_EXPERTS; }
SortShape shape_of(const ExpertPlan &p, int num_cus) {
    if (!by_chunks(p)) return sort_shape(p, num_cus);
    return chunk_shape(p, p.rows * p.k <= FEW_SLOTS ? CHUNK<4> : CHUNK<16>);
}

template <int R>
hipError_t sort_chunks(hipStream_t s, const ExpertPlan &p, const SortShape &sh, int bits,
                       uint32_t *table, uint32_t *total) {
    for (const void *f : {reinterpret_cast<const void *>(k_expert_place_chunks<R, true>),
                          reinterpret_cast<const void *>(k_expert_place_chunks<R, false>)}) {
        const hipError_t e = allow_all_lds(f);
        if (e != hipSuccess) return e;
    }
    const int64_t slots = p.rows * p.k;
    const dim3 g((uint32_t)sh.units), b(64 * CHUNK_WAVES);
    const size_t lds = sizeof(uint32_t) *
                       (CHUNK_WAVES + CHUNK<R> + (size_t)(CHUNK_WAVES + 2) * p.experts);
    hipLaunchKernelGGL((k_expert_count_chunks<R>), g, b, sizeof(uint32_t) * p.experts, s, p.expert,
                       slots, p.experts, sh.per, sh.units, table);
    if (p.experts <= DIRECT_EXPERTS && (int64_t)p.experts * sh.units <= DIRECT_COUNTERS) {
        hipLaunchKernelGGL((k_expert_place_chunks<R, true>), g, b, lds, s, p.expert, slots,
                           p.experts, bits, sh.per, sh.units, table, p.offsets, p.source, p.slot);
    } else {
        hipLaunchKernelGGL(k_expert_scan, dim3((uint32_t)p.experts), dim3(SCAN), 0, s, table,
                           sh.units, total);
        hipLaunchKernelGGL(k_expert_offsets, dim3(1), dim3(1024), 0, s, total, p.experts,
                           p.offsets);
        hipLaunchKernelGGL((k_expert_place_chunks<R, false>), g, b, lds, s, p.expert, slots,
                           p.experts, bits, sh.per, sh.units, table, p.offsets, p.source, p.slot);
    }
    return hipGetLastError();
}

}  // namespace

size_t expert_scratch(const ExpertPlan &p, int num_cus) {
    const SortShape sh = shape_of(p, num_cus);
    return ((size_t)p.experts * sh.units + p.experts + 1) * sizeof(uint32_t);
}

hipError_t launch_expert_sort(hipStream_t s, const ExpertPlan &p, int num_cus, char *scratch) {
    const SortShape sh = shape_of(p, num_cus);
    const int64_t slots = p.rows * p.k;
    uint32_t *table = reinterpret_cast<uint32_t *>(scratch);
    uint32_t *total = table + (size_t)p.experts * sh.units;
    int32_t *trash = reinterpret_cast<int32_t *>(total + p.experts);
    int bits = 0;
    while (bits < 31 && (1 << bits) < p.experts) ++bits;
    for (const void *f : {reinterpret_cast<const void *>(k_expert_count),
                          reinterpret_cast<const void *>(k_expert_place),
                          reinterpret_cast<const void *>(k_expert_sort_small)}) {
        const hipError_t e = allow_all_lds(f);
        if (e != hipSuccess) return e;
    }
    if (slots <= SMALL_SLOTS && p.experts <= SMALL_EXPERTS) {
        const int64_t per = ((slots + SMALL_WAVES - 1) / SMALL_WAVES + 63) / 64 * 64;
        hipLaunchKernelGGL(k_expert_sort_small, dim3(1), dim3(64 * SMALL_WAVES),
                           (size_t)SMALL_WAVES * (p.experts + 1) * sizeof(uint32_t), s, p.expert,
                           slots, p.experts, bits, per, p.offsets, p.source, p.slot, trash);
        return hipGetLastError();
    }
    if (by_chunks(p))
        return slots <= FEW_SLOTS ? sort_chunks<4>(s, p, sh, bits, table, total)
                                  : sort_chunks<16>(s, p, sh, bits, table, total);
    const dim3 g((uint32_t)((sh.units + SORT_WAVES - 1) / SORT_WAVES)), b(64 * SORT_WAVES);
    const size_t lds = (size_t)SORT_WAVES * p.experts * sizeof(uint32_t);
    hipLaunchKernelGGL(k_expert_count, g, b, lds, s, p.expert, slots, p.experts, sh.per, sh.units,
                       table);
    hipLaunchKernelGGL(k_expert_scan, dim3((uint32_t)p.experts), dim3(SCAN), 0, s, table, sh.units,
                       total);
    hipLaunchKernelGGL(k_expert_offsets, dim3(1), dim3(1024), 0, s, total, p.experts, p.offsets);
    hipLaunchKernelGGL(k_expert_place, g, b, lds, s, p.expert, slots, p.experts, bits, sh.per,
                       sh.units, table, p.offsets, p.source, p.slot, trash);
    return hipGetLastError();
}

hipError_t launch_expert_gather(hipStream_t s, const ExpertPlan &p, const ExpertMatrix &x,
                                void *sorted) {
    return x.bf16 ? gather<__bf16>(s, p, x, sorted) : gather<float>(s, p, x, sorted);
}

hipError_t launch_expert_combine(hipStream_t s, const ExpertPlan &p, const void *sorted,
                                 const float *weights, const ExpertMatrix &out) {
    return out.bf16 ? combine<__bf16>(s, p, sorted, weights, out)
                    : combine<float>(s, p, sorted, weights, out);
}

hipError_t launch_expert_combine_grad(hipStream_t s, const ExpertPlan &p,
                                      const ExpertMatrix &dout, const void *sorted,
                                      const float *weights, void *d_sorted, float *d_weights) {
    return dout.bf16 ? combine_grad<__bf16>(s, p, dout, sorted, weights, d_sorted, d_weights)
                     : combine_grad<float>(s, p, dout, sorted, weights, d_sorted, d_weights);
}

}  // namespace mbk
