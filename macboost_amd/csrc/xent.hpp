// xent.hpp — what the kernels of the many-class loss share: the packed operands and
// the matrix instruction on them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "grid.hpp"
#include "ops.h"

namespace mbk {

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;       // 8 operands
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef unsigned short u16;

constexpr float LOG2E = 1.44269504088896341f;
// Values beyond this (2^60) in a row that is out count as not finite: times a finite W they
// could still overflow.
constexpr uint32_t XENT_HUGE = 0x5D800000u;
// So does the whole row where its power of two is below 2^this: its scores may pass 2^100.
constexpr int FAR_ROW = -100;

// ---- control words -----------------------------------------------------------
// A maximum over the workgroups of a kernel: each leaves its own, and those of a later one
// look them all over.  (Atomics on one word took 15 to 20 ns each, 42 us for the largest of
// 16300 x 1000 f32 by 2048 workgroups, and a launch to clear it.)
constexpr int MOST_GROUPS = 1024;
struct XentMax {
    uint32_t part[MOST_GROUPS];
    uint32_t all;                        // a later kernel's first workgroup leaves it here
};
struct XentCtl {
    XentMax offered;                     // 1: a class is
    XentMax row;                         // see kernels_xent_fused.hip, and this
    uint32_t far;
};

__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t b = __float_as_uint(fabsf(x));
    return b < 0x7F800000u ? b : 0u;
}
// Packed operands lie below 2^TOP_EXP.
constexpr int TOP_EXP = 14;
// e, where |x| is in [2^(e-1), 2^e); NO_EXP for 0 and what is not finite.
constexpr int NO_EXP = -(1 << 20);
__device__ __forceinline__ int exponent_of(float x) {
    return finite_bits(x) ? __builtin_amdgcn_frexp_expf(x) : NO_EXP;
}
// 2^e, at most 2^127: 0 times it is 0.
__device__ __forceinline__ float power_of_2(int e) { return ldexpf(1.0f, min(e, 127)); }

template <typename V> __device__ __forceinline__ V wave_max(V v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (V)__shfl_xor((int)v, o, 64));
    return v;
}
// Of a workgroup of WAVES wavefronts; all of its threads call it.  lds: WAVES words, free
// again at the end.
template <int WAVES, typename V> __device__ __forceinline__ V largest(V v, V *lds) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) v = max(v, lds[i]);
    __syncthreads();
    return v;
}
template <int WAVES>
__device__ __forceinline__ uint32_t largest_of(const XentMax &m, int32_t groups, uint32_t *lds) {
    uint32_t v = 0;
    for (int g = threadIdx.x; g < groups; g += 64 * WAVES) v = max(v, m.part[g]);
    return largest<WAVES>(v, lds);
}

__device__ __forceinline__ u16 bits_of(_Float16 v) { return __builtin_bit_cast(u16, v); }

// x in two f16 terms.
__device__ __forceinline__ void split_f16(float x, u16 &hi, u16 &lo) {
    const _Float16 h = (_Float16)x;
    hi = bits_of(h);
    lo = bits_of((_Float16)(x - (float)h));
}

// What the kernels read: operands in rows of ld 16-bit elements, zeros behind the
// sizes, P planes of them.
struct XentPack {
    int64_t n, v, n_pad, v_pad;
    int32_t d, ld;
    int32_t w_groups, hg_groups;         // that look at W's and w h's columns
    int32_t pack_w_groups, pack_h_groups;
    bool few;                            // groups: those that pack sum them up
    XentCtl *ctl;
    int32_t *w_part, *hg_part;           // [group][ld] a column's largest exponent
    int32_t *w_exp, *hg_exp;             // [ld] a column is packed times 2^this
    u16 *h, *hg, *w;                     // planes of n_pad * ld, v_pad * ld; hg: gradients only
    float *bias;                         // [v_pad] the bias, -inf: not offered
    float *row_scale;                    // [n_pad] the scale of a score
    int32_t *label;                      // [n_pad], -1: out, -2: out and not finite
    float *weight;                       // [n_pad], 0: out
};

template <int P>
__device__ __forceinline__ f32x16 mma(const u32x4 (&a)[P], const u32x4 (&b)[P], f32x16 c) {
    const f16x8 a0 = __builtin_bit_cast(f16x8, a[0]), b0 = __builtin_bit_cast(f16x8, b[0]);
    if constexpr (P == 2) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a[1]), b0, c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0, __builtin_bit_cast(f16x8, b[1]), c, 0, 0, 0);
    }
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a0, b0, c, 0, 0, 0);
}

// Scores are kept as they are, base e: times log2 e a finite bias below -2.4e38 would become
// the -inf of a class that is not offered.  What is left of a score behind its row's
// maximum takes the factor.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// A row's sum of exp(z - reference), as its logarithm apart from the reference: together in one
// f32 a reference of 2^24 would leave nothing of it.
struct LogSum {
    float base2;
    double natural;
};
// Of sum / 2^shift.  The exponent apart, since the logarithm instruction rounds down, by up to
// a step of a result of 2^4.
__device__ __forceinline__ LogSum log_sum(float sum, int shift = 0) {
    if (!(sum > 0.0f && sum < INFINITY)) {
        const float l = log2f(sum);
        return {l, l};
    }
    const int e = __builtin_amdgcn_frexp_expf(sum) - shift;
    const double l = (double)e + log2f(__builtin_amdgcn_frexp_mantf(sum));
    return {(float)l, l * 0.693147180559945309};
}
// lse and, of a score z, lse - z.
__device__ __forceinline__ float lse_of(float ref, const LogSum &l) {
    return (float)((ref == -INFINITY ? 0.0 : (double)ref) + l.natural);
}
__device__ __forceinline__ float loss_of(float ref, const LogSum &l, float z) {
    return (float)(((double)ref - z) + l.natural);
}

// ---- copies from memory to LDS
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// The copies that this wavefront has started are in LDS; a barrier alone does not wait
// for them.
__device__ __forceinline__ void copies_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }

__device__ __forceinline__ uint32_t lds_address(const char *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p;
}
// A number that a generic lambda takes as a constant.
template <int N> struct At {
    static constexpr int value = N;
};

// The kernels of up to XENT_FUSED_DIM outputs (kernels_xent_fused.hip): scores, their
// exponentials and the product with them in one pass for dh and one for dW.  128 is what a
// wavefront's registers hold of both operands; up to there they win at every size (us, fused
// and by products: f32 20000 x 128 x 10000 loss 204 and 228, with gradients 611 and 1233, 1000 x
// 128 x 1000 57 and 87; bf16 20000 x 32 x 10000 180 and 537).
constexpr int XENT_FUSED_DIM = 128;
size_t xent_fused_scratch(const XentCall &c);
hipError_t launch_xent_fused(hipStream_t s, const XentCall &c, char *scratch);

// The loss of few rows (kernels_xent_few.hip), whose work is one reading of W.
bool xent_few(const XentCall &c);
size_t xent_few_scratch(const XentCall &c);
hipError_t launch_xent_few(hipStream_t s, const XentCall &c, char *scratch);

}  // namespace mbk
