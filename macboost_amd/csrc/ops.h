// ops.h — kernel launchers of the seam's many-class loss (kernels_xent.hip) and
// of rows sorted by expert (kernels_expert.hip); ops.cpp checks the arguments.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mbk {

// ---- cross entropy over many classes ----------------------------------------

struct XentCall {
    int64_t rows, classes;
    int32_t dim;
    bool bf16;                       // h, w, dh, dw: bf16, else f32
    int64_t h_stride, w_stride;
    const void *h, *w;
    const float *bias;               // NULL: none
    const int32_t *labels;
    const float *weights;            // NULL: 1
    float *loss, *lse;
    bool grad;
    void *dh, *dw;                   // NULL: not asked for
    float *dbias;
    int num_cus;
};
// Bytes of scratch that the call takes.
size_t xent_scratch(const XentCall &c);
hipError_t launch_xent(hipStream_t s, const XentCall &c, char *scratch);

// ---- rows sorted by expert ---------------------------------------------------

struct ExpertPlan {
    int64_t rows;
    int32_t k, experts;
    const int32_t *expert;           // [rows][k]
    int32_t *offsets, *source, *slot;
};
// The rows' matrix: element (i, f) at data[i * row_stride + f * col_stride].
struct ExpertMatrix {
    void *data;
    int64_t row_stride, col_stride;
    int32_t cols;
    bool bf16;                       // else f32
    bool blocked;                    // layout of the sorted matrix
};
size_t expert_scratch(const ExpertPlan &p, int num_cus);
hipError_t launch_expert_sort(hipStream_t s, const ExpertPlan &p, int num_cus, char *scratch);
hipError_t launch_expert_gather(hipStream_t s, const ExpertPlan &p, const ExpertMatrix &x,
                                void *sorted);
hipError_t launch_expert_combine(hipStream_t s, const ExpertPlan &p, const void *sorted,
                                 const float *weights, const ExpertMatrix &out);
hipError_t launch_expert_combine_grad(hipStream_t s, const ExpertPlan &p,
                                      const ExpertMatrix &dout, const void *sorted,
                                      const float *weights, void *d_sorted, float *d_weights);

}  // namespace mbk
