// ops.cpp — the seam's operators beside the tree build: the loss over many classes
// (mbk_xent, mbk_xent_grad) and rows sorted by expert (mbk_expert_*).  Each call
// checks its arguments (the context last), queues its kernels on the context's stream and
// returns; it allocates only when it needs more scratch than the context holds.  Calls that
// use scratch are queued whole, one after another, whichever threads make them.
#include "../../include/macboost.h"
#include "abi.hpp"
#include "core.hpp"
#include "ops.h"

namespace {

void need(bool ok, const char *what) {
    if (!ok) mb::invalid(what);
}

constexpr int64_t MOST_ROWS = 0x7FFFFF00;
constexpr int32_t MOST_EXPERTS = 8192;       // counters of four wavefronts in LDS
constexpr int64_t MOST_STRIDE = (int64_t)1 << 40;

bool is_bf16(int32_t type) {
    need(type == MBK_F32 || type == MBK_BF16, "type must be MBK_F32 or MBK_BF16");
    return type == MBK_BF16;
}

mbk::XentCall xent_call(const mbk_xent_shape *sh, const void *h,
                        const void *w, const float *bias, const int32_t *labels,
                        const float *weights, float *loss, float *lse) {
    need(sh != nullptr, "null shape");
    need(sh->rows >= 0 && sh->rows <= MOST_ROWS, "rows must be in 0..2^31-256");
    need(sh->classes >= 1 && sh->classes <= MOST_ROWS, "classes must be in 1..2^31-256");
    need(sh->dim >= 1 && sh->dim <= (1 << 20), "dim must be in 1..2^20");
    need(sh->h_stride >= sh->dim && sh->w_stride >= sh->dim,
         "h_stride and w_stride must be at least dim");
    need(sh->h_stride <= MOST_STRIDE && sh->w_stride <= MOST_STRIDE,
         "h_stride and w_stride must be at most 2^40");
    need(w && (!sh->rows || (h && labels && loss && lse)), "null argument");
    mbk::XentCall c{};
    c.rows = sh->rows;
    c.classes = sh->classes;
    c.dim = sh->dim;
    c.bf16 = is_bf16(sh->type);
    c.h_stride = sh->h_stride;
    c.w_stride = sh->w_stride;
    c.h = h;
    c.w = w;
    c.bias = bias;
    c.labels = labels;
    c.weights = weights;
    c.loss = loss;
    c.lse = lse;
    return c;
}

void run_xent(mbk_context *ctx, mbk::XentCall c) {
    need(ctx != nullptr, "null kernel-seam context");
    c.num_cus = mb::context_cus(ctx);
    mb::OnDevice here(mb::context_device(ctx));
    std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
    char *scratch = mb::context_scratch(ctx, mbk::xent_scratch(c));
    MB_HIP(mbk::launch_xent(mb::context_stream(ctx), c, scratch));
}

mbk::ExpertPlan expert_plan(const mbk_expert_plan *p) {
    need(p != nullptr, "null plan");
    need(p->rows >= 0 && p->k >= 1 && p->rows <= MOST_ROWS / p->k,
         "rows must be >= 0, k >= 1 and rows * k at most 2^31-256");
    need(p->experts >= 1 && p->experts <= MOST_EXPERTS, "experts must be in 1..8192");
    need(p->offsets && (!p->rows || (p->expert && p->source && p->slot)), "null plan array");
    return {p->rows, p->k, p->experts, p->expert, p->offsets, p->source, p->slot};
}

mbk::ExpertMatrix expert_matrix(const mbk_expert_matrix *m, int64_t rows) {
    need(m != nullptr, "null matrix");
    need(m->cols >= 1, "cols must be positive");
    need(m->cols <= (1 << 30), "cols must be at most 2^30");
    need(m->data || !rows, "null matrix data");
    // no element twice: rows apart by a row's columns, or columns by a column's rows
    const int64_t rs = m->row_stride, cs = m->col_stride;
    need(rs >= 1 && cs >= 1 && rs <= MOST_STRIDE && cs <= MOST_STRIDE &&
             ((m->cols - 1) <= (rs - 1) / cs || rows - 1 <= (cs - 1) / rs),
         "row_stride and col_stride must be in 1..2^40 and keep the elements apart");
    return {m->data, m->row_stride, m->col_stride, m->cols, is_bf16(m->type), m->blocked != 0};
}

}  // namespace

extern "C" {

int mbk_xent(mbk_context *ctx, const mbk_xent_shape *shape, const void *h, const void *w,
             const float *bias, const int32_t *labels, const float *weights, float *loss,
             float *lse, char **err) {
    return mb::guarded(err, [&]() -> int {
        run_xent(ctx, xent_call(shape, h, w, bias, labels, weights, loss, lse));
        return 0;
    }, -1);
}

int mbk_xent_grad(mbk_context *ctx, const mbk_xent_shape *shape, const void *h, const void *w,
                  const float *bias, const int32_t *labels, const float *weights, float *loss,
                  float *lse, void *dh, void *dw, float *dbias, char **err) {
    return mb::guarded(err, [&]() -> int {
        mbk::XentCall c = xent_call(shape, h, w, bias, labels, weights, loss, lse);
        c.grad = dh || dw || dbias;
        c.dh = dh;
        c.dw = dw;
        c.dbias = dbias;
        run_xent(ctx, c);
        return 0;
    }, -1);
}

int mbk_expert_sort(mbk_context *ctx, const mbk_expert_plan *plan, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::ExpertPlan p = expert_plan(plan);
        need(ctx != nullptr, "null kernel-seam context");
        mb::OnDevice here(mb::context_device(ctx));
        const int cus = mb::context_cus(ctx);
        std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
        char *scratch = mb::context_scratch(ctx, mbk::expert_scratch(p, cus));
        MB_HIP(mbk::launch_expert_sort(mb::context_stream(ctx), p, cus, scratch));
        return 0;
    }, -1);
}

int mbk_expert_gather(mbk_context *ctx, const mbk_expert_plan *plan, const mbk_expert_matrix *x,
                      void *sorted, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::ExpertPlan p = expert_plan(plan);
        const mbk::ExpertMatrix m = expert_matrix(x, p.rows);
        need(sorted || !p.rows, "null argument");
        need(ctx != nullptr, "null kernel-seam context");
        if (!p.rows) return 0;
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_expert_gather(mb::context_stream(ctx), p, m, sorted));
        return 0;
    }, -1);
}

int mbk_expert_combine(mbk_context *ctx, const mbk_expert_plan *plan, const void *sorted,
                       const float *weights, const mbk_expert_matrix *out, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::ExpertPlan p = expert_plan(plan);
        const mbk::ExpertMatrix m = expert_matrix(out, p.rows);
        need(sorted || !p.rows, "null argument");
        need(ctx != nullptr, "null kernel-seam context");
        if (!p.rows) return 0;
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_expert_combine(mb::context_stream(ctx), p, sorted, weights, m));
        return 0;
    }, -1);
}

int mbk_expert_combine_grad(mbk_context *ctx, const mbk_expert_plan *plan,
                            const mbk_expert_matrix *dout, const void *sorted,
                            const float *weights, void *d_sorted, float *d_weights, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::ExpertPlan p = expert_plan(plan);
        const mbk::ExpertMatrix m = expert_matrix(dout, p.rows);
        need((sorted && d_sorted && d_weights) || !p.rows, "null argument");
        need(ctx != nullptr, "null kernel-seam context");
        if (!p.rows) return 0;
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_expert_combine_grad(mb::context_stream(ctx), p, m, sorted, weights,
                                               d_sorted, d_weights));
        return 0;
    }, -1);
}

}  // extern "C"
