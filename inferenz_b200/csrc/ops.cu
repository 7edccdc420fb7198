// ops.cu -- the C entries of the 8-bit floating point operators (include/inzg.h): argument checks, the context's
// device and stream, launch, status. They allocate nothing and keep nothing; of the context they use its device, stream
// and error word.
#include <cuda_runtime.h>

#include "../../include/inzg.h"
#include "host/op_check.h"
#include "inzg_internal.h"
#include "k_launch.h"

// defined in ctx.cu (hidden)
extern "C" void inzg__op_view(const inzg_ctx *ctx, int *device, int *num_sms, int *lists_cluster, void **stream,
                              int32_t **err);
extern "C" void inzg__set_error(inzg_ctx *ctx, const char *msg);

namespace {

constexpr size_t kErrLen = 160;

// the context's device for the duration of a call
struct OpDevice {
    int saved = -1, device = 0, num_sms = 0, lists_cluster = 1;
    cudaStream_t st = nullptr;
    int32_t *err = nullptr;
    cudaError_t e = cudaSuccess;
    OpDevice(const inzg_ctx *c, void *stream) {
        void *own = nullptr;
        inzg__op_view(c, &device, &num_sms, &lists_cluster, &own, &err);
        st = static_cast<cudaStream_t>(stream ? stream : own);
        e = cudaGetDevice(&saved);
        if (e == cudaSuccess && saved != device) e = cudaSetDevice(device);
    }
    ~OpDevice() {
        if (saved >= 0 && saved != device) cudaSetDevice(saved);
    }
};

inzg_status refuse(inzg_ctx *c, inzg_status st, const char *msg) {
    inzg__set_error(c, msg);
    return st;
}

// runs `launch` on the context's device; launch returns the number of kernels, or -1 when no tensor map could be made
template <class F>
inzg_status run(inzg_ctx *c, void *stream, const char *what, F launch) {
    OpDevice d(c, stream);
    if (d.e == cudaSuccess) {
        if (launch(d) < 0) return refuse(c, INZG_UNSUPPORTED, what);
        d.e = cudaGetLastError();
    }
    return d.e == cudaSuccess ? INZG_OK : refuse(c, INZG_CUDA, cudaGetErrorString(d.e));
}

}  // namespace

extern "C" {

inzg_status inzg_rmsnorm_q8(inzg_ctx *c, const inzg_rmsnorm_q8_args *a) {
    if (!c) return INZG_BAD_ARG;
    char msg[kErrLen];
    const inzg_status s = inzg__check_rmsnorm_q8(a, msg, sizeof(msg));
    if (s != INZG_OK) return refuse(c, s, msg);
    if (a->n == 0) return INZG_OK;
    return run(c, a->stream, "rmsnorm_q8", [&](const OpDevice &d) { return inzg::launch_rmsnorm_q8(*a, d.num_sms, d.st); });
}

inzg_status inzg_silu_mul_q8(inzg_ctx *c, const inzg_silu_mul_q8_args *a) {
    if (!c) return INZG_BAD_ARG;
    char msg[kErrLen];
    const inzg_status s = inzg__check_silu_mul_q8(a, msg, sizeof(msg));
    if (s != INZG_OK) return refuse(c, s, msg);
    if (a->n == 0) return INZG_OK;
    return run(c, a->stream, "silu_mul_q8", [&](const OpDevice &d) { return inzg::launch_silu_mul_q8(*a, d.num_sms, d.st); });
}

inzg_status inzg_expert_lists(inzg_ctx *c, int n, int topk, int n_expert, const int32_t *sel, const float *w, int32_t *off,
                              int32_t *rows, int32_t *slots, float *w_out, void *stream) {
    if (!c) return INZG_BAD_ARG;
    char msg[kErrLen];
    const inzg_status s = inzg__check_expert_lists(n, topk, n_expert, sel, w, off, rows, slots, w_out, msg, sizeof(msg));
    if (s != INZG_OK) return refuse(c, s, msg);
    return run(c, stream, "expert_lists", [&](const OpDevice &d) {
        return inzg::launch_expert_lists(n, topk, n_expert, sel, w, off, rows, slots, w_out, d.lists_cluster, d.err, d.st);
    });
}

inzg_status inzg_matmul_q8(inzg_ctx *c, const inzg_matmul_q8_args *a) {
    if (!c) return INZG_BAD_ARG;
    char msg[kErrLen];
    const inzg_status s = inzg__check_matmul_q8(a, msg, sizeof(msg));
    if (s != INZG_OK) return refuse(c, s, msg);
    if (a->m == 0) return INZG_OK;
    inzg_grouped_matmul_args g{};  // one group of all rows
    g.type = INZG_T_E4M3;
    g.groups = 1;
    g.n = a->n;
    g.k = a->k;
    g.a_rows = g.entries = g.out_rows_n = a->m;
    g.a = a->a;
    g.lda = a->lda;
    g.a_scale = a->a_scale;
    g.lda_scale = a->lda_scale;
    g.w = a->w;
    g.ldw = a->ldw;
    g.w_scale = a->w_scale;
    g.out = a->out;
    g.ldo = a->ldo;
    g.out_type = a->out_type;
    return run(c, a->stream, "matmul_q8: no tensor map for these operands",
               [&](const OpDevice &d) { return inzg::launch_grouped_matmul(g, d.num_sms, d.err, d.st); });
}

inzg_status inzg_grouped_matmul(inzg_ctx *c, const inzg_grouped_matmul_args *a) {
    if (!c) return INZG_BAD_ARG;
    char msg[kErrLen];
    const inzg_status s = inzg__check_grouped_matmul(a, msg, sizeof(msg));
    if (s != INZG_OK) return refuse(c, s, msg);
    if (a->entries == 0) return INZG_OK;
    return run(c, a->stream, "grouped_matmul: no tensor map for these operands",
               [&](const OpDevice &d) { return inzg::launch_grouped_matmul(*a, d.num_sms, d.err, d.st); });
}

}  // extern "C"
