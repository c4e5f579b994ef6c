// hpf_softmax.hip -- the C entries of the full-catalogue softmax loss (kernels and formulas: hpf_softmax_dev.h).
#include "hpf_softmax_dev.h"

namespace {

using hpf_softmax::Call;

int64_t run(int type, const Call &C) { return type == HPF_F32 ? hpf_softmax::run_f32(C) : type == HPF_BF16 ? hpf_softmax::run_bf16(C) : hpf_softmax::run_f16(C); }

bool sizes_ok(int64_t n, int64_t v, int64_t k) { return n >= 0 && v > 0 && k > 0 && n < hpf_softmax::kNoTarget - 31 && v < hpf_softmax::kNoTarget - 31 && k < (1 << 20); }

bool scale_ok(float scale) { return fabsf(scale) < 0x1p127f; }    // (times log2(e) it is a number)

}  // namespace

extern "C" int64_t hpf_hip_softmax_workspace(int64_t n, int64_t v, int64_t k, int type, int grad, int cu_count)
{
    if (!sizes_ok(n, v, k) || cu_count <= 0)
        return HPF_EINVAL;
    if (type < HPF_F32 || type > HPF_F16)
        return HPF_EUNSUPPORTED;
    if (n == 0)
        return 0;
    Call C = {};
    C.n = n;
    C.v = v;
    C.k = k;
    C.grad = grad != 0;
    C.cus = cu_count;
    return run(type, C);
}

extern "C" int hpf_hip_softmax_nll(const void *x, int64_t ldx, const void *items, int64_t ld_items, const int64_t *target, const float *bias,
                                   float scale, int64_t n, int64_t v, int64_t k, int type, float *loss, float *lse, void *workspace,
                                   int64_t workspace_bytes, int cu_count, void *stream)
{
    if (!sizes_ok(n, v, k) || cu_count <= 0 || ldx < k || ld_items < k || !scale_ok(scale))
        return HPF_EINVAL;
    if (type < HPF_F32 || type > HPF_F16)
        return HPF_EUNSUPPORTED;
    if (n == 0)
        return 0;
    if (!x || !items || !target || !loss || !workspace || ((uintptr_t)workspace & 255))
        return HPF_EINVAL;
    Call C = {};
    C.x = x;
    C.w = items;
    C.target = target;
    C.bias = bias;
    C.loss = loss;
    C.lse = lse;
    C.n = n;
    C.v = v;
    C.k = k;
    C.ldx = ldx;
    C.ldw = ld_items;
    C.scale = scale;
    C.cus = cu_count;
    C.ws = (char *)workspace;
    C.ws_bytes = workspace_bytes;
    C.st = (hipStream_t)stream;
    return (int)run(type, C);
}

extern "C" int hpf_hip_softmax_nll_grad(const void *x, int64_t ldx, const void *items, int64_t ld_items, const int64_t *target,
                                        const float *weight, const float *bias, float scale, int64_t n, int64_t v, int64_t k, int type,
                                        float *loss, void *dx, int64_t ld_dx, void *ditems, int64_t ld_ditems, float *dbias, void *workspace,
                                        int64_t workspace_bytes, int cu_count, void *stream)
{
    if (!sizes_ok(n, v, k) || cu_count <= 0 || ldx < k || ld_items < k || ld_dx < k || ld_ditems < k || !scale_ok(scale))
        return HPF_EINVAL;
    if (type < HPF_F32 || type > HPF_F16)
        return HPF_EUNSUPPORTED;
    if (!ditems || (bias != nullptr) != (dbias != nullptr))
        return HPF_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    if (n == 0) {              // no rows: the items' gradients are zero
        using hpf_softmax::zero_rows_kernel;
        if (type == HPF_F32)
            zero_rows_kernel<<<1024, 256, 0, st>>>((float *)ditems, v, (int)k, ld_ditems);
        else
            zero_rows_kernel<<<1024, 256, 0, st>>>((_Float16 *)ditems, v, (int)k, ld_ditems);
        if (dbias)
            zero_rows_kernel<<<64, 256, 0, st>>>(dbias, v, 1, 1);
        return (int)hipGetLastError();
    }
    if (!x || !items || !target || !loss || !dx || !workspace || ((uintptr_t)workspace & 255))
        return HPF_EINVAL;
    Call C = {};
    C.x = x;
    C.w = items;
    C.target = target;
    C.weight = weight;
    C.bias = bias;
    C.loss = loss;
    C.dx = dx;
    C.dw = ditems;
    C.dbias = dbias;
    C.n = n;
    C.v = v;
    C.k = k;
    C.ldx = ldx;
    C.ldw = ld_items;
    C.lddx = ld_dx;
    C.lddw = ld_ditems;
    C.scale = scale;
    C.grad = true;
    C.cus = cu_count;
    C.ws = (char *)workspace;
    C.ws_bytes = workspace_bytes;
    C.st = st;
    return (int)run(type, C);
}
