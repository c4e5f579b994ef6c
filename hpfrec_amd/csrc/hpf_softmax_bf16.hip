// hpf_softmax_bf16.hip -- the bfloat16 kernels of hpf_softmax_dev.h.
#include "hpf_softmax_dev.h"

int64_t hpf_softmax::run_bf16(const Call &C)
{
    if (is_few(C))
        return run_few<B16>(C);
    return C.k <= 256 ? run_any_narrow<B16>(C) : run_wide<B16>(C);
}
