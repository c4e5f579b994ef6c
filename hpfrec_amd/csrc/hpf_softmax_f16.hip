// hpf_softmax_f16.hip -- the float16 kernels of hpf_softmax_dev.h.
#include "hpf_softmax_dev.h"

int64_t hpf_softmax::run_f16(const Call &C)
{
    if (is_few(C))
        return run_few<H16>(C);
    return C.k <= 256 ? run_any_narrow<H16>(C) : run_wide<H16>(C);
}
