// hpf_softmax_f32.hip -- the float32 kernels of hpf_softmax_dev.h.
#include "hpf_softmax_dev.h"

int64_t hpf_softmax::run_f32(const Call &C)
{
    if (is_few(C))
        return run_few<W32>(C);
    return C.k <= 256 ? run_any_narrow<F32>(C) : run_wide<W32>(C);
}
