// zz_fp8_gated.hip -- zz_fp8_ep.h's kernels for gated pairs of matrices.
#include "zz_fp8_ep.h"

int zz_launch_fp8_gated(const ZzF8EpCall &c, hipStream_t st) {
    return (c.dtype == 0 ? launch_ep<float, 2>(c, st) : launch_ep<zz_bf16, 2>(c, st)) && hipGetLastError() == hipSuccess;
}
