// zz_fp8_ep.hip -- zz_fp8_ep.h's kernels for plain matrices.
#include "zz_fp8_ep.h"

int zz_launch_fp8_ep(const ZzF8EpCall &c, hipStream_t st) {
    return (c.dtype == 0 ? launch_ep<float, 1>(c, st) : launch_ep<zz_bf16, 1>(c, st)) && hipGetLastError() == hipSuccess;
}
