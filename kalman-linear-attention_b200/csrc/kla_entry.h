// What the entry points of one translation unit (kla_capi.cu) lend to those of the others.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace kla {

struct WaitCtl;

namespace entry {

int cuda_fail(cudaError_t e);  // remembers the error for kla_b200_strerror; KLA_B200_ECUDA
void count_launch();
int wait_ctl(WaitCtl *w);      // the current device's status word with the wait settings; a C-ABI status

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn();

}  // namespace entry
}  // namespace kla
