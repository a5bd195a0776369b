// Attention over a paged key/value cache in bf16.
#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"
#include "qmm_paged_attention.cuh"

namespace qmm {
cudaError_t attend_bf16(const AttendArgs& a, const AttendScratch& sc, int sms, cudaStream_t st) {
    return launch_hd<__nv_bfloat16>(a, sc, sms, st);
}
}  // namespace qmm
