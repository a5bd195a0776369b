// Attention over a paged key/value cache in f32.
#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"
#include "qmm_paged_attention.cuh"

namespace qmm {
cudaError_t attend_f32(const AttendArgs& a, const AttendScratch& sc, int sms, cudaStream_t st) {
    return launch_hd<float>(a, sc, sms, st);
}
}  // namespace qmm
