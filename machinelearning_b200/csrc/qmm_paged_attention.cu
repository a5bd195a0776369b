// Attention over a paged key/value cache: workspace and choice of the kernels
// (qmm_paged_attention.cuh) by cache type.
#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"
#include "qmm_paged_attention.cuh"

namespace qmm {

namespace {

size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

// Carves the workspace; returns its size.
size_t carve(const PagedKv& kv, int nq, bool weights, int grid, void* base, AttendScratch* sc) {
    size_t off = 0;
    auto take = [&](size_t bytes) {
        void* p = static_cast<uint8_t*>(base) + off;
        off += aligned(bytes);
        return p;
    };
    const int heads = pass_heads(kv, nq);
    sc->head_tiles = (nq / kv.nkv + heads - 1) / heads;
    sc->ml = static_cast<float2*>(take((size_t)grid * 2 * heads * sizeof(float2)));
    sc->acc = static_cast<float*>(take((size_t)grid * 2 * heads * kv.hd * sizeof(float)));
    sc->whole = nullptr;
    sc->scores = nullptr;
    if (weights) {
        sc->whole = static_cast<float2*>(take((size_t)kv.n_seqs * nq * sizeof(float2)));
        sc->scores = static_cast<float*>(take((size_t)kv.n_seqs * nq * kv.capacity() * sizeof(float)));
    }
    return off;
}

}  // namespace

size_t paged_attention_workspace(const PagedKv& kv, int nq, bool weights) {
    AttendScratch sc;
    return carve(kv, nq, weights, paged_sm_count() * kMaxAttendCtas, nullptr, &sc);
}

cudaError_t launch_paged_attention(const AttendArgs& a, void* ws, cudaStream_t st) {
    if (a.kv.n_seqs <= 0) return cudaSuccess;
    const int sms = paged_sm_count();
    AttendScratch sc;
    carve(a.kv, a.nq, a.weights != nullptr, sms * kMaxAttendCtas, ws, &sc);
    switch (a.kv.dtype) {
        case kKvF32: return attend_f32(a, sc, sms, st);
        case kKvF16: return attend_f16(a, sc, sms, st);
        case kKvBF16: return attend_bf16(a, sc, sms, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace qmm
