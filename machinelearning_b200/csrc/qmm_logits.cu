// Logits of the next token before sampling (sm_100a): penalties for repeated
// tokens, biases and a grammar mask in one pass over the vocabulary. Per row,
// with seen = the token is in the history, count = how often it is in the
// history after the prompt:
//
//   x' = seen ? (x > 0 ? x / r : x r) : x           (repetition r)
//   x' = x' - f count - p [count > 0]               (frequency f, presence p)
//   x' = x' + sum of the token's biases, in list order
//   x' = mask bit set ? x' : -infinity
#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"

namespace qmm {

namespace {

constexpr int kThreads = 512;
constexpr int kSlice = 8192;  // vocabulary entries per CTA, one counter each
constexpr uint32_t kInPrompt = 0x80000000u;

// A CTA owns a slice of one row's vocabulary: it counts the history's tokens
// that fall into the slice in shared memory (integer atomics: the order does
// not matter), then streams the slice.
__global__ void __launch_bounds__(kThreads) process_logits_kernel(const LogitsArgs a) {
    __shared__ uint32_t count[kSlice];
    __shared__ int ids[kMaxBias];
    const int row = blockIdx.y;
    const int v0 = blockIdx.x * kSlice;
    const int len = min(kSlice, a.vocab - v0);
    const float* x = a.logits + row * a.ld + v0;
    float* y = a.out + row * a.ld_out + v0;
    for (int i = threadIdx.x; i < len; i += kThreads) count[i] = 0;
    for (int i = threadIdx.x; i < a.n_bias; i += kThreads) ids[i] = a.bias_ids[(int64_t)row * a.n_bias + i];
    __syncthreads();
    if (a.tokens) {
        const int total = min(max(a.token_lengths[row], 0), a.max_tokens);
        const int prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
        const int* tok = a.tokens + row * a.ld_tokens;
        for (int i = threadIdx.x; i < total; i += kThreads) {
            const unsigned t = (unsigned)(tok[i] - v0);
            if (tok[i] >= v0 && t < (unsigned)len) {
                if (i < prompt) atomicOr(&count[t], kInPrompt);
                else atomicAdd(&count[t], 1u);
            }
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float pres = a.presence ? a.presence[row] : 0.0f;
    const float freq = a.frequency ? a.frequency[row] : 0.0f;
    int mrow = a.mask ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
    if (mrow >= a.n_masks) mrow = -1;
    const int* mask = mrow >= 0 ? a.mask + (int64_t)mrow * ((a.vocab + 31) / 32) : nullptr;
    auto value = [&](int i, float v) {
        const uint32_t c = count[i];
        if (c) {
            v = v > 0.0f ? v / rep : v * rep;
            const uint32_t n = c & ~kInPrompt;
            if (n) v = v - freq * (float)n - pres;
        }
        return v;
    };
    auto allowed = [&](int i) {
        const int t = v0 + i;
        return !mask || ((mask[t >> 5] >> (t & 31)) & 1);
    };
    // the biased entries first: in place, their logits are still there
    for (int j = threadIdx.x; j < a.n_bias; j += kThreads) {
        const int i = ids[j] - v0;
        if (ids[j] < v0 || i >= len) continue;
        bool leader = true;
        for (int k = 0; k < j && leader; ++k) leader = ids[k] != ids[j];
        if (!leader) continue;
        float v = value(i, x[i]);
        for (int k = j; k < a.n_bias; ++k)
            if (ids[k] == ids[j]) v += a.bias_values[(int64_t)row * a.n_bias + k];
        y[i] = allowed(i) ? v : -INFINITY;
        count[i] = 0xffffffffu;  // done
    }
    __syncthreads();
    for (int i = threadIdx.x; i < len; i += kThreads)
        if (count[i] != 0xffffffffu) y[i] = allowed(i) ? value(i, x[i]) : -INFINITY;
}

}  // namespace

cudaError_t launch_process_logits(const LogitsArgs& a, cudaStream_t st) {
    if (a.rows <= 0 || a.vocab <= 0) return cudaSuccess;
    process_logits_kernel<<<dim3((a.vocab + kSlice - 1) / kSlice, a.rows), kThreads, 0, st>>>(a);
    note_launch();
    return cudaGetLastError();
}

}  // namespace qmm
