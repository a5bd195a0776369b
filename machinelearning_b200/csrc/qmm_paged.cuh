// Shared by the kernels over a paged key/value cache (qmm_paged.cu,
// qmm_paged_attention.cu, qmm_evict.cu) and their C entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace qmm {

enum KvType : int { kKvF32 = 0, kKvF16 = 1, kKvBF16 = 30 };  // GGML type ids

constexpr int kMinPage = 16;  // an attention tile of 16 slots lies in one page

// A layer's pages: row (page p, kv head h, slot s) of head_dim values starts
// at k + p * page_stride + h * head_stride + s * slot_stride (elements; the
// same in v). table[seq * table_stride + i] is the page of slots
// [i * page, (i + 1) * page) of a sequence; an entry outside [0, n_pages)
// names no page (its slots are neither read nor written).
struct PagedKv {
    void* k;
    void* v;
    int dtype;
    int nkv, hd;
    int page_shift;  // log2 of the page size
    int64_t n_pages;
    int64_t page_stride, head_stride, slot_stride;
    const int* table;
    int n_seqs, max_pages;
    int64_t table_stride;

    __host__ __device__ int64_t capacity() const { return (int64_t)max_pages << page_shift; }
    // Element offset of slot `slot` (0 <= slot < capacity) of sequence `seq`,
    // head `h`; -1 where the table names no page.
    __device__ __forceinline__ int64_t row(int seq, int h, int64_t slot) const {
        const int page = table[seq * table_stride + (slot >> page_shift)];
        if (page < 0 || page >= n_pages) return -1;
        return page * page_stride + h * head_stride + (slot & ((1 << page_shift) - 1)) * slot_stride;
    }
};

// SMs of the current device; a B200's where there is none.
inline int paged_sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
        return 148;
    return sms;
}

inline int kv_type_size(int dtype) { return dtype == kKvF32 ? 4 : ((dtype == kKvF16 || dtype == kKvBF16) ? 2 : 0); }

template <typename T>
__device__ __forceinline__ float kv_to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
    else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T f32_to_kv(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

struct AppendArgs {
    PagedKv kv;
    const float* qkv;  // rows of (nq + 2 nkv) hd values, ld apart
    int64_t ld;
    int tokens, nq;
    const float* q_norm;  // null: no norm
    const float* k_norm;
    float offset, eps;
    const float* cos_t;  // [ctx][hd / 2]
    const float* sin_t;
    int ctx;
    const int* positions;
    const int* slots;
    const int* seqs;  // null: token i belongs to sequence i
    float* q_out;     // [tokens][nq][hd]
};
cudaError_t launch_paged_append(const AppendArgs& a, bool interleaved, cudaStream_t st);

struct AttendArgs {
    PagedKv kv;
    const float* q;  // [n_seqs] rows of nq hd values, ldq apart
    int64_t ldq;
    int nq;
    const int* lengths;
    float scale;
    int window;  // 0: all slots
    const float* weights;  // null, or [n_seqs][nkv][capacity]
    float* weights_out;
    float* out;  // [n_seqs][nq][hd]
};
size_t paged_attention_workspace(const PagedKv& kv, int nq, bool weights);
cudaError_t launch_paged_attention(const AttendArgs& a, void* ws, cudaStream_t st);

struct EvictArgs {
    PagedKv kv;
    const int* lengths;         // [n_seqs]
    const float* weights;       // [n_seqs][nkv][capacity]
    const int* positions;       // [n_seqs][nkv][capacity]
    const int* next_positions;  // [n_seqs]
    int budget, recent;
    int* lengths_out;
    float* weights_out;
    int* positions_out;
};
size_t paged_evict_workspace(const PagedKv& kv, int budget);
cudaError_t launch_paged_evict(const EvictArgs& a, void* ws, cudaStream_t st);

struct LogitsArgs {
    const float* logits;
    int64_t ld;
    int rows, vocab;
    const int* tokens;  // null: no history; rows ld_tokens apart
    int64_t ld_tokens;
    int max_tokens;
    const int* token_lengths;
    const int* prompt_lengths;  // null: no prompt
    const float* repetition;    // null: 1
    const float* presence;      // null: 0
    const float* frequency;     // null: 0
    const int* bias_ids;        // null: none; [rows][n_bias]
    const float* bias_values;
    int n_bias;
    const int* mask;  // null: none; [n_masks][(vocab + 31) / 32]
    int n_masks;
    const int* mask_rows;  // null: row i uses mask i
    float* out;
    int64_t ld_out;
};
constexpr int kMaxBias = 1024;
constexpr int kMaxHistory = (1 << 30) - 1;  // a token's count and two flags share a word
cudaError_t launch_process_logits(const LogitsArgs& a, cudaStream_t st);

}  // namespace qmm
