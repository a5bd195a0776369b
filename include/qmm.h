/*
 * qmm.h -- C ABI of the B200 (sm_100a) quantized-matmul library (libqmm.so).
 *
 * Drop-in device path for the quantized-matmul hot path of
 * sweengineeringlabs/machinelearning (crate swe-llmmodel-kernel, called from
 * Linear::forward). Every entry point is `extern "C"`, takes plain pointers and
 * sizes, returns a qmm_status, never throws, never aborts the process, and
 * frees only what it allocated (conventions of the reference's FFI crate,
 * llminference/main/features/inference/ffi/main/src/lib.rs:12-40).
 *
 * Reference files cited below are paths inside the reference project.
 *
 * Weights are the raw GGUF / quantizer block bytes, uploaded unchanged:
 *   Q8_0 (id 8)  34 B / 32 values  [f16 d][32 x i8]            d*q
 *   Q4_0 (id 2)  18 B / 32 values  [f16 d][16 nibble bytes]    d*(n-8)
 *   Q4_1 (id 3)  20 B / 32 values  [f16 d][f16 m][16 nibble bytes]  d*n+m
 * Nibble order is GGML's (low nibble of byte j = element j, high = j+16), the
 * order every reference matmul reads (simd.rs:30-52).
 */
#ifndef QMM_H
#define QMM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QMM_API __attribute__((visibility("default")))

/* Status codes. 1-4 mirror QuantError (kernel/main/src/api/error.rs:5-18). */
typedef enum qmm_status {
    QMM_OK = 0,
    QMM_ERR_BLOCK_ALIGNMENT = 1, /* in_features (or element count) not a multiple of 32 */
    QMM_ERR_SHAPE_MISMATCH = 2,  /* a buffer is shorter than the shape needs (the reference panics) */
    QMM_ERR_DTYPE_MISMATCH = 3,  /* unknown or unsupported block type */
    QMM_ERR_INVALID_DATA = 4,
    QMM_ERR_CUDA = 5,            /* a CUDA call failed; see qmm_last_error_message() */
    QMM_ERR_NCCL = 6,
    QMM_ERR_TIMEOUT = 7,         /* a bounded device-side wait gave up (see qmm_device_error) */
    QMM_ERR_INVALID_INPUT = 8,   /* null pointer, misaligned pointer, bad enum */
    QMM_ERR_NO_DEVICE = 9        /* no CUDA device / the library's kernels cannot run here */
} qmm_status;

/* Block types (GGML ids, gguf/main/src/api/types.rs:8-12). */
typedef enum qmm_dtype { QMM_Q4_0 = 2, QMM_Q4_1 = 3, QMM_Q8_0 = 8 } qmm_dtype;

/* Activation handling, the reference's Linear flags (linear.rs:24-29):
 *   QMM_ACT_F32  : f32 activations x dequantised weights   (matmul_f32_q4 / _q8 / _q4_1)
 *   QMM_ACT_Q8_0 : activations quantised to Q8_0, integer block dots
 *                  (matmul_f32_q4_native / _q8_v2 / _q4_1_native; use_native_q4/q8 = true).
 *                  Q8_0 weights use quantize_q8_0 (quantize.rs:451), Q4 weights use
 *                  quantize_row_q8_0 (quantize.rs:676), exactly as the reference. */
typedef enum qmm_act { QMM_ACT_F32 = 0, QMM_ACT_Q8_0 = 1 } qmm_act;

QMM_API int qmm_version(void);
QMM_API const char* qmm_status_string(int status);
/* Detail of the last failing call on this host thread ("" if none). */
QMM_API const char* qmm_last_error_message(void);
/* Number of CUDA devices the library can use (0 on a host without GPUs). */
QMM_API int qmm_device_count(void);
/* Reads and clears the device-side error word of `device` (0 = none, 1 = a
 * bounded wait timed out). Synchronises the device. */
QMM_API int qmm_device_error(int device, int* out_error);
/* The same check as a status: synchronises `device`, reads and clears its
 * error word, and returns QMM_OK, or QMM_ERR_TIMEOUT when a bounded wait of a
 * kernel gave up since the last check (the reference's FFI turns every
 * failure into a code, ffi/main/src/lib.rs:15-21). */
QMM_API int qmm_device_status(int device);
/* Launches, on `stream`, one wait on a shared-memory barrier that nothing
 * completes, bounded to `probes` probes (1..2^20) instead of the library's
 * 2^20, after which the kernel records a timeout in the error word and
 * returns, as every wait of the hot path does. For testing the timeout path
 * without hanging or faulting a GPU: qmm_device_status then reports
 * QMM_ERR_TIMEOUT and the context stays usable. No counterpart in the
 * reference (a CPU library). */
QMM_API int qmm_selftest_bounded_wait(unsigned probes, void* stream);
/* Number of kernel launches this library has issued in this process (stream
 * captures included), for launch accounting in benchmarks. No counterpart in
 * the reference (a CPU library). */
QMM_API unsigned long long qmm_launch_count(void);

/* ------------------------------------------------------------------------
 * Reference-signature host entry points. Host buffers in, host buffers out,
 * exactly the arguments of the Rust functions they replace; `output` holds
 * m*out_features floats. Each call runs on the current CUDA device and
 * synchronises. If `weight_bytes` was registered with
 * qmm_register_host_weight(), its resident device copy is used; otherwise the
 * weights are copied to the device for this call.
 * ------------------------------------------------------------------------ */
/* matmul_f32_q8 (quantize.rs:297-303) */
QMM_API int qmm_matmul_f32_q8(const float* input_data, size_t input_len, const uint8_t* weight_bytes,
                              size_t weight_len, size_t m, size_t in_features, size_t out_features,
                              float* output);
/* matmul_f32_q8_v2 (quantize.rs:429-435) */
QMM_API int qmm_matmul_f32_q8_v2(const float* input_data, size_t input_len, const uint8_t* weight_bytes,
                                 size_t weight_len, size_t m, size_t in_features, size_t out_features,
                                 float* output);
/* matmul_f32_q4 (quantize.rs:535-541) */
QMM_API int qmm_matmul_f32_q4(const float* input_data, size_t input_len, const uint8_t* weight_bytes,
                              size_t weight_len, size_t m, size_t in_features, size_t out_features,
                              float* output);
/* matmul_f32_q4_native (quantize.rs:646-652) */
QMM_API int qmm_matmul_f32_q4_native(const float* input_data, size_t input_len, const uint8_t* weight_bytes,
                                     size_t weight_len, size_t m, size_t in_features, size_t out_features,
                                     float* output);
/* matmul_f32_q4_1 (quantize.rs:807-813) */
QMM_API int qmm_matmul_f32_q4_1(const float* input_data, size_t input_len, const uint8_t* weight_bytes,
                                size_t weight_len, size_t m, size_t in_features, size_t out_features,
                                float* output);
/* matmul_f32_q4_1_native (quantize.rs:938-944) */
QMM_API int qmm_matmul_f32_q4_1_native(const float* input_data, size_t input_len, const uint8_t* weight_bytes,
                                       size_t weight_len, size_t m, size_t in_features, size_t out_features,
                                       float* output);

/* quantize_q8_0 (quantize.rs:15-48): n % 32 == 0, out holds n/32*34 bytes. */
QMM_API int qmm_quantize_q8_0(const float* data, size_t n, uint8_t* out);
/* quantize_q4_0 (quantize.rs:124-165, interleaved nibble packing as the reference writes it). */
QMM_API int qmm_quantize_q4_0(const float* data, size_t n, uint8_t* out);
/* quantize_q4_1 (quantize.rs:207-251). */
QMM_API int qmm_quantize_q4_1(const float* data, size_t n, uint8_t* out);
/* quantize_row_q8_0 (quantize.rs:260-289): also writes the f32(f16) scales (n/32 floats). */
QMM_API int qmm_quantize_row_q8_0(const float* input, size_t n, uint8_t* out, float* scales);
/* Tensor::to_f32 for block types (tensor.rs:527-630; Q4_0 in GGML order). */
QMM_API int qmm_dequantize(int dtype, const uint8_t* raw, size_t raw_len, size_t n_elements, float* out);

/* Registers a host weight buffer (e.g. an mmap'd GGUF tensor, tensor.rs:405-414)
 * whose bytes are uploaded once to the current device and reused by the
 * reference-signature calls above for as long as it stays registered. The
 * caller must not change those bytes while registered. */
QMM_API int qmm_register_host_weight(const uint8_t* weight_bytes, size_t weight_len, int dtype, size_t n, size_t k);
QMM_API int qmm_unregister_host_weight(const uint8_t* weight_bytes);

/* ------------------------------------------------------------------------
 * Device API (the hot path). Pointers ending in _dev are device pointers;
 * `stream` is a cudaStream_t (NULL = legacy default stream). Calls are
 * asynchronous on `stream` and do not synchronise.
 * ------------------------------------------------------------------------ */
typedef struct qmm_weight qmm_weight;

/* Uploads an [n, k] block matrix (n rows of k/32 blocks, the GGUF layout) to
 * `device` with one host-to-device copy, byte for byte, no repacking. */
QMM_API int qmm_weight_create(int dtype, size_t n, size_t k, const uint8_t* host_bytes, size_t len, int device,
                              qmm_weight** out);
/* Same, from bytes already on `device` (device-to-device copy). */
QMM_API int qmm_weight_create_from_device(int dtype, size_t n, size_t k, const uint8_t* dev_bytes, size_t len,
                                          int device, qmm_weight** out);
QMM_API int qmm_weight_destroy(qmm_weight* w);
QMM_API int qmm_weight_info(const qmm_weight* w, int* dtype, size_t* n, size_t* k, const uint8_t** dev_bytes,
                            int* device);

/* Activation functions (qmm_gated_forward: GELU and SiLU; qmm_gated_act_dev:
 * all three). */
#define QMM_GELU 0
#define QMM_SILU 1
#define QMM_RELU 2

/* Fused projections (reference: Attention::fuse_qkv_weights,
 * llmserve/llmmodel/layers/main/src/core/attention.rs:306-339, and
 * FeedForward::fuse_gate_up_weights, feed_forward.rs:147-187).
 *
 * qmm_weight_fuse_rows: a new weight whose bytes are the parts' bytes
 * concatenated in order (rows = sum of the parts' rows), as the reference's
 * fused QKV / gate+up tensors are; y of the fused weight is the parts' outputs
 * side by side. Parts: same block type (Q8_0, Q4_0 or Q4_1; the reference fuses
 * Q8_0 only), same in_features, same device. The parts stay valid.
 *
 * qmm_weight_fuse_gate_up: a gate/up weight for qmm_gated_forward. Same rules,
 * plus gate and up of equal shape [hidden, k]. Its rows interleave gate and up
 * in groups of 16 (rows 32j..32j+15 = gate rows 16j.., rows 32j+16..32j+31 = up
 * rows 16j..), zero rows padding hidden to a multiple of 16, so one output tile
 * of the matmul holds matching gate and up values. qmm_linear_forward rejects
 * it; qmm_weight_gate_hidden reports hidden (0 for an ordinary weight).
 *
 * qmm_gated_forward: out_dev[m][hidden] = act(x . gate^T) * (x . up^T), act =
 * QMM_GELU or QMM_SILU, the activation applied in the matmul's epilogue (one
 * launch for decode shapes). The matmul is the f32-activation form for every
 * block type, as the reference's fused Linear (use_native_* false). */
QMM_API int qmm_weight_fuse_rows(const qmm_weight* const* parts, size_t count, qmm_weight** out);
QMM_API int qmm_weight_fuse_gate_up(const qmm_weight* gate, const qmm_weight* up, qmm_weight** out);
QMM_API int qmm_weight_gate_hidden(const qmm_weight* w, size_t* hidden);
QMM_API int qmm_gated_forward(const qmm_weight* w, const float* x_dev, size_t m, float* out_dev, int act_fn,
                              void* stream);

/* 64-bit position-weighted checksum of device bytes: the sum over their
 * little-endian 32-bit words w_i (the tail zero-padded) of w_i * (2i + 1),
 * modulo 2^64 -- for verifying that an upload (a GGUF tensor's file range,
 * reference gguf/main/src/core/parser.rs:501-576) arrived byte for byte.
 * Synchronous. qmm_checksum_dev: data_dev 4-byte aligned, on the current
 * device. No counterpart in the reference (its mmap path has no device copy
 * to verify). */
QMM_API int qmm_checksum_dev(const void* data_dev, size_t len, void* stream, unsigned long long* out);
QMM_API int qmm_weight_checksum(const qmm_weight* w, unsigned long long* out);

/* y_dev[m, n] = x_dev[m, k] . W^T on the weight's device, workspace managed by
 * the library (one buffer per device and stream, grown on demand with
 * cudaMalloc; grow it with qmm_reserve_workspace before capturing a graph).
 * A graph keeps the buffer that it was captured with: a later call that needs a
 * larger one gets a new one, and the old one is not freed. Replay the graph on
 * the stream it was captured on, or while nothing else runs there. Host threads
 * may call on one stream at the same time: the launches of a call stay together. */
QMM_API int qmm_linear_forward(const qmm_weight* w, const float* x_dev, size_t m, float* y_dev, int act,
                               void* stream);
/* Host-buffer variant of qmm_linear_forward: copies x in and y out on `stream`
 * (pinned buffers make the copies asynchronous) and synchronises the stream. */
QMM_API int qmm_linear_forward_host(const qmm_weight* w, const float* x_host, size_t m, float* y_host, int act,
                                    void* stream);
QMM_API int qmm_reserve_workspace(int device, void* stream, size_t bytes);

/* Fully caller-managed form: raw device weight bytes and a caller workspace of
 * at least qmm_workspace_size() bytes (256-byte aligned, not shared by
 * concurrent calls). w_dev must be 16-byte aligned. */
QMM_API size_t qmm_workspace_size(int dtype, int act, size_t m, size_t n, size_t k);
QMM_API int qmm_matmul_dev(int dtype, int act, const float* x_dev, const uint8_t* w_dev, size_t w_len, size_t m,
                           size_t k, size_t n, float* y_dev, void* workspace_dev, size_t workspace_bytes,
                           void* stream);

/* Allocation-free form of qmm_matmul_dev (no counterpart in the reference, which
 * has no device code). For callers that may not allocate device memory: a
 * plugin whose host framework owns the device memory pool, or a serving loop
 * that cannot take cudaMalloc's implicit device-wide synchronisation. The
 * workspace is a fixed 4 MiB device array inside the library
 * (QMM_NOALLOC_SCRATCH_BYTES; held by every device that loads the library until
 * the process exits); shapes whose workspace does not fit are rejected with
 * QMM_ERR_INVALID_INPUT. The first call on a device, with that device current,
 * looks the array's address up (make it before any stream capture). The array
 * is shared: calls that overlap on the GPU race, so keep them ordered (one
 * stream, or explicit synchronisation). It runs the GEMV kernels only (rows
 * in chunks of at most 64): calls with 17 or more rows of f32 activations,
 * which qmm_matmul_dev sends to the tensor-core GEMM, are slower here.
 * Arguments as qmm_matmul_dev. */
#define QMM_NOALLOC_SCRATCH_BYTES (4u << 20)
QMM_API int qmm_matmul_dev_noalloc(int dtype, int act, const float* x_dev, const uint8_t* w_dev, size_t w_len,
                                   size_t m, size_t k, size_t n, float* y_dev, void* stream);

/* Device quantisers, bit-identical to the reference's:
 *   variant 0: quantize_q8_0   (unrounded inverse scale), dtype QMM_Q8_0
 *   variant 1: quantize_row_q8_0 (f16-rounded inverse scale), dtype QMM_Q8_0; scales_dev optional
 *   dtype QMM_Q4_0 / QMM_Q4_1: quantize_q4_0 / quantize_q4_1 (variant ignored). */
QMM_API int qmm_quantize_dev(int dtype, int variant, const float* x_dev, size_t n, uint8_t* out_dev,
                             float* scales_dev, void* stream);
/* Device dequantiser with Tensor::to_f32 semantics. */
QMM_API int qmm_dequantize_dev(int dtype, const uint8_t* w_dev, size_t w_len, size_t n_elements, float* out_dev,
                               void* stream);

/* Element-wise activation step of FeedForward::forward (reference
 * layers/main/src/core/feed_forward.rs:198-251), for gate and up produced by
 * separate matmuls or by one matmul over qmm_weight_fuse_rows(gate, up):
 * out_dev[m][hidden] = act(gate_dev[i * ld + j]) * up_dev[i * ld + j], in f32,
 * act = QMM_GELU (tanh approximation), QMM_SILU or QMM_RELU; up_dev may be null
 * (the ungated activations: out = act(gate)). ld >= hidden is the row stride of
 * gate and up in elements (2 * hidden for the [gate | up] output of a fused
 * weight, with up_dev = gate_dev + hidden). Launched with programmatic
 * dependent launch, so it overlaps the tail of the matmul before it. */
QMM_API int qmm_gated_act_dev(int act_fn, const float* gate_dev, const float* up_dev, size_t m, size_t hidden,
                              size_t ld, float* out_dev, void* stream);

/* ---- Decode-step pieces around the matmuls (device pointers, stream-ordered).
 * A Gemma-3 decode step is these plus the matmuls above (fused QKV, fused
 * gate/up with the GeGLU epilogue, o, down, lm_head). The reference runs them
 * on f32 host tensors; each entry cites the Rust code it replaces.
 * The decode position is read from device memory (pos_dev) so a captured step
 * can be replayed while qmm_add_int_dev advances it. */

/* x[b] = scale * dequant(emb row tokens[b]) from a Q8_0 [vocab][hidden] tied
 * embedding; token ids are clamped to [0, vocab). Replaces TokenEmbedding::
 * forward + mul_scalar(embedding_scale) (model/main/src/core/forward.rs:122-127). */
QMM_API int qmm_embed_q8_dev(const uint8_t* emb_dev, size_t vocab, size_t hidden, const int* tokens_dev,
                             size_t batch, float scale, float* x_dev, void* stream);
/* y = x / sqrt(mean(x^2) + eps) * (w + offset) per row; y rows ld_y floats
 * apart (0: dim; wider rows keep their tail). Replaces RMSNorm::forward
 * (layers/main/src/core/rms_norm.rs:66-85, tensor math.rs:334-380). */
QMM_API int qmm_rmsnorm_dev(const float* x_dev, const float* w_dev, float offset, float eps, size_t rows, size_t dim,
                            float* y_dev, size_t ld_y, void* stream);
/* x += rmsnorm(branch, w_post); then (w_next non-null) h = rmsnorm(x, w_next),
 * h rows ld_h floats apart (0: dim): a sandwich post-norm and residual add
 * fused with the next pre-norm (layers/main/src/core/transformer_block.rs:424-449). */
QMM_API int qmm_residual_rmsnorm_dev(float* x_dev, const float* branch_dev, const float* w_post_dev,
                                     const float* w_next_dev, float offset, float eps, size_t rows, size_t dim,
                                     float* h_dev, size_t ld_h, void* stream);
/* From fused q|k|v rows [batch][(n_heads + 2 n_kv_heads) head_dim]: per-head
 * RMSNorm of q and k, half-split RoPE with cos/sin tables [ctx][head_dim/2]
 * at position *pos_dev; q into q_out [batch][n_heads][head_dim], k and v into
 * the caches [batch][n_kv_heads][ctx][head_dim] at that position. head_dim a
 * multiple of 64, at most 256 (layers/main/src/core/attention.rs:505-540,
 * rope.rs:7-130). */
QMM_API int qmm_qk_rope_cache_dev(const float* qkv_dev, size_t batch, int n_heads, int n_kv_heads, int head_dim,
                                  const float* q_norm_dev, const float* k_norm_dev, float offset, float eps,
                                  const float* cos_dev, const float* sin_dev, const int* pos_dev, int ctx,
                                  float* q_out_dev, float* k_cache_dev, float* v_cache_dev, void* stream);
/* Floats of the partial-result buffer qmm_attention_decode_dev needs. */
QMM_API size_t qmm_attention_partial_floats(size_t batch, int n_heads, int head_dim, int ctx);
/* Single-token attention over cache positions 0..*pos_dev: scores q.k *
 * inv_scale, softmax, weighted sum of v; grouped-query heads share their kv
 * head. out [batch][n_heads * head_dim]. At most 8 heads and head_dim 256
 * (layers/main/src/core/attention.rs:545-600, decode: no mask). */
QMM_API int qmm_attention_decode_dev(const float* q_dev, const float* k_cache_dev, const float* v_cache_dev,
                                     size_t batch, int n_heads, int n_kv_heads, int head_dim, const int* pos_dev,
                                     int ctx, float inv_scale, float* partial_dev, float* out_dev, void* stream);
/* qmm_qk_rope_cache_dev and qmm_attention_decode_dev in one pass (one launch
 * fewer per layer): every attention CTA normalises and rotates the q heads
 * itself; the one holding the position writes k and v to the caches. Same
 * arguments and limits (context at most 2048). */
QMM_API int qmm_attention_decode_fused_dev(const float* qkv_dev, size_t batch, int n_heads, int n_kv_heads,
                                           int head_dim, const float* q_norm_dev, const float* k_norm_dev, float offset,
                                           float eps, const float* cos_dev, const float* sin_dev, const int* pos_dev,
                                           int ctx, float* k_cache_dev, float* v_cache_dev, float inv_scale,
                                           float* partial_dev, float* out_dev, void* stream);
/* *p_dev += value, stream-ordered (advances a captured step's position). */
QMM_API int qmm_add_int_dev(int* p_dev, int value, void* stream);

/* ---- Serving over a paged key/value cache (device pointers, stream-ordered). -----------
 * A layer's cache is a pool of pages shared by all sequences; each sequence
 * has its own length, its own pages (a block table) and any number of query
 * heads. One decode step of a layer: qmm_paged_append_dev (the new token's q,
 * k, v), qmm_paged_attention_dev, and, under a cache budget,
 * qmm_paged_evict_dev; after the lm_head, qmm_process_logits_dev. The
 * reference keeps one dense f32 cache per sequence and has none of the other
 * steps. Lengths, positions, slots and tables are read from device memory, so
 * a captured step can be replayed as they advance; values outside their range
 * are never dereferenced (each entry says what they do). */

/* Cache element types (GGML ids, gguf/main/src/api/types.rs:8-12). */
#define QMM_KV_F32 0
#define QMM_KV_F16 1
#define QMM_KV_BF16 30

/* A layer's pages. Row (page p, kv head h, slot s) is head_dim values at
 * k_dev + p * page_stride + h * head_stride + s * slot_stride, in elements, the
 * same in v_dev. k_dev, v_dev and the strides are multiples of 16 bytes.
 * head_dim: a multiple of 64, at most 256; page_size: a power of two, 16 to
 * 1024; n_heads of the calls: a multiple of n_kv_heads. Slots [i * page_size,
 * (i + 1) * page_size) of sequence s are on page table_dev[s * table_stride + i],
 * i < max_pages; its capacity is max_pages * page_size (at most 2^30). An
 * entry outside [0, n_pages) names no page: its slots are neither written nor
 * attended to. A page may be on the tables of several sequences (a shared prefix) as
 * long as its slots are only attended to: append and evict write through the table.
 * With n_seqs 0 the pointers may be null. At most 65535 sequences, kv heads and
 * query heads. */
typedef struct qmm_paged_kv {
    void* k_dev;
    void* v_dev;
    int dtype;
    int n_kv_heads;
    int head_dim;
    int page_size;
    long long n_pages;
    long long page_stride;
    long long head_stride;
    long long slot_stride;
    const int* table_dev;
    int n_seqs;
    int max_pages;
    long long table_stride;
} qmm_paged_kv;

/* For each of `tokens` fused q|k|v rows ((n_heads + 2 n_kv_heads) head_dim
 * floats, rows ld_qkv floats apart): per-head RMSNorm of q and k (q_norm_dev and
 * k_norm_dev both null: none), rotation by row positions_dev[i] of the cos/sin
 * tables [ctx][head_dim / 2] (pairs half a head apart, or, interleaved != 0,
 * neighbours), q to q_out_dev [tokens][n_heads][head_dim], k and v rounded to the
 * cache's type into slot slots_dev[i] of sequence seqs_dev[i] (seqs_dev null:
 * sequence i). The (sequence, slot) pairs are distinct. A position outside
 * [0, ctx) gives a zero q row and stores nothing; a slot or sequence outside the
 * table stores nothing (padding rows carry slot -1). Pointers 16-byte aligned,
 * ld_qkv a multiple of 4. (attention.rs:505-540, rope.rs:7-130) */
QMM_API int qmm_paged_append_dev(const qmm_paged_kv* kv, const float* qkv_dev, size_t ld_qkv, size_t tokens,
                                 int n_heads, const float* q_norm_dev, const float* k_norm_dev, float offset,
                                 float eps, const float* cos_dev, const float* sin_dev, int ctx, int interleaved,
                                 const int* positions_dev, const int* slots_dev, const int* seqs_dev,
                                 float* q_out_dev, void* stream);

/* One new token per sequence: out_dev [n_seqs][n_heads][head_dim] = softmax(scale
 * q . k) v over the sequence's slots [max(0, n - window), n), n = lengths_dev[s]
 * clamped to [0, capacity], window 0: all. A sequence without slots gives
 * zeros. q rows ld_q floats apart (a multiple of 4); float pointers 16-byte aligned.
 * weights_dev and weights_out_dev (both or neither; they may be equal), f32
 * [n_seqs][n_kv_heads][capacity]: out = in, plus at each attended slot the sum
 * over the kv head's query heads of the slot's softmax weight. A score of -infinity
 * (an infinite key) has weight 0, and a sequence with none but those gives zeros; one
 * of +infinity or NaN makes its head's output NaN; 0 times an infinite v is NaN. Sums
 * are in 32 bits; queries, weights and f32 caches go through the tensor cores as sums
 * of parts, 22 bits of f32 and f16 caches, 24 of bf16. Workspace: the library's, of
 * the current device and `stream`; reserve qmm_paged_attention_workspace_size bytes
 * before a stream capture. With weights it holds a score for every slot of the table
 * (n_seqs * n_heads * capacity floats), so size tables by what sequences can hold.
 * (attention.rs:545-600) */
QMM_API size_t qmm_paged_attention_workspace_size(const qmm_paged_kv* kv, int n_heads, int with_weights);
QMM_API int qmm_paged_attention_dev(const qmm_paged_kv* kv, const float* q_dev, size_t ld_q, int n_heads,
                                    const int* lengths_dev, float scale, int window, const float* weights_dev,
                                    float* weights_out_dev, float* out_dev, void* stream);

/* Brings every sequence down to at most `budget` slots, per kv head. Of a
 * sequence with n = lengths_dev[s] > budget slots those are kept whose position
 * positions_dev [n_seqs][n_kv_heads][capacity] is at least next_positions_dev[s]
 * - recent, then those with the largest weights_dev (same shape; NaN ranks as
 * -infinity), ties and a surplus of recent slots by the lowest slot. Kept slots
 * at or above `budget` move, in slot order, into the evicted ones below it (k and
 * v in place, so the pages below a sequence's length are on no other sequence's
 * table, nor twice on its own: others would see the moved rows); weights_out_dev and positions_out_dev (not the inputs) hold the
 * moved arrays, 0 and -1 beyond the new length; lengths_out_dev [n_seqs] (not
 * lengths_dev) the new lengths. Weights and positions 16-byte aligned; at most
 * 65535 (sequence, kv head) rows. Workspace as above. */
QMM_API size_t qmm_paged_evict_workspace_size(const qmm_paged_kv* kv, int budget);
QMM_API int qmm_paged_evict_dev(const qmm_paged_kv* kv, const int* lengths_dev, const float* weights_dev,
                                const int* positions_dev, const int* next_positions_dev, int budget, int recent,
                                int* lengths_out_dev, float* weights_out_dev, int* positions_out_dev, void* stream);

/* Logits [rows][vocab] (rows ld floats apart) before sampling, to out_dev (rows
 * ld_out apart; may be logits_dev). Row i's history is the first token_lengths_dev[i]
 * (clamped to [0, max_tokens]) ids of tokens_dev + i * ld_tokens, the first
 * prompt_lengths_dev[i] of them the prompt. A token in the history: x > 0 ? x /
 * repetition[i] : x * repetition[i]; in the history after the prompt, count
 * times: x - frequency[i] * count - presence[i]. Then x + the values of the
 * token's entries among the row's n_bias (at most 1024) bias_ids_dev, in list
 * order. Then -infinity where bit t % 32 of word t / 32 of grammar state
 * mask_rows_dev[i] of mask_dev [n_masks][ceil(vocab / 32)] is clear (a state
 * outside [0, n_masks): no mask; mask_rows_dev null: state i). Null tokens_dev,
 * bias_ids_dev or mask_dev: that step is left out; null prompt_lengths_dev: no
 * prompt; null penalties: 1, 0, 0. Ids outside [0, vocab) are ignored (bias lists
 * of uneven length are padded with -1). At most 65535 rows; max_tokens is below
 * 2^30, vocab below 2^31 - 65536. */
#define QMM_MAX_BIAS 1024
QMM_API int qmm_process_logits_dev(const float* logits_dev, size_t ld, size_t rows, size_t vocab,
                                   const int* tokens_dev, size_t ld_tokens, size_t max_tokens,
                                   const int* token_lengths_dev, const int* prompt_lengths_dev,
                                   const float* repetition_dev, const float* presence_dev,
                                   const float* frequency_dev, const int* bias_ids_dev,
                                   const float* bias_values_dev, size_t n_bias, const int* mask_dev,
                                   size_t n_masks, const int* mask_rows_dev, float* out_dev, size_t ld_out,
                                   void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QMM_H */
