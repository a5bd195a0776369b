// Appending tokens to a paged key/value cache (sm_100a): from fused q|k|v rows,
// per-head RMSNorm and position rotation of q and k, k and v into their pages
// in the cache's type, q out in f32.
//
//   x' = x / sqrt(mean(x^2) + eps) * (w + offset)          (per head vector)
//   (a, b) -> (a cos - b sin, a sin + b cos)               (per pair)
//
// The pairs of a head are (i, i + head_dim / 2), the reference's half split
// (llmserve/llmmodel/layers/main/src/core/rope.rs:7-130), or the neighbours
// (2 i, 2 i + 1), the order GGUF files of Llama-type models are written for.
#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"

namespace qmm {

namespace {

constexpr int kAppendThreads = 256;

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = v;
    } else {
        T t[4] = {f32_to_kv<T>(v.x), f32_to_kv<T>(v.y), f32_to_kv<T>(v.z), f32_to_kv<T>(v.w)};
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(t);
    }
}

// One group of G lanes (head_dim / 8 of them active) per head vector: a lane
// holds elements [4 l, 4 l + 4) of each half, whole pairs in either order.
// G: 8, 16 or 32.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a, int G) {
    const int lane = threadIdx.x & (G - 1);
    const int hd = a.kv.hd, half = hd / 2;
    const int heads = a.nq + 2 * a.kv.nkv;
    const int64_t vec = (int64_t)blockIdx.x * (kAppendThreads / G) + threadIdx.x / G;
    const int64_t token = vec / heads;
    const int head = (int)(vec - token * heads);
    const bool live = token < a.tokens && lane * 8 < hd;
    float4 x = make_float4(0, 0, 0, 0), y = x;
    int pos = -1;
    if (live) {
        const float* src = a.qkv + token * a.ld + (int64_t)head * hd;
        x = *reinterpret_cast<const float4*>(src + 4 * lane);
        y = *reinterpret_cast<const float4*>(src + half + 4 * lane);
        pos = a.positions[token];
    }
    const bool is_q = head < a.nq, is_v = head >= a.nq + a.kv.nkv;
    const float* w = is_v ? nullptr : (is_q ? a.q_norm : a.k_norm);
    // every lane of the warp takes part in the shuffles
    float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + (y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w);
    for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!live) return;
    const bool placed = pos >= 0 && pos < a.ctx;  // a rotation exists for the position
    if (w) {
        const float inv = 1.0f / sqrtf(ss / (float)hd + a.eps);
        const float4 w0 = *reinterpret_cast<const float4*>(w + 4 * lane);
        const float4 w1 = *reinterpret_cast<const float4*>(w + half + 4 * lane);
        x.x = x.x * inv * (w0.x + a.offset);
        x.y = x.y * inv * (w0.y + a.offset);
        x.z = x.z * inv * (w0.z + a.offset);
        x.w = x.w * inv * (w0.w + a.offset);
        y.x = y.x * inv * (w1.x + a.offset);
        y.y = y.y * inv * (w1.y + a.offset);
        y.z = y.z * inv * (w1.z + a.offset);
        y.w = y.w * inv * (w1.w + a.offset);
    }
    if (!is_v && placed) {
        const float* ct = a.cos_t + (int64_t)pos * half;
        const float* sn = a.sin_t + (int64_t)pos * half;
        const float4 p = x, r = y;
        if constexpr (kInterleaved) {  // pairs 2 l, 2 l + 1 of the first half, and of the second
            const float2 c0 = *reinterpret_cast<const float2*>(ct + 2 * lane);
            const float2 s0 = *reinterpret_cast<const float2*>(sn + 2 * lane);
            const float2 c1 = *reinterpret_cast<const float2*>(ct + half / 2 + 2 * lane);
            const float2 s1 = *reinterpret_cast<const float2*>(sn + half / 2 + 2 * lane);
            x = make_float4(p.x * c0.x - p.y * s0.x, p.x * s0.x + p.y * c0.x, p.z * c0.y - p.w * s0.y,
                            p.z * s0.y + p.w * c0.y);
            y = make_float4(r.x * c1.x - r.y * s1.x, r.x * s1.x + r.y * c1.x, r.z * c1.y - r.w * s1.y,
                            r.z * s1.y + r.w * c1.y);
        } else {
            const float4 c = *reinterpret_cast<const float4*>(ct + 4 * lane);
            const float4 s = *reinterpret_cast<const float4*>(sn + 4 * lane);
            x = make_float4(p.x * c.x - r.x * s.x, p.y * c.y - r.y * s.y, p.z * c.z - r.z * s.z,
                            p.w * c.w - r.w * s.w);
            y = make_float4(p.x * s.x + r.x * c.x, p.y * s.y + r.y * c.y, p.z * s.z + r.z * c.z,
                            p.w * s.w + r.w * c.w);
        }
    }
    if (is_q) {
        if (!placed) x = y = make_float4(0, 0, 0, 0);
        float* dst = a.q_out + (token * a.nq + head) * hd;
        *reinterpret_cast<float4*>(dst + 4 * lane) = x;
        *reinterpret_cast<float4*>(dst + half + 4 * lane) = y;
        return;
    }
    if (!placed) return;
    const int seq = a.seqs ? a.seqs[token] : (int)token;
    const int slot = a.slots[token];
    if (seq < 0 || seq >= a.kv.n_seqs || slot < 0 || slot >= a.kv.capacity()) return;
    const int64_t row = a.kv.row(seq, head - a.nq - (is_v ? a.kv.nkv : 0), slot);
    if (row < 0) return;
    T* dst = static_cast<T*>(is_v ? a.kv.v : a.kv.k) + row;
    store4(dst + 4 * lane, x);
    store4(dst + half + 4 * lane, y);
}

template <typename T>
cudaError_t launch_append(const AppendArgs& a, bool interleaved, cudaStream_t st) {
    const int lanes = a.kv.hd / 8;
    const int G = lanes <= 8 ? 8 : (lanes <= 16 ? 16 : 32);
    const int64_t vecs = (int64_t)a.tokens * (a.nq + 2 * a.kv.nkv);
    const int64_t per = kAppendThreads / G;
    const unsigned grid = (unsigned)((vecs + per - 1) / per);
    if (interleaved) paged_append_kernel<T, true><<<grid, kAppendThreads, 0, st>>>(a, G);
    else paged_append_kernel<T, false><<<grid, kAppendThreads, 0, st>>>(a, G);
    note_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_append(const AppendArgs& a, bool interleaved, cudaStream_t st) {
    if (a.tokens <= 0) return cudaSuccess;
    switch (a.kv.dtype) {
        case kKvF32: return launch_append<float>(a, interleaved, st);
        case kKvF16: return launch_append<__half>(a, interleaved, st);
        case kKvBF16: return launch_append<__nv_bfloat16>(a, interleaved, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace qmm
