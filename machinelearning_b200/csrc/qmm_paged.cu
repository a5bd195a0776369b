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

// A group of G lanes (head_dim / 8 of them active; G is 8, 16 or 32) per head
// vector, CTAs of neighbouring heads of a token; a lane holds elements [4 l, 4 l + 4)
// of each half, whole pairs in either order. Bound by HBM for long prompts as long
// as a vector takes few instructions and registers (all of an SM's threads keep
// their 32 bytes on the way): exact root and divide, 64-bit index arithmetic and
// one vector per group 125 us for 8192 tokens, 64/8 heads of 128, bf16; four
// vectors a group 134 us; persistent groups with two tokens on the way 127 us, bound
// by instructions; this 102 us (6.26 TB/s).
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads, 8) paged_append_kernel(const AppendArgs a, int G) {
    const int lane4 = 4 * (threadIdx.x & (G - 1));
    const int hd = a.kv.hd, half = hd >> 1;
    const int token = blockIdx.x, head = blockIdx.y * (kAppendThreads / G) + threadIdx.x / G;
    const bool is_q = head < a.nq, is_v = head >= a.nq + a.kv.nkv;
    const bool live = lane4 < half && head < a.nq + 2 * a.kv.nkv;
    pdl_launch_dependents();
    pdl_wait();
    float4 x = make_float4(0, 0, 0, 0), y = x;
    if (live) {
        const float* src = a.qkv + token * a.ld + (head * hd + lane4);
        x = __ldcs(reinterpret_cast<const float4*>(src));
        y = __ldcs(reinterpret_cast<const float4*>(src + half));
    }
    const int pos = a.positions[token];
    const bool placed = pos >= 0 && pos < a.ctx;  // a rotation exists for the position
    if (a.q_norm) {                                // every lane of the warp takes part in the shuffles
        float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + (y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w);
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (live && !is_v) {
            const float* w = (is_q ? a.q_norm : a.k_norm) + lane4;
            const float inv = rsqrtf(ss * (1.0f / (float)hd) + a.eps);  // to 2 ulp
            const float4 w0 = *reinterpret_cast<const float4*>(w);
            const float4 w1 = *reinterpret_cast<const float4*>(w + half);
            x = make_float4(x.x * inv * (w0.x + a.offset), x.y * inv * (w0.y + a.offset),
                            x.z * inv * (w0.z + a.offset), x.w * inv * (w0.w + a.offset));
            y = make_float4(y.x * inv * (w1.x + a.offset), y.y * inv * (w1.y + a.offset),
                            y.z * inv * (w1.z + a.offset), y.w * inv * (w1.w + a.offset));
        }
    }
    if (!live) return;
    if (!is_v && placed) {
        const float* ct = a.cos_t + (int64_t)pos * half;
        const float* st = a.sin_t + (int64_t)pos * half;
        const float4 u = x, z = y;
        if constexpr (kInterleaved) {  // pairs of the first half, then of the second
            const int l = lane4 >> 1;
            const float2 c0 = *reinterpret_cast<const float2*>(ct + l), s0 = *reinterpret_cast<const float2*>(st + l);
            x = make_float4(u.x * c0.x - u.y * s0.x, u.x * s0.x + u.y * c0.x, u.z * c0.y - u.w * s0.y,
                            u.z * s0.y + u.w * c0.y);
            const float2 c1 = *reinterpret_cast<const float2*>(ct + (half >> 1) + l);
            const float2 s1 = *reinterpret_cast<const float2*>(st + (half >> 1) + l);
            y = make_float4(z.x * c1.x - z.y * s1.x, z.x * s1.x + z.y * c1.x, z.z * c1.y - z.w * s1.y,
                            z.z * s1.y + z.w * c1.y);
        } else {
            const float4 c = *reinterpret_cast<const float4*>(ct + lane4);
            const float4 s = *reinterpret_cast<const float4*>(st + lane4);
            x = make_float4(u.x * c.x - z.x * s.x, u.y * c.y - z.y * s.y, u.z * c.z - z.z * s.z,
                            u.w * c.w - z.w * s.w);
            y = make_float4(u.x * s.x + z.x * c.x, u.y * s.y + z.y * c.y, u.z * s.z + z.z * c.z,
                            u.w * s.w + z.w * c.w);
        }
    }
    if (is_q) {
        if (!placed) x = y = make_float4(0, 0, 0, 0);
        float* dst = a.q_out + ((int64_t)token * a.nq + head) * hd + lane4;
        store4(dst, x);
        store4(dst + half, y);
        return;
    }
    const int slot = a.slots[token], seq = a.seqs ? a.seqs[token] : token;
    if (!placed || seq < 0 || seq >= a.kv.n_seqs || slot < 0 || slot >= a.kv.capacity()) return;
    const int64_t row = a.kv.row(seq, head - a.nq - (is_v ? a.kv.nkv : 0), slot);
    if (row < 0) return;
    T* dst = static_cast<T*>(is_v ? a.kv.v : a.kv.k) + row + lane4;
    store4(dst, x);
    store4(dst + half, y);
}

template <typename T>
cudaError_t launch_append(const AppendArgs& a, bool interleaved, cudaStream_t st) {
    const int lanes = a.kv.hd / 8;
    const int G = lanes <= 8 ? 8 : (lanes <= 16 ? 16 : 32), groups = kAppendThreads / G;
    const dim3 grid(a.tokens, (a.nq + 2 * a.kv.nkv + groups - 1) / groups);
    AppendArgs aa = a;
    int g = G;
    void* args[] = {&aa, &g};
    return launch_pdl_kernel(interleaved ? (const void*)paged_append_kernel<T, true>
                                         : (const void*)paged_append_kernel<T, false>,
                             grid, dim3(kAppendThreads), 0, st, args);
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
