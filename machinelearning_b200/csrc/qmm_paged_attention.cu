// Attention of one new token per sequence over a paged key/value cache
// (sm_100a).
//
//   s_t = scale q . k_t,   out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m)
//
// over the slots t in [max(0, n - window), n) of a sequence of n cached
// slots; m is the largest score. A sequence without slots gives zeros.
// Optionally every slot's weight sum over the kv head's query heads of
// e^(s_t - m) / sum e^(s - m) is added to a running total.
#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"

namespace qmm {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxHd = 256;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ void slot_range(const AttendArgs& a, int b, int64_t* first, int64_t* n) {
    const int64_t cap = a.kv.capacity();
    int64_t len = a.lengths[b];
    len = len < 0 ? 0 : (len > cap ? cap : len);
    *n = len;
    *first = a.window > 0 && len > a.window ? len - a.window : 0;
}

// One CTA per (query head, sequence): each warp takes every eighth slot with a
// running maximum and sum, the warps are joined at the end.
template <typename T>
__global__ void __launch_bounds__(kThreads) attend_kernel(const AttendArgs a, float* scores, float2* stats) {
    __shared__ float acc_s[kWarps][kMaxHd];
    __shared__ float m_s[kWarps], l_s[kWarps];
    const int h = blockIdx.x, b = blockIdx.y;
    const int hd = a.kv.hd, per = hd / 32;
    const int kvh = h / (a.nq / a.kv.nkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int64_t first, n;
    slot_range(a, b, &first, &n);
    const float* q = a.q + b * a.ldq + (int64_t)h * hd;
    float qr[8], acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        qr[j] = j < per ? q[lane + 32 * j] : 0.0f;
        acc[j] = 0.0f;
    }
    // l is summed with its rounding error carried in c: tens of thousands of
    // small weights beside a large one would each round to nothing
    float m = -INFINITY, l = 0.0f, c = 0.0f;
    float* srow = scores ? scores + ((int64_t)b * a.nq + h) * a.kv.capacity() : nullptr;
    for (int64_t t = first + warp; t < n; t += kWarps) {
        const int64_t row = a.kv.row(b, kvh, t);
        if (row < 0) {
            if (srow && lane == 0) srow[t] = -INFINITY;
            continue;
        }
        const T* k = static_cast<const T*>(a.kv.k) + row;
        const T* v = static_cast<const T*>(a.kv.v) + row;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < per) s = fmaf(qr[j], kv_to_f32(k[lane + 32 * j]), s);
        s = warp_sum(s) * a.scale;
        if (srow && lane == 0) srow[t] = s;
        const float m2 = fmaxf(m, s);
        const float f = m2 == -INFINITY ? 1.0f : expf(m - m2);
        const float p = m2 == -INFINITY ? 0.0f : expf(s - m2);
        m = m2;
        l *= f;
        c = fmaf(c, f, p);
        const float l2 = l + c;
        c -= l2 - l;
        l = l2;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < per) acc[j] = acc[j] * f + p * kv_to_f32(v[lane + 32 * j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < per) acc_s[warp][lane + 32 * j] = acc[j];
    if (lane == 0) {
        m_s[warp] = m;
        l_s[warp] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, m_s[w]);
    float f[kWarps];
    for (int w = 0; w < kWarps; ++w) {
        f[w] = m_s[w] == -INFINITY ? 0.0f : expf(m_s[w] - M);
        L += l_s[w] * f[w];
    }
    for (int d = threadIdx.x; d < hd; d += kThreads) {
        float s = 0.0f;
        for (int w = 0; w < kWarps; ++w) s += acc_s[w][d] * f[w];
        a.out[((int64_t)b * a.nq + h) * hd + d] = L > 0.0f ? s / L : 0.0f;
    }
    if (stats && threadIdx.x == 0) stats[(int64_t)b * a.nq + h] = make_float2(M, L);
}

// weights_out[b][kv][t] = weights[b][kv][t] + sum over the kv head's query heads of the slot's weight.
__global__ void __launch_bounds__(kThreads) weights_kernel(const AttendArgs a, const float* scores,
                                                           const float2* stats) {
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int64_t cap = a.kv.capacity();
    const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (t >= cap) return;
    int64_t first, n;
    slot_range(a, b, &first, &n);
    const int64_t at = ((int64_t)b * a.kv.nkv + kvh) * cap + t;
    float w = a.weights[at];
    if (t >= first && t < n) {
        const int g = a.nq / a.kv.nkv;
        float p = 0.0f;
        for (int j = 0; j < g; ++j) {
            const int64_t h = (int64_t)b * a.nq + kvh * g + j;
            const float2 ml = stats[h];
            if (ml.y > 0.0f) p += expf(scores[h * cap + t] - ml.x) / ml.y;
        }
        w += p;
    }
    a.weights_out[at] = w;
}

}  // namespace

size_t paged_attention_workspace(const PagedKv& kv, int nq, bool weights) {
    if (!weights) return 0;
    return (size_t)kv.n_seqs * nq * (sizeof(float2) + (size_t)kv.capacity() * sizeof(float));
}

cudaError_t launch_paged_attention(const AttendArgs& a, void* ws, cudaStream_t st) {
    if (a.kv.n_seqs <= 0) return cudaSuccess;
    float2* stats = nullptr;
    float* scores = nullptr;
    if (a.weights) {
        stats = static_cast<float2*>(ws);
        scores = reinterpret_cast<float*>(stats + (size_t)a.kv.n_seqs * a.nq);
    }
    const dim3 grid(a.nq, a.kv.n_seqs);
    if (a.kv.dtype == kKvF32) attend_kernel<float><<<grid, kThreads, 0, st>>>(a, scores, stats);
    else if (a.kv.dtype == kKvF16) attend_kernel<__half><<<grid, kThreads, 0, st>>>(a, scores, stats);
    else attend_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a, scores, stats);
    note_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || !a.weights) return e;
    const dim3 wgrid((unsigned)((a.kv.capacity() + kThreads - 1) / kThreads), a.kv.nkv, a.kv.n_seqs);
    weights_kernel<<<wgrid, kThreads, 0, st>>>(a, scores, stats);
    note_launch();
    return cudaGetLastError();
}

}  // namespace qmm
