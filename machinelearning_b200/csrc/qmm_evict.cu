// Eviction from a paged key/value cache by accumulated attention weight
// (sm_100a). Per (sequence, kv head) with more than `budget` cached slots the
// kept slots are, in this order of preference: those of the last `recent`
// positions, then those with the most accumulated weight (equal weights: the
// lowest slot first; NaN ranks with -infinity). Kept slots at or above
// `budget` move into the evicted slots below it, the r-th of the former into
// the r-th of the latter: attention does not depend on the order of the
// slots (each keeps its own position), a move reads slots that no move
// writes, and no more rows are moved than have to be.
#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"

namespace qmm {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

// Unsigned order of the preference: a total order on the floats, protected
// slots above all of them. w + 0 turns -0 into +0, its equal.
__device__ __forceinline__ uint32_t slot_key(float w, bool is_recent) {
    if (is_recent) return 0xffffffffu;
    if (w != w) w = -INFINITY;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix of v over the CTA's threads; *total is the CTA's sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();  // warp_sums is reused between calls
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    int base = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
        const int c = warp_sums[w];
        if (w < warp) base += c;
        all += c;
    }
    *total = all;
    return base + s - v;
}

// One CTA per (kv head, sequence): the threshold key by four rounds of 8-bit
// counting, then the lists of holes and movers in slot order, then the moves.
__global__ void __launch_bounds__(kThreads) evict_kernel(const EvictArgs a, int size, int* lists) {
    __shared__ int hist[256];
    __shared__ int warp_sums[kWarps];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int h = blockIdx.x, b = blockIdx.y;
    const int64_t cap = a.kv.capacity();
    const int64_t base = ((int64_t)b * a.kv.nkv + h) * cap;
    int n = a.lengths[b];
    n = n < 0 ? 0 : (n > cap ? (int)cap : n);
    const int kept = n < a.budget ? n : a.budget;
    if (h == 0 && threadIdx.x == 0) a.lengths_out[b] = kept;
    const float* w = a.weights + base;
    const int* pos = a.positions + base;
    float* w_out = a.weights_out + base;
    int* pos_out = a.positions_out + base;
    for (int64_t t = threadIdx.x; t < cap; t += kThreads) {
        w_out[t] = t < kept ? w[t] : 0.0f;
        pos_out[t] = t < kept ? pos[t] : -1;
    }
    if (n <= a.budget) return;
    const int64_t limit = (int64_t)a.next_positions[b] - a.recent;
    uint32_t prefix = 0;
    int need = a.budget;  // slots still to take among those that match the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        __syncthreads();
        for (int t = threadIdx.x; t < n; t += kThreads) {
            const uint32_t key = slot_key(w[t], pos[t] >= limit);
            if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
                atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int left = need, d = 255;
            while (hist[d] < left) left -= hist[d--];
            s_prefix = prefix | ((uint32_t)d << shift);
            s_need = left;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
    }
    int* holes = lists + ((int64_t)b * a.kv.nkv + h) * 2 * a.budget;
    int* movers = holes + a.budget;
    int n_ties = 0, n_holes = 0, n_movers = 0;
    for (int t0 = 0; t0 < n; t0 += kThreads) {
        const int t = t0 + threadIdx.x;
        const uint32_t key = t < n ? slot_key(w[t], pos[t] >= limit) : 0;
        const bool tie = t < n && key == prefix;
        int total;
        const int rank = n_ties + block_scan(tie, warp_sums, &total);
        n_ties += total;
        const bool keep = t < n && (key > prefix || (tie && rank < need));
        const bool hole = t < a.budget && !keep, mover = keep && t >= a.budget;
        const int r = block_scan((hole ? 1 : 0) | (mover ? 1 << 16 : 0), warp_sums, &total);
        if (hole) holes[n_holes + (r & 0xffff)] = t;
        if (mover) movers[n_movers + (r >> 16)] = t;
        n_holes += total & 0xffff;
        n_movers += total >> 16;
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int units = a.kv.hd * size / 16;  // 16-byte units of a row
    for (int i = warp; i < n_movers; i += kWarps) {
        const int to = holes[i], of = movers[i];
        if (lane == 0) {
            w_out[to] = w[of];
            pos_out[to] = pos[of];
        }
        const int64_t dst = a.kv.row(b, h, to), src = a.kv.row(b, h, of);
        if (dst < 0 || src < 0) continue;
        for (int j = lane; j < units; j += 32) {
            const uint4 kx = reinterpret_cast<const uint4*>(static_cast<const char*>(a.kv.k) + src * size)[j];
            const uint4 vx = reinterpret_cast<const uint4*>(static_cast<const char*>(a.kv.v) + src * size)[j];
            reinterpret_cast<uint4*>(static_cast<char*>(a.kv.k) + dst * size)[j] = kx;
            reinterpret_cast<uint4*>(static_cast<char*>(a.kv.v) + dst * size)[j] = vx;
        }
    }
}

}  // namespace

size_t paged_evict_workspace(const PagedKv& kv, int budget) {
    const int64_t cap = kv.capacity();
    const size_t lists = (size_t)(budget < cap ? budget : cap);
    return (size_t)kv.n_seqs * kv.nkv * 2 * lists * sizeof(int);
}

cudaError_t launch_paged_evict(const EvictArgs& a0, void* ws, cudaStream_t st) {
    if (a0.kv.n_seqs <= 0) return cudaSuccess;
    EvictArgs a = a0;
    if (a.budget > a.kv.capacity()) a.budget = (int)a.kv.capacity();  // no sequence is longer
    evict_kernel<<<dim3(a.kv.nkv, a.kv.n_seqs), kThreads, 0, st>>>(a, kv_type_size(a.kv.dtype), static_cast<int*>(ws));
    note_launch();
    return cudaGetLastError();
}

}  // namespace qmm
