// Logits of the next token before sampling (sm_100a): penalties for repeated
// tokens, biases and a grammar mask in one pass over the vocabulary. Per row,
// with seen = the token is in the history, count = how often it is in the
// history after the prompt:
//
//   x' = seen ? (x > 0 ? x / r : x r) : x           (repetition r)
//   x' = x' - f count - p [count > 0]               (frequency f, presence p)
//   x' = x' + sum of the token's biases, in list order
//   x' = mask bit set ? x' : -infinity
//
// Bound by HBM for batches (every logit is read and written once), by the
// latency of a CTA's chain -- history, counts, logits -- for single rows.
#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"

namespace qmm {

namespace {

constexpr int kLogitThreads = 512;
constexpr int kMaxSlice = 32 * kLogitThreads;  // a bit of a register for each of a thread's entries
constexpr int kMinSlice = 4 * kLogitThreads;
// A vocabulary entry's word: in the history, biased, times in the output.
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3fffffffu;

template <bool kVec>
__device__ __forceinline__ float4 load4(const float* p, int i, int lo, int hi) {
    float4 v = make_float4(0, 0, 0, 0);
    if (kVec && i >= lo && i + 3 < hi) return *reinterpret_cast<const float4*>(p + i);
    if (i >= lo && i < hi) v.x = p[i];
    if (i + 1 >= lo && i + 1 < hi) v.y = p[i + 1];
    if (i + 2 >= lo && i + 2 < hi) v.z = p[i + 2];
    if (i + 3 >= lo && i + 3 < hi) v.w = p[i + 3];
    return v;
}
template <bool kVec>
__device__ __forceinline__ void store4(float* p, int i, int lo, int hi, const float4& v) {
    if (kVec && i >= lo && i + 3 < hi) {
        *reinterpret_cast<float4*>(p + i) = v;
        return;
    }
    if (i >= lo && i < hi) p[i] = v.x;
    if (i + 1 >= lo && i + 1 < hi) p[i + 1] = v.y;
    if (i + 2 >= lo && i + 2 < hi) p[i + 2] = v.z;
    if (i + 3 >= lo && i + 3 < hi) p[i + 3] = v.w;
}

// A CTA owns a slice of one row. It has the slice's logits fetched into L2, notes
// the history's tokens and the biases that fall into the slice in shared memory
// (integer atomics: the order does not matter), works out the few touched
// entries, streams the slice through the mask, and puts the touched entries in
// their places (a thread's own, so nothing waits). Slices start on 16-byte
// boundaries of the row; kVec: the rows of logits and out are alike in that (else
// single words).
// Every CTA of a row reads the row's whole history, so slices are long, and an
// untouched entry gets no more than a load, a mask bit and a store. 64 rows of
// 262144, 4096 tokens of history, 300 biases: with the logits in 32 registers of
// unrolled code, which did not fit the instruction cache, 94 us; staged in shared
// memory 50 us; every entry's word looked at on the way 57 us; this 39 us. As two
// launches side by side (all logits through the mask; the touched ones from a hash
// table) it took 43 us, the two in each other's way on registers.
template <bool kVec>
__global__ void __launch_bounds__(kLogitThreads, 3) process_logits_kernel(const LogitsArgs a, int slice) {
    extern __shared__ __align__(16) uint32_t word[];  // [slice], then the slice's words of the mask
    __shared__ uint16_t bias_id[kMaxBias];             // those in the slice, in any order
    __shared__ uint16_t bias_at[kMaxBias];             // their places in the row's list
    __shared__ float bias_value[kMaxBias];             // a first bias: then the entry's logit
    __shared__ int n_bias_s;
    __shared__ bool twice_s;  // an entry has several biases
    uint32_t* mask_s = word + slice;
    const int row = blockIdx.y;
    const float* x = a.logits + row * a.ld;
    float* y = a.out + row * a.ld_out;
    const int shift = kVec ? (int)(((uintptr_t)x >> 2) & 3) : 0;  // entries before the row's first boundary
    const int v0 = (int)blockIdx.x * slice - shift;                // entry 0 of the slice (may be before the row)
    const int lo = v0 < 0 ? -v0 : 0, hi = min(slice, a.vocab - v0);
    pdl_launch_dependents();
    pdl_wait();
    if (hi <= lo) return;
    x += v0;
    y += v0;

    for (int i = lo + 32 * threadIdx.x; i < hi; i += 32 * kLogitThreads)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(x + i));
    // the history: ids before the first 16-byte boundary, fours, the rest; four rounds' loads in flight
    constexpr int kRounds = 4;
    const int total = a.tokens ? min(max(a.token_lengths[row], 0), a.max_tokens) : 0;
    const int prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    const int* tok = a.tokens + row * a.ld_tokens;
    const int head = min(total, (int)((4 - ((uintptr_t)tok >> 2)) & 3)), fours = (total - head) / 4;
    int4 t[kRounds];
    auto fetch = [&](int q0) {
#pragma unroll
        for (int j = 0; j < kRounds; ++j) {
            const int q = q0 + j * kLogitThreads;
            if (q < fours) t[j] = reinterpret_cast<const int4*>(tok + head)[q];
        }
    };
    fetch(threadIdx.x);
    const int* ids = a.bias_ids + (int64_t)row * a.n_bias;
    int id = (int)threadIdx.x < a.n_bias ? ids[threadIdx.x] : 0;
    int mrow = a.mask ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
    if (mrow >= a.n_masks) mrow = -1;
    const int word0 = (v0 + lo) >> 5, words = (a.vocab + 31) / 32;  // mask_s[0] is word word0 of the mask
    if (mrow >= 0)
        for (int i = threadIdx.x; i < slice / 32 + 2; i += kLogitThreads)
            mask_s[i] = word0 + i < words ? (uint32_t)a.mask[(int64_t)mrow * words + word0 + i] : 0u;
    for (int i = threadIdx.x; i < slice / 4; i += kLogitThreads)
        reinterpret_cast<uint4*>(word)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) n_bias_s = 0, twice_s = false;
    __syncthreads();

    for (int i = threadIdx.x; i < a.n_bias;) {
        const int u = id - v0;
        if (id >= 0 && u >= lo && u < hi) {
            const int k = atomicAdd(&n_bias_s, 1);
            bias_id[k] = (uint16_t)u;
            bias_at[k] = (uint16_t)i;
            bias_value[k] = a.bias_values[(int64_t)row * a.n_bias + i];
            if (atomicOr(&word[u], kBiased) & kBiased) twice_s = true;
        }
        i += kLogitThreads;
        if (i < a.n_bias) id = ids[i];
    }
    auto note = [&](int token, int i) {
        const int u = token - v0;
        if (u < lo || u >= hi) return;
        if (i >= prompt) atomicAdd(&word[u], 1u);
        else if (!(word[u] & kSeen)) atomicOr(&word[u], kSeen);  // frequent tokens would wait for one another
    };
    for (int q0 = threadIdx.x; q0 < fours;) {
#pragma unroll
        for (int j = 0; j < kRounds; ++j) {
            const int q = q0 + j * kLogitThreads, i = head + 4 * q;
            if (q < fours) {
                note(t[j].x, i);
                note(t[j].y, i + 1);
                note(t[j].z, i + 2);
                note(t[j].w, i + 3);
            }
        }
        q0 += kRounds * kLogitThreads;
        if (q0 < fours) fetch(q0);
    }
    if ((int)threadIdx.x < head) note(tok[threadIdx.x], threadIdx.x);
    const int tail = head + 4 * fours + (int)threadIdx.x;
    if (tail < total) note(tok[tail], tail);
    __syncthreads();

    const int i0 = 4 * threadIdx.x;
    // bit 4 j + e: entry e of this thread's four in round j is touched
    auto entry = [&](uint32_t bits) {
        const int b = __ffs(bits) - 1;
        return i0 + 4 * kLogitThreads * (b >> 2) + (b & 3);
    };
    uint32_t mine = 0;
    if (total > 0 || a.n_bias > 0) {
        const float rep = a.repetition ? a.repetition[row] : 1.0f;
        const float pres = a.presence ? a.presence[row] : 0.0f;
        const float freq = a.frequency ? a.frequency[row] : 0.0f;
        auto penalised = [&](uint32_t c, float f) {
            if (c & (kSeen | kCount)) {
                f = f > 0.0f ? f / rep : f * rep;
                const uint32_t n = c & kCount;
                if (n) f = f - freq * (float)n - pres;
            }
            return f;
        };
        // Biased entries by the thread of their first bias; the word then says where the logit is.
        const int n_bias = n_bias_s;
        if (n_bias) {
            for (int k = threadIdx.x; k < n_bias; k += kLogitThreads) {
                const int u = bias_id[k], at = bias_at[k];
                bool first = true, alone = true;
                for (int m = 0; twice_s && m < n_bias; ++m)
                    if (bias_id[m] == u && m != k) alone = false, first = first && bias_at[m] > at;
                if (!first) continue;
                float f = penalised(word[u], x[u]) + bias_value[k];
                for (int last = at; !alone;) {  // the others one by one, in the list's order
                    int next = kMaxBias, from = 0;
                    for (int m = 0; m < n_bias; ++m)
                        if (bias_id[m] == u && bias_at[m] > last && bias_at[m] < next) next = bias_at[m], from = m;
                    if (next == kMaxBias) break;
                    f += bias_value[from];
                    last = next;
                }
                bias_value[k] = f;  // nobody else reads a first bias's value
                word[u] = kBiased | (uint32_t)k;
            }
            __syncthreads();
        }
#pragma unroll 4
        for (int j = 0; j < slice / (4 * kLogitThreads); ++j) {
            const uint4 c = reinterpret_cast<const uint4*>(word)[threadIdx.x + kLogitThreads * j];
            if (c.x | c.y | c.z | c.w)
                mine |= ((c.x ? 1u : 0u) | (c.y ? 2u : 0u) | (c.z ? 4u : 0u) | (c.w ? 8u : 0u)) << (4 * j);
        }
        for (uint32_t left = mine; left;) {  // four logits on their way at once
            float f[4];
            uint32_t l = left;
#pragma unroll
            for (int j = 0; j < 4; ++j, l &= l - 1)
                if (l) f[j] = x[entry(l)];
#pragma unroll
            for (int j = 0; j < 4; ++j, left &= left - 1)
                if (left) {
                    const int i = entry(left);
                    const uint32_t c = word[i];
                    word[i] = __float_as_uint(c & kBiased ? bias_value[c & kCount] : penalised(c, f[j]));
                }
        }
    }
    auto masked = [&](float4 v, uint32_t m) {
        if (!(m & 1)) v.x = -INFINITY;
        if (!(m & 2)) v.y = -INFINITY;
        if (!(m & 4)) v.z = -INFINITY;
        if (!(m & 8)) v.w = -INFINITY;
        return v;
    };
    const int rounds = slice / (4 * kLogitThreads), bit = v0 + i0 - 32 * word0;
    if (kVec && lo == 0 && hi == slice) {  // no edge: nothing but loads, mask bits and stores
        const float4* from = reinterpret_cast<const float4*>(x + i0);
        float4* to = reinterpret_cast<float4*>(y + i0);
        if (mrow < 0) {
#pragma unroll 8
            for (int j = 0; j < rounds; ++j) to[j * kLogitThreads] = from[j * kLogitThreads];
        } else {
            const uint32_t* m = mask_s + (bit >> 5);
#pragma unroll 8
            for (int j = 0; j < rounds; ++j, m += kLogitThreads / 8)
                to[j * kLogitThreads] = masked(from[j * kLogitThreads], __funnelshift_r(m[0], m[1], bit & 31));
        }
    } else {
#pragma unroll 2
        for (int i = i0; i < hi; i += 4 * kLogitThreads) {
            float4 v = load4<kVec>(x, i, lo, hi);
            if (mrow >= 0) {  // four bits, from the word of the first entry on; entries before the row have none
                const int at = bit + i - i0;
                v = masked(v, at >= 0 ? __funnelshift_r(mask_s[at >> 5], mask_s[(at >> 5) + 1], at & 31)
                                      : mask_s[0] << -at);
            }
            store4<kVec>(y, i, lo, hi, v);
        }
    }
    for (; mine; mine &= mine - 1) {
        const int i = entry(mine), at = v0 + i - 32 * word0;
        if (mrow < 0 || ((mask_s[at >> 5] >> (at & 31)) & 1)) y[i] = __uint_as_float(word[i]);
    }
}

}  // namespace

cudaError_t launch_process_logits(const LogitsArgs& a, cudaStream_t st) {
    if (a.rows <= 0 || a.vocab <= 0) return cudaSuccess;
    // 16-byte accesses where the rows of logits and out begin alike
    const bool vec = (((uintptr_t)a.logits ^ (uintptr_t)a.out) & 15) == 0 && (a.rows == 1 || (a.ld - a.ld_out) % 4 == 0);
    // the longest slices that leave two CTAs for every SM
    int slice = kMaxSlice;
    while (slice > kMinSlice && (int64_t)a.rows * (a.vocab / slice) < 2 * 148) slice /= 2;
    const void* fn = vec ? (const void*)process_logits_kernel<true> : (const void*)process_logits_kernel<false>;
    const size_t smem = (size_t)(slice + slice / 32 + 2) * sizeof(uint32_t);
    const cudaError_t e = ensure_dynamic_smem(fn, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(((int64_t)a.vocab + 3 + slice - 1) / slice), a.rows);
    LogitsArgs aa = a;
    void* args[] = {&aa, &slice};
    return launch_pdl_kernel(fn, grid, dim3(kLogitThreads), smem, st, args);
}

}  // namespace qmm
