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
constexpr int kLogitCtas = 4;  // per SM: all its threads
constexpr int kMaxSlice = 32 * kLogitThreads;  // a bit of a register for each of a thread's entries
constexpr int kMinSlice = 4 * kLogitThreads;

// What is known of a vocabulary entry: in the history, biased, times in the
// output. 16 bits of shared memory where no history is longer than their count.
template <bool kShort>
struct Word {
    static constexpr uint32_t kBiased = kShort ? 0x4000u : 0x40000000u, kSeen = 2 * kBiased, kCount = kBiased - 1;
    __device__ static __forceinline__ uint32_t get(const uint32_t* words, int u) {
        return kShort ? reinterpret_cast<const uint16_t*>(words)[u] : words[u];
    }
    __device__ static __forceinline__ void add(uint32_t* words, int u) {
        if (kShort) atomicAdd(&words[u >> 1], 1u << (16 * (u & 1)));
        else atomicAdd(&words[u], 1u);
    }
    __device__ static __forceinline__ uint32_t set(uint32_t* words, int u, uint32_t bit) {  // the word before
        if (kShort) return atomicOr(&words[u >> 1], bit << (16 * (u & 1))) >> (16 * (u & 1)) & 0xffffu;
        return atomicOr(&words[u], bit);
    }
    // bit e: entry 4 q + e is known of
    __device__ static __forceinline__ uint32_t four(const uint32_t* words, int q) {
        if (kShort) {
            const uint2 c = reinterpret_cast<const uint2*>(words)[q];
            if (!(c.x | c.y)) return 0;
            return (c.x & 0xffffu ? 1u : 0u) | (c.x >> 16 ? 2u : 0u) | (c.y & 0xffffu ? 4u : 0u) | (c.y >> 16 ? 8u : 0u);
        }
        const uint4 c = reinterpret_cast<const uint4*>(words)[q];
        if (!(c.x | c.y | c.z | c.w)) return 0;
        return (c.x ? 1u : 0u) | (c.y ? 2u : 0u) | (c.z ? 4u : 0u) | (c.w ? 8u : 0u);
    }
};

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

// A CTA owns a slice of one row. It streams the slice through the mask, notes the
// history's tokens and the biases that fall into it in shared memory (integer
// atomics: the order does not matter), and then rewrites the few entries so
// touched from their logits, which are still there: in x, or, in place, where the
// mask let them through, and the others stay -infinity. Slices start on 16-byte
// boundaries of the row; kVec: the rows of logits and out are alike in that (else
// single words).
// Every CTA of a row reads the row's whole history, so slices are long; an
// untouched entry gets no more than a load, a mask bit and a store; and a CTA's
// chain of loads, counts and loads is long, so four share an SM. 64 rows of 262144,
// 4096 tokens of history, 300 biases: with the logits in 32 registers of unrolled
// code, which did not fit the instruction cache, 94 us; staged in shared memory 50
// us; every entry's word looked at on the way 57 us; touched entries apart, counted
// before the stream in 32-bit words, three CTAs per SM, 39 us; this 33 us. As two
// launches side by side (all logits through the mask; the touched ones from a hash
// table) it took 43 us, the two in each other's way on registers.
template <bool kVec, bool kShort>
__global__ void __launch_bounds__(kLogitThreads, kLogitCtas) process_logits_kernel(const LogitsArgs a, int slice) {
    using W = Word<kShort>;
    extern __shared__ __align__(16) uint32_t word[];  // slice words, then the slice's words of the mask
    __shared__ uint16_t bias_id[kMaxBias];             // those in the slice, in any order
    __shared__ uint16_t bias_at[kMaxBias];             // their places in the row's list
    __shared__ float bias_value[kMaxBias];
    __shared__ int n_bias_s;
    __shared__ bool twice_s;  // an entry has several biases
    const int words = kShort ? slice / 2 : slice;
    uint32_t* mask_s = word + words;
    // the first slices of all rows, then the second ones: frequent tokens have low ids, and the longest go first
    const unsigned nth = blockIdx.x / (unsigned)a.rows;
    const int row = (int)(blockIdx.x - nth * (unsigned)a.rows);
    const float* x = a.logits + row * a.ld;
    float* y = a.out + row * a.ld_out;
    const int shift = kVec ? (int)(((uintptr_t)x >> 2) & 3) : 0;  // entries before the row's first boundary
    const int v0 = (int)nth * slice - shift;                // entry 0 of the slice (may be before the row)
    const int lo = v0 < 0 ? -v0 : 0, hi = min(slice, a.vocab - v0);
    pdl_launch_dependents();
    pdl_wait();
    if (hi <= lo) return;
    x += v0;
    y += v0;
    int mrow = a.mask ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
    if (mrow >= a.n_masks) mrow = -1;
    const int total = a.tokens ? min(max(a.token_lengths[row], 0), a.max_tokens) : 0;
    const int word0 = (v0 + lo) >> 5;  // mask_s[0] is this word of the mask
    if (mrow >= 0) {
        const int all = (a.vocab + 31) / 32;
        for (int i = threadIdx.x; i < slice / 32 + 2; i += kLogitThreads)
            mask_s[i] = word0 + i < all ? (uint32_t)a.mask[(int64_t)mrow * all + word0 + i] : 0u;
    }
    for (int i = threadIdx.x; i < words / 4; i += kLogitThreads)
        reinterpret_cast<uint4*>(word)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) n_bias_s = 0, twice_s = false;
    __syncthreads();

    // the stream
    const int i0 = 4 * threadIdx.x, rounds = slice / (4 * kLogitThreads), bit = v0 + i0 - 32 * word0;
    auto masked = [&](float4 v, uint32_t m) {
        if (!(m & 1)) v.x = -INFINITY;
        if (!(m & 2)) v.y = -INFINITY;
        if (!(m & 4)) v.z = -INFINITY;
        if (!(m & 8)) v.w = -INFINITY;
        return v;
    };
    if (kVec && lo == 0 && hi == slice) {  // no edge: nothing but loads, mask bits and stores
        const float4* from = reinterpret_cast<const float4*>(x + i0);
        float4* to = reinterpret_cast<float4*>(y + i0);
        if (mrow < 0) {
#pragma unroll 4
            for (int j = 0; j < rounds; ++j) to[j * kLogitThreads] = from[j * kLogitThreads];
        } else {
            const uint32_t* m = mask_s + (bit >> 5);
#pragma unroll 4
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
    if (total == 0 && a.n_bias == 0) return;

    // the counts
    for (int i = threadIdx.x; i < a.n_bias; i += kLogitThreads) {
        const int id = a.bias_ids[(int64_t)row * a.n_bias + i], u = id - v0;
        if (id >= 0 && u >= lo && u < hi) {
            const int k = atomicAdd(&n_bias_s, 1);
            bias_id[k] = (uint16_t)u;
            bias_at[k] = (uint16_t)i;
            bias_value[k] = a.bias_values[(int64_t)row * a.n_bias + i];
            if (W::set(word, u, W::kBiased) & W::kBiased) twice_s = true;
        }
    }
    const int prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    auto note = [&](int token, int i) {
        const int u = token - v0;
        if (u < lo || u >= hi) return;
        if (i >= prompt) W::add(word, u);
        else if (!(W::get(word, u) & W::kSeen)) W::set(word, u, W::kSeen);  // frequent ones would wait for one another
    };
    // the history: ids before the first 16-byte boundary, fours, the rest; two rounds' loads in flight
    const int* tok = a.tokens + row * a.ld_tokens;
    const int head = min(total, (int)((4 - ((uintptr_t)tok >> 2)) & 3)), fours = (total - head) / 4;
    for (int q0 = threadIdx.x; q0 < fours; q0 += 2 * kLogitThreads) {
        const int4* from = reinterpret_cast<const int4*>(tok + head) + q0;
        const bool more = q0 + kLogitThreads < fours;
        const int4 t0 = from[0];
        int4 t1 = t0;
        if (more) t1 = from[kLogitThreads];
        const int i = head + 4 * q0;
        note(t0.x, i);
        note(t0.y, i + 1);
        note(t0.z, i + 2);
        note(t0.w, i + 3);
        if (more) {
            note(t1.x, i + 4 * kLogitThreads);
            note(t1.y, i + 4 * kLogitThreads + 1);
            note(t1.z, i + 4 * kLogitThreads + 2);
            note(t1.w, i + 4 * kLogitThreads + 3);
        }
    }
    if ((int)threadIdx.x < head) note(tok[threadIdx.x], threadIdx.x);
    const int tail = head + 4 * fours + (int)threadIdx.x;
    if (tail < total) note(tok[tail], tail);
    __syncthreads();

    // the touched entries
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float pres = a.presence ? a.presence[row] : 0.0f;
    const float freq = a.frequency ? a.frequency[row] : 0.0f;
    auto allowed = [&](int i) {
        const int at = v0 + i - 32 * word0;
        return mrow < 0 || ((mask_s[at >> 5] >> (at & 31)) & 1);
    };
    auto penalised = [&](uint32_t c, float f) {
        if (c & (W::kSeen | W::kCount)) {
            f = f > 0.0f ? f / rep : f * rep;
            const uint32_t n = c & W::kCount;
            if (n) f = f - freq * (float)n - pres;
        }
        return f;
    };
    // biased ones by the thread of their first bias
    const int n_bias = n_bias_s;
    for (int k = threadIdx.x; k < n_bias; k += kLogitThreads) {
        const int u = bias_id[k], at = bias_at[k];
        bool first = true;
        int others = 0;
        for (int m = 0; twice_s && m < n_bias; ++m)
            if (bias_id[m] == u && m != k) ++others, first = first && bias_at[m] > at;
        if (!first || !allowed(u)) continue;
        float f = penalised(W::get(word, u), x[u]) + bias_value[k];
        // the others in the list's order: one by one from the slice's, or, many of them (a list padded with one
        // id, say), by a scan of the whole list (1024 biases, 1000 of them on one token: 62.7 ms one by one)
        if (others * n_bias <= a.n_bias) {
            for (int last = at; others > 0; --others) {
                int next = kMaxBias, from = 0;
                for (int m = 0; m < n_bias; ++m)
                    if (bias_id[m] == u && bias_at[m] > last && bias_at[m] < next) next = bias_at[m], from = m;
                f += bias_value[from];
                last = next;
            }
        } else {
            const int* ids = a.bias_ids + (int64_t)row * a.n_bias;
            const float* values = a.bias_values + (int64_t)row * a.n_bias;
#pragma unroll 4
            for (int m = at + 1; m < a.n_bias; ++m)
                if (ids[m] == v0 + u) f += values[m];
        }
        y[u] = f;
    }
    if (total == 0) return;
    // the others by threads in turn; bit 4 j + e: entry e of this thread's four in round j
    uint32_t mine = 0;
#pragma unroll 4
    for (int j = 0; j < rounds; ++j) mine |= W::four(word, threadIdx.x + kLogitThreads * j) << (4 * j);
    while (mine) {  // two logits on their way at once
        float f[2];
        int at[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            at[j] = -1;
            if (!mine) continue;
            const int b = __ffs(mine) - 1, i = i0 + 4 * kLogitThreads * (b >> 2) + (b & 3);
            mine &= mine - 1;
            if ((W::get(word, i) & W::kBiased) || !allowed(i)) continue;
            at[j] = i;
            f[j] = x[i];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (at[j] >= 0) y[at[j]] = penalised(W::get(word, at[j]), f[j]);
    }
}

template <bool kVec, bool kShort>
cudaError_t launch(LogitsArgs a, int slice, cudaStream_t st) {
    const void* fn = (const void*)process_logits_kernel<kVec, kShort>;
    const size_t smem = ((size_t)(kShort ? slice / 2 : slice) + slice / 32 + 2) * sizeof(uint32_t);
    const cudaError_t e = ensure_dynamic_smem(fn, smem);
    if (e != cudaSuccess) return e;
    const int64_t grid = ((int64_t)a.vocab + 3 + slice - 1) / slice * a.rows;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    void* args[] = {&a, &slice};
    return launch_pdl_kernel(fn, dim3((unsigned)grid), dim3(kLogitThreads), smem, st, args);
}

}  // namespace

cudaError_t launch_process_logits(const LogitsArgs& a, cudaStream_t st) {
    if (a.rows <= 0 || a.vocab <= 0) return cudaSuccess;
    // 16-byte accesses where the rows of logits and out begin alike
    const bool vec = (((uintptr_t)a.logits ^ (uintptr_t)a.out) & 15) == 0 && (a.rows == 1 || (a.ld - a.ld_out) % 4 == 0);
    // the longest slices that leave two CTAs for every SM
    int slice = kMaxSlice;
    const int sms = paged_sm_count();
    while (slice > kMinSlice && (int64_t)a.rows * (a.vocab / slice) < 2 * sms) slice /= 2;
    if (a.max_tokens < (int)Word<true>::kBiased)
        return vec ? launch<true, true>(a, slice, st) : launch<false, true>(a, slice, st);
    return vec ? launch<true, false>(a, slice, st) : launch<false, false>(a, slice, st);
}

}  // namespace qmm
