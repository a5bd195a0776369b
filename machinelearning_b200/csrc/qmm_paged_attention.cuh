// Attention of one new token per sequence over a paged key/value cache
// (sm_100a): the kernels, compiled per cache type by qmm_paged_attention_*.cu.
//
//   s_t = scale q . k_t,   out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m)
//
// over the slots t in [max(0, n - window), n) of a sequence of n cached
// slots; m is the largest score. A sequence without slots gives zeros, and so
// does one whose scores are all -infinity.
// Optionally every slot's weight sum over the kv head's query heads of
// e^(s_t - m) / sum e^(s - m) is added to a running total.
//
// What bounds it: every K and V element is read once and takes 2 g
// multiply-adds (g query heads per kv head), so HBM, as long as the products
// run on the tensor cores: at g = 8 in f32 on the CUDA cores they would take
// most of the machine.
//
// One pass with a running maximum and sum (attend_kernel), the work divided
// evenly over a fixed grid whatever the lengths are, then a join of the pieces
// of sequences that were divided (join_kernel).
#pragma once

#include <cuda_bf16.h>

#include "qmm_common.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"

namespace qmm {

// The workspace of a call. A piece is a CTA's part of a (sequence, head tile); one
// that is not the whole leaves (acc, m, l) behind: in the CTA's slot 0 if earlier
// CTAs hold the beginning, in slot 1 if not.
struct AttendScratch {
    float2* ml;      // [grid][2][kHeads]: reference and sum of a piece (see kSlack)
    float* acc;      // [grid][2][kHeads][hd]
    float2* whole;   // [n_seqs][nq], with weights: the same of undivided head tiles
    float* scores;   // [n_seqs][nq][capacity], with weights: scores in units of log 2
    int head_tiles;  // per kv head
    int grid;        // CTAs of attend_kernel
};

// launch_paged_attention's, per cache type; sms: of the current device.
cudaError_t attend_f32(const AttendArgs& a, const AttendScratch& sc, int sms, cudaStream_t st);
cudaError_t attend_f16(const AttendArgs& a, const AttendScratch& sc, int sms, cudaStream_t st);
cudaError_t attend_bf16(const AttendArgs& a, const AttendScratch& sc, int sms, cudaStream_t st);

// Query heads of a pass over K and V: one set of 8, or two.
inline int pass_heads(const PagedKv& kv, int nq) { return nq / kv.nkv > 8 ? 16 : 8; }
constexpr int kMaxAttendCtas = 2;  // per SM, of any shape

namespace {

using Scratch = AttendScratch;

constexpr float kLog2e = 1.4426950408889634f;

// ---- matrix instructions ----------------------------------------------------------
// D (16 x 8, f32) += A (16 x 16, row) B (16 x 8, col); for f32 caches
// D += A (16 x 8, tf32) B (8 x 8, tf32).
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 4)
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    else if constexpr (std::is_same_v<T, __half>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t tf32_rna(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}

// f32 values as sums of the instruction's operands: two f16 or tf32 (22 bits; a third
// part would take another instruction of four), three bf16 (24 bits; two leave 2^-17,
// and the outputs four times as far from the exact ones as f32 arithmetic does). The
// distance of the outputs from the exact ones, beside elementary f32 operations, over
// head_dims 64 to 256 and 40 to 6000 slots: f32 6.5e-7 (4.8e-7), f16 5.9e-7 (5.2e-7),
// bf16 5.4e-7 (4.9e-7).
template <typename T>
constexpr int kParts = std::is_same_v<T, __nv_bfloat16> ? 3 : 2;

template <typename T>
__device__ __forceinline__ void split(float x, T (&part)[kParts<T>]) {
#pragma unroll
    for (int i = 0; i < kParts<T>; ++i) {
        if constexpr (sizeof(T) == 4) part[i] = __uint_as_float(tf32_rna(x));
        else part[i] = f32_to_kv<T>(x);
        x -= kv_to_f32<T>(part[i]);
    }
}
// The same for two values at once, packed (16-bit types).
template <typename T>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&part)[kParts<T>]) {
#pragma unroll
    for (int i = 0; i < kParts<T>; ++i) {
        if constexpr (std::is_same_v<T, __half>) {
            const __half2 h = __floats2half2_rn(x, y);
            const float2 f = __half22float2(h);
            part[i] = *reinterpret_cast<const uint32_t*>(&h);
            x -= f.x, y -= f.y;
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
            const float2 f = __bfloat1622float2(h);
            part[i] = *reinterpret_cast<const uint32_t*>(&h);
            x -= f.x, y -= f.y;
        }
    }
}
__device__ __forceinline__ float ex2(float x) {  // 2^x to 2^-22; 0 below 2^-126
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 16 bytes to shared memory, zeros where !live (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ float quad_max(float v) {  // over the four lanes of a head
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// e^(m - M) of a piece's maximum m, 0 for a piece that saw no slot.
__device__ __forceinline__ float piece_factor(float m, float M) { return m == -INFINITY ? 0.0f : ex2(m - M); }

// ---- division of the work -----------------------------------------------------------
// The slots [first, n) of a sequence, in steps ("tiles") of kSlots aligned slots.
struct Slots {
    int first, n;
    int tile0, tiles;
};
// kWaited: the kernel has waited for the ones before; join_kernel reads lengths before
// its wait, and from L2.
template <int kSlots, bool kWaited = false>
__device__ __forceinline__ Slots slots_of(const AttendArgs& a, int b) {
    Slots s;
    const int64_t cap = a.kv.capacity();
    const int len = kWaited ? a.lengths[b] : __ldcg(a.lengths + b);
    s.n = len < 0 ? 0 : (len > cap ? (int)cap : len);
    s.first = a.window > 0 && s.n > a.window ? s.n - a.window : 0;
    s.tile0 = s.first / kSlots;
    s.tiles = (s.n + kSlots - 1) / kSlots - s.tile0;
    return s;
}

// The list of all (sequence, head tile)s -- each kSetup units for starting and
// ending it, then one unit per step -- is cut into equal shares, one per CTA.
// (Without the setup's units a CTA got dozens of short sequences where another
// had part of one: 64 sequences of 1 to 8192 slots, 64/8 heads of 128, f16 take
// 119 us instead of 40.)


// Units of a sequence.
template <typename S>
__device__ __forceinline__ int64_t units_of(const Slots& s, int heads) {
    return s.tiles ? (int64_t)(s.tiles + S::kSetup) * heads : 0;
}
// Units per CTA; a step per warp at least.
template <typename S>
__device__ __forceinline__ int64_t share_of(int64_t total, int grid) {
    const int64_t share = (total + grid - 1) / grid, least = S::kSetup + S::kWarps;
    return share < least ? least : share;
}
__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The CTAs that hold the pieces of a (sequence, head tile).
struct Pieces {
    int first, count;
    // Slot of piece p among the CTAs' slots.
    __device__ __forceinline__ int64_t slot(int p) const { return p == 0 ? 2 * first + 1 : 2 * (first + p); }
};
// base: the unit of the first step.
__device__ __forceinline__ Pieces pieces_of(int64_t base, int tiles, int64_t share) {
    const int64_t first = base / share, last = (base + tiles - 1) / share;
    return Pieces{(int)first, (int)(last - first) + 1};
}
struct Place {
    int64_t start, share;  // unit at which the sequence starts, units per CTA
    int tiles;
    template <typename S>
    __device__ __forceinline__ Pieces pieces(int h) const {
        return pieces_of(start + (int64_t)h * (tiles + S::kSetup) + S::kSetup, tiles, share);
    }
};
template <typename S>
__device__ __forceinline__ Place place_of(const AttendArgs& a, const Scratch& sc, int b) {
    const int heads = a.kv.nkv * sc.head_tiles;
    int64_t total = 0, before = 0;
#pragma unroll 4
    for (int i = threadIdx.x & 31; i < a.kv.n_seqs; i += 32) {
        const int64_t u = units_of<S>(slots_of<S::kSlots>(a, i), heads);
        total += u;
        if (i < b) before += u;
    }
    return Place{warp_sum64(before), share_of<S>(warp_sum64(total), sc.grid), slots_of<S::kSlots>(a, b).tiles};
}

// SETS sets of 8 query heads of a kv head share a pass over its K and V: two
// where there are more than 8 (8 x 49152 slots, 16 heads of 128 on one, bf16: a
// pass for each eight 70 us, one for both 53 us).
// kTile slots are the K of one instruction's P; a step takes kTiles of them. A
// warp's ring holds three units of a step's K or V rows: one in use, two on
// their way (16 warps per SM with 4 KB units: 128 KB in flight, above the 44 KB
// that 6.5 TB/s and 1 us need).
template <typename T, int HD, int SETS>
struct Shape {
    static constexpr int kHeads = 8 * SETS;
    static constexpr int kTile = sizeof(T) == 4 ? 8 : 16;
    static constexpr int kTiles = HD <= 64 || (HD <= 128 && SETS > 1) ? 2 : 1;
    static constexpr int kSlots = kTile * kTiles;
    static constexpr int kRow = HD * (int)sizeof(T);             // bytes
    static constexpr int kChunks = kRow / 64;                    // 16-byte units of a K row per lane
    static constexpr int kLines = kRow / 128;                    // of a row; 16-byte units of a V row per lane
    static constexpr int kVRows = kTile / 4;                     // V rows of a tile per lane
    static constexpr int kUnit = kSlots * HD * (int)sizeof(T);
    static constexpr int kUnits = 3;
    // Eight warps where their rings leave room for two CTAs on an SM and 128 registers hold the results, else
    // four (head_dim 192, one set: five 68 us, four 65 us for 16 x 16000 slots, 12/2 heads, bf16, 76 and 67 us
    // for 8 in f32; head_dim 64, two sets: eight spill, 83 us, four 74 us for 32 x 8000, 64/4 heads, bf16).
    static constexpr int kWarps = HD <= 128 && SETS == 1 ? 8 : 4;
    // A tile's P V summed apart and added in 32 bits, as the instruction cuts off what it adds to large sums.
    // Head_dim 64 with two sets has the most steps a warp, and single heads there were more than four times as
    // far from the exact outputs as elementary f32 operations (70 us without). Elsewhere it brings bf16 from 1.1
    // to 1.0 and f32 from 1.3 to 1.2 times, for up to 9% more time (64 ragged sequences, 64/8 heads of 128, f16).
    static constexpr bool kFresh = SETS == 2 && HD == 64;
    static constexpr int kQPairs = kChunks * 2 * 32 * 16;        // of a set: first two parts; a third takes half
    static constexpr int kQBytes = kQPairs + (kParts<T> - 2) * kQPairs / 2;
    // A piece's fixed cost, in steps: the time of 160 KB of K and V. With 80 KB for it 64 ragged sequences of
    // up to 8192 slots, 64/8 heads of 128, f16, take 50 us for 40.5 and one of 512 in f32 11.2 for 12.8; with
    // 240 KB 40 and 14.4.
    static constexpr int kSetup = 163840 / (2 * kUnit);
    static constexpr int kAccRow = HD + 4;                       // floats; spreads the rows over the banks
    static constexpr size_t kSmem =
        (size_t)kWarps * kUnits * kUnit + SETS * kQBytes + kWarps * kHeads * 8 + kHeads * 4;
    static constexpr int kCtas = 2 * (kSmem + 1024) <= 228 * 1024 ? 2 : 1;  // per SM
    static_assert(kHeads * kAccRow * 4 <= kUnits * kUnit, "a warp's result fits in its ring");
};

// The (sequence, head tile) that unit share * nth + shift of the list belongs to, by a
// warp; b < 0: none. Neighbouring lanes read neighbouring lengths, and join_kernel
// lets one warp do it: with a run of sequences per lane and every warp reading all of
// them from L2, 560 sequences of 300 slots, 4/1 heads of 256, took 146 us, 90 of them
// in join_kernel.
struct Found {
    int64_t share, base;  // base: the unit of the first step of (b, h)
    int b, h;
    Slots s;
};
template <typename S, bool kWaited>
__device__ __forceinline__ Found find(const AttendArgs& a, const Scratch& sc, int64_t nth, int shift) {
    const int lane = threadIdx.x & 31, heads = a.kv.nkv * sc.head_tiles, B = a.kv.n_seqs;
    auto units_at = [&](int b) {
        return b < B ? units_of<S>(slots_of<S::kSlots, kWaited>(a, b), heads) : (int64_t)0;
    };
    auto scan = [&](int64_t u) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, u, o);
            if (lane >= o) u += v;
        }
        return u;
    };
    int64_t upto = scan(units_at(lane));  // of the first 32 sequences
    const int64_t first = __shfl_sync(0xffffffffu, upto, 31);
    int64_t total = first;
    if (B > 32) {
        int64_t mine = 0;
#pragma unroll 4
        for (int b = 32 + lane; b < B; b += 32) mine += units_at(b);
        total += warp_sum64(mine);
    }
    Found f;
    f.share = share_of<S>(total, sc.grid);
    f.b = -1;
    const int64_t unit = f.share * nth + shift;
    if (unit >= total) return f;
    int64_t off = unit;
    int b0 = 0;  // the 32 sequences that hold it
    if (off >= first) {
        off -= first;
        int64_t held = -1;
        for (b0 = 32; held < 0;) {
            int64_t u[4], sum[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) u[r] = units_at(b0 + 32 * r + lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[r] = warp_sum64(u[r]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (held < 0) {
                    if (off < sum[r]) {
                        held = u[r];
                    } else {
                        off -= sum[r];
                        b0 += 32;
                    }
                }
        }
        upto = scan(held);
    }
    const int owner = __ffs(__ballot_sync(0xffffffffu, off < upto)) - 1;
    f.b = b0 + owner;
    if (owner) off -= __shfl_sync(0xffffffffu, upto, owner - 1);
    f.s = slots_of<S::kSlots, kWaited>(a, f.b);
    f.h = (int)(off / (f.s.tiles + S::kSetup));
    f.base = unit - (off - (int64_t)f.h * (f.s.tiles + S::kSetup)) + S::kSetup;
    return f;
}

// A query's largest element is brought to 2^kRaise: f16 parts of smaller elements
// keep their bits down to 2^-24 (from 1 on, one element of 2^15 among others of 1
// left those 2^-10 of error).
template <typename T>
constexpr int kRaise = std::is_same_v<T, __half> ? 14 : 0;

// Weights are relative to 2^m with m at most kSlack below the largest score so
// far (in units of log 2): the sums are rescaled when it grows by more, not at
// every new maximum (a few times a warp). f16 holds 2^-24 to 2^16: there the
// weights are scaled by 2^14, so that small ones keep their bits, and kSlack is 1.
template <typename T>
constexpr float kWeightBias = std::is_same_v<T, __half> ? 14.0f : 0.0f;
template <typename T>
constexpr float kSlack = std::is_same_v<T, __half> ? 1.0f : 8.0f;

// A piece of one query head in 32 bits, by a warp, where the products by parts are
// not finite: what an infinity in K or V meets, a part of zero or of the other sign,
// makes NaN of it. Lanes sum the four columns at v_cols of their own; known: M and L
// are, and only the columns asked for. scores null, or the head's row of them. For
// data with infinities only: 131071 slots of 64/8 heads of 128, bf16, with some in
// every page take 3.4 ms instead of 93 us.
template <typename T>
struct PlainPiece {
    const float* q;
    const T* k;  // the kv head's rows
    const T* v_cols;
    const int* table;
    int64_t page_stride, slot_stride;
    int page_shift, n_pages, first, last;  // slots [first, last)
    float scale;                           // log2(e) in it
    float* scores;
};
template <typename T, int HD>
__device__ __noinline__ float4 plain_piece(PlainPiece<T> a, bool known, float& M, float& L) {
    constexpr int kElems = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
    auto row_of = [&](int slot) -> int64_t {
        const int page = slot < a.last ? a.table[slot >> a.page_shift] : -1;
        if (page < 0 || page >= a.n_pages) return -1;
        return page * a.page_stride + (slot & ((1 << a.page_shift) - 1)) * a.slot_stride;
    };
    auto score = [&](int64_t row) {
        if (row < 0) return -INFINITY;
        float s = 0.0f;
#pragma unroll 1
        for (int u = 0; u < HD / kElems; ++u) {
            const uint4 bits = *reinterpret_cast<const uint4*>(a.k + row + u * kElems);
            const T* e = reinterpret_cast<const T*>(&bits);
#pragma unroll
            for (int i = 0; i < kElems; ++i) s = fmaf(a.q[u * kElems + i], kv_to_f32<T>(e[i]), s);
        }
        return s * a.scale;
    };
    if (!known) {
        bool nan = false;
        for (int d = lane; d < HD; d += 32) nan = nan || a.q[d] != a.q[d];
        if (__any_sync(0xffffffffu, nan)) return make_float4(NAN, NAN, NAN, NAN);  // and L is as it was
        M = -INFINITY;
        nan = false;
        for (int slot = a.first + lane; slot < a.last; slot += 32) {
            const float s = score(row_of(slot));
            if (a.scores) a.scores[slot] = s;
            nan = nan || s != s;
            M = fmaxf(M, s);
        }
        M = warp_max(M);
        if (__any_sync(0xffffffffu, nan)) return make_float4(NAN, NAN, NAN, NAN);
    }
    const float zero = M == -INFINITY ? 0.0f : M - kWeightBias<T>;
    float sum = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    for (int s0 = a.first; s0 < a.last; s0 += 32) {
        const int64_t mine = row_of(s0 + lane);
        const float p_mine = ex2(score(mine) - zero);
        sum += p_mine;
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
            const int64_t row = __shfl_sync(0xffffffffu, mine, i);
            const float p = __shfl_sync(0xffffffffu, p_mine, i);
            if (row < 0) continue;
            const T* v = a.v_cols + row;
            o.x += p * kv_to_f32<T>(v[0]);
            o.y += p * kv_to_f32<T>(v[1]);
            o.z += p * kv_to_f32<T>(v[2]);
            o.w += p * kv_to_f32<T>(v[3]);
        }
    }
    if (!known) L = warp_sum(sum);
    return o;
}

// Every warp takes each kWarps-th step of the piece, and runs on its own until
// the piece ends. The lane layout of the matrix instructions is met without a
// transpose: lane (g, t) = (lane / 4, lane % 4)
//  * as operand B of S = Q K^T holds K row g of 8 slots, at column pairs that
//    depend on t. Which columns is free as long as Q has the same order, so it
//    takes whole 16-byte units t, t + 4, ... of the row;
//  * as operand A of O^T = V^T P^T holds rows (columns of V) g and g + 8, at the
//    slot pairs 2 t, 2 t + 1 (+ 8, + 9). Which columns is free again: it takes 8
//    (f32: 4) consecutive ones, two by two, and pairs two slots' values by byte
//    permutes (16 bit).
// S's layout is that of the operand B of V^T P^T: P stays in registers.
// In S, operand A has 16 rows for the 8 heads of a set: rows 0-7 are the first,
// rows 8-15 the second parts of Q, so the products are those of f32 queries with
// the cache's, at no cost (a third part takes an instruction); P's parts take an
// instruction each. (O = P V
// with the parts as rows took as many, but twice the accumulators: 8 warps per SM
// for 16.) K and V in f32
// are split too.
template <typename T, int HD, int SETS>
__global__ void __launch_bounds__(Shape<T, HD, SETS>::kWarps * 32, Shape<T, HD, SETS>::kCtas)
    attend_kernel(const AttendArgs a, const Scratch sc) {
    using S = Shape<T, HD, SETS>;
    constexpr int W = S::kWarps, kSlots = S::kSlots, kTiles = S::kTiles, kTile = S::kTile;
    constexpr int kElems = 16 / (int)sizeof(T);  // of a 16-byte unit
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * S::kUnits * S::kUnit;
    // Eight neighbouring lanes copy a line: with the lines' quarters copied by lanes apart each was
    // fetched from L2 twice (131071 slots, 64/8 heads of 128, bf16: 807 MB for 537, 111 us for 90).
    // A row's 16-byte units lie in the ring exchanged within their line so that neither the copies (eight
    // lanes a line) nor the reads (K: four lanes a row, two rows at a time; V: two units of four rows) meet
    // in a bank: unit c of K row r at c ^ 4 (r % 2), of V row r at c ^ 2 (r / 2 % 4).
    const uint32_t dst = smem_u32(ring) + (lane >> 3) * S::kRow;
    const uint32_t k_dst = dst + ((lane & 7) ^ (((lane >> 3) & 1) * 4)) * 16;
    const uint32_t v_dst[2] = {dst + ((lane & 7) ^ ((lane >> 4) * 2)) * 16,
                               dst + ((lane & 7) ^ ((lane >> 4) * 2) ^ 4) * 16};
    const uint8_t* k_src = ring + g * S::kRow + t * 16;
    const int k_half[2] = {(g & 1) * 64, 64 - (g & 1) * 64};
    const uint8_t* v_src = ring + 2 * t * S::kRow + (g ^ (2 * t)) * 16;
    uint8_t* qs = smem + W * S::kUnits * S::kUnit;
    float2* ml_s = reinterpret_cast<float2*>(qs + SETS * S::kQBytes);  // [W][kHeads]
    float* unit_s = reinterpret_cast<float*>(ml_s + W * S::kHeads);    // [kHeads]
    const int group = a.nq / a.kv.nkv;
    const int heads = a.kv.nkv * sc.head_tiles;  // head tiles of a sequence

    // join_kernel reads the lengths and the running weights before it waits for this kernel: it may start
    // only once all that came before has ended, the last join among it
    pdl_wait();
    pdl_launch_dependents();

    const Found found = find<S, true>(a, sc, blockIdx.x, 0);
    if (found.b < 0) return;
    const int64_t share = found.share, begin = share * blockIdx.x, end = begin + share;
    int b = found.b, h = found.h;
    int64_t base = found.base;
    Slots s = found.s;

    while (base < end) {
        const int tile = (int)max(begin - base, (int64_t)0);
        const int count = (int)min(end - base, (int64_t)s.tiles) - tile;  // at least 1: see the step to the next
        const int kvh = h / sc.head_tiles, q0 = (h - kvh * sc.head_tiles) * S::kHeads;
        const int nh = min(S::kHeads, group - q0);
        const int head0 = kvh * group + q0;
        const int* table = a.kv.table + b * a.kv.table_stride;
        const int mask = (1 << a.kv.page_shift) - 1;
        const int my = count > warp ? (count - warp + W - 1) / W : 0;  // steps of this warp
        const int my_slot0 = (s.tile0 + tile + warp) * kSlots;         // step i starts at slot my_slot0 + i W kSlots

        // The pages of a step's tiles (a tile lies in one page), -1: none.
        struct Pages {
            int p[kTiles];
        };
        auto pages_of = [&](int i) {
            Pages r;
#pragma unroll
            for (int u = 0; u < kTiles; ++u) {
                const int slot = my_slot0 + i * (W * kSlots) + u * kTile;
                r.p[u] = i < my && slot < s.n ? table[slot >> a.kv.page_shift] : -1;
            }
            return r;
        };
        // Copies step i's rows of K (or V) into a unit of the ring; zeros where a slot is not seen.
        auto issue = [&](int i, const Pages& pages, const void* pool, int unit, bool is_v) {
            if (i < my) {
#pragma unroll
                for (int u = 0; u < kTiles; ++u) {
                    const int slot0 = my_slot0 + i * (W * kSlots) + u * kTile;
                    const int page = pages.p[u];
                    const bool ok = page >= 0 && page < a.kv.n_pages;
                    const T* rows = static_cast<const T*>(pool) + ((ok ? page : 0) * a.kv.page_stride +
                                                                   kvh * a.kv.head_stride +
                                                                   (slot0 & mask) * a.kv.slot_stride);
                    // four rows' 128-byte lines an instruction, a line by eight neighbouring lanes
#pragma unroll
                    for (int r = 0; r < kTile / 4; ++r) {
                        const int row = 4 * r + (lane >> 3);
                        const T* src = rows + row * a.kv.slot_stride + (lane & 7) * kElems;
                        const bool live = ok && slot0 + row >= s.first && slot0 + row < s.n;
                        const uint32_t dst = (is_v ? v_dst[r & 1] : k_dst) + unit * S::kUnit +
                                             (u * kTile + 4 * r) * S::kRow;
#pragma unroll
                        for (int j = 0; j < S::kLines; ++j) copy16(dst + j * 128, src + j * 8 * kElems, live);
                    }
                }
            }
            copy_commit();
        };
        // K of step i is issued a step ahead, V half a step later, their page numbers half a step before
        Pages pages = pages_of(0);
        issue(0, pages, a.kv.k, 0, false);
        issue(0, pages, a.kv.v, 1, true);
        Pages seen = pages;
        pages = pages_of(1);

        // Q of the head tile in the order of operand A, its power of two taken out
        for (int j = warp; j < S::kHeads; j += W) {
            const float* q = a.q + b * a.ldq + (int64_t)(head0 + j) * HD;
            float x[HD / 32], top = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                x[i] = j < nh ? q[lane + 32 * i] : 0.0f;
                top = fmaxf(top, fabsf(x[i]));
            }
            top = warp_max(top);
            int e = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
            e = max(-126, min(127, e - kRaise<T>));
            const float down = exp2f((float)-e);
            if (lane == 0) unit_s[j] = a.scale * kLog2e * exp2f((float)e);
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                const int d = lane + 32 * i, c = d / kElems, r = d % kElems;
                const int step = (c >> 2) * 2 + r / (kElems / 2), p = r % (kElems / 2);
                T part[kParts<T>];
                split<T>(x[i] * down, part);
                uint8_t* set = qs + (j >> 3) * S::kQBytes;
                const int at = step * 32 + (j & 7) * 4 + (c & 3);
                T* dst = reinterpret_cast<T*>(set + at * 16);
                if constexpr (sizeof(T) == 4) {
                    dst[2 * p] = part[0];
                    dst[2 * p + 1] = part[1];
                } else {
                    dst[(p >> 1) * 4 + (p & 1)] = part[0];
                    dst[(p >> 1) * 4 + 2 + (p & 1)] = part[1];
                    if constexpr (kParts<T> == 3) reinterpret_cast<T*>(set + S::kQPairs + at * 8)[p] = part[2];
                }
            }
        }
        __syncthreads();
        const uint8_t* qs_l = qs + lane * 16;
        const uint8_t* qs3_l = qs + S::kQPairs + lane * 8;
        float unit[SETS], m[SETS], l[SETS], lc[SETS];
        float* srow[SETS];
        float acc[SETS][HD / 16][4];  // [two columns]: head 2 t, head 2 t + 1 at the first; the same at the second
#pragma unroll
        for (int q = 0; q < SETS; ++q) {
            unit[q] = unit_s[8 * q + g];
            srow[q] = sc.scores && 8 * q + g < nh
                          ? sc.scores + ((int64_t)b * a.nq + head0 + 8 * q + g) * a.kv.capacity()
                          : nullptr;
            m[q] = -INFINITY;
            l[q] = lc[q] = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) acc[q][i][0] = acc[q][i][1] = acc[q][i][2] = acc[q][i][3] = 0.0f;
        }

        int at = 0;  // the unit of K of step i; V follows
        for (int i = 0; i < my; ++i) {
            const int at_v = at == 2 ? 0 : at + 1, spare = at_v == 2 ? 0 : at_v + 1;
            copy_wait<1>();
            __syncwarp();  // the other lanes' copies have landed too, and they have read the spare unit
            issue(i + 1, pages, a.kv.k, spare, false);
            const Pages after = pages_of(i + 2);
            const uint8_t* src = k_src + at * S::kUnit;
            // scores: per 8 slots and set two chains of at most four instructions, whose sums are added in 32
            // bits (an instruction cuts off where it adds; a unit of f32 or bf16 rows takes two of a chain, one
            // of f16 rows one). Chains of eight: f32 1.6 times as far from the exact outputs as elementary f32
            // operations, bf16 1.3 times; of four: 1.3 and 1.1 times, in up to 3% more time (16 heads on one of
            // 256, bf16: 60 us for 58).
            constexpr int kX = kSlots / 4, kR = kSlots / 8 < 2 ? 1 : 2;
            constexpr int kMost = S::kChunks % 4 == 0 ? 4 : (S::kChunks % 3 == 0 ? 3 : 2);  // units of an f16 chain
            constexpr int kRun = std::is_same_v<T, __half> ? kMost : 2;
            static_assert(S::kChunks % kRun == 0, "runs divide a row");
            float x[SETS][kX] = {};
#pragma unroll
            for (int r0 = 0; r0 < kSlots / 8; r0 += kR) {
#pragma unroll
                for (int j0 = 0; j0 < S::kChunks; j0 += kRun) {
                    float c0[kR][SETS][4] = {}, c1[kR][SETS][4] = {};
#pragma unroll
                    for (int j = j0; j < j0 + kRun; ++j) {
                        uint4 k[kR];
#pragma unroll
                        for (int r = 0; r < kR; ++r)
                            k[r] = lds16(src + 8 * (r0 + r) * S::kRow + (j >> 1) * 128 + k_half[j & 1]);
#pragma unroll
                        for (int q = 0; q < SETS; ++q) {
                            const uint4 qa = lds16(qs_l + q * S::kQBytes + (2 * j) * 512);
                            const uint4 qb = lds16(qs_l + q * S::kQBytes + (2 * j + 1) * 512);
                            uint2 ta = make_uint2(0, 0), tb = ta;
                            if constexpr (kParts<T> == 3) {
                                ta = *reinterpret_cast<const uint2*>(qs3_l + q * S::kQBytes + (2 * j) * 256);
                                tb = *reinterpret_cast<const uint2*>(qs3_l + q * S::kQBytes + (2 * j + 1) * 256);
                            }
#pragma unroll
                            for (int r = 0; r < kR; ++r) {
                                if constexpr (sizeof(T) == 4) {
                                    float f0[2], f1[2], f2[2], f3[2];
                                    split<T>(__uint_as_float(k[r].x), f0);
                                    split<T>(__uint_as_float(k[r].y), f1);
                                    split<T>(__uint_as_float(k[r].z), f2);
                                    split<T>(__uint_as_float(k[r].w), f3);
#pragma unroll
                                    for (int e = 1; e >= 0; --e) {
                                        mma<T>(c0[r][q], qa, __float_as_uint(f0[e]), __float_as_uint(f1[e]));
                                        mma<T>(c1[r][q], qb, __float_as_uint(f2[e]), __float_as_uint(f3[e]));
                                    }
                                } else {
                                    if constexpr (kParts<T> == 3) {
                                        mma<T>(c0[r][q], make_uint4(ta.x, 0, ta.y, 0), k[r].x, k[r].y);
                                        mma<T>(c1[r][q], make_uint4(tb.x, 0, tb.y, 0), k[r].z, k[r].w);
                                    }
                                    mma<T>(c0[r][q], qa, k[r].x, k[r].y);
                                    mma<T>(c1[r][q], qb, k[r].z, k[r].w);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < kR; ++r)
#pragma unroll
                        for (int q = 0; q < SETS; ++q) {
                            x[q][2 * (r0 + r)] += (c0[r][q][0] + c1[r][q][0]) + (c0[r][q][2] + c1[r][q][2]);
                            x[q][2 * (r0 + r) + 1] += (c0[r][q][1] + c1[r][q][1]) + (c0[r][q][3] + c1[r][q][3]);
                        }
                }
            }
#pragma unroll
            for (int q = 0; q < SETS; ++q)
#pragma unroll
                for (int r = 0; r < kX; ++r) x[q][r] *= unit[q];
            // lane (g, t) has the scores of heads g, g + 8 at slots 2 t, 2 t + 1 of every eight
            const int slot0 = my_slot0 + i * (W * kSlots);
            bool whole = slot0 >= s.first && slot0 + kSlots <= s.n;
#pragma unroll
            for (int u = 0; u < kTiles; ++u) whole = whole && seen.p[u] >= 0 && seen.p[u] < a.kv.n_pages;
            if (!whole) {
#pragma unroll
                for (int r = 0; r < kX; ++r) {
                    const int slot = slot0 + 2 * t + (r & 1) + 8 * (r >> 1);
                    const int page = seen.p[r * 4 / kTile];
                    if (page < 0 || page >= a.kv.n_pages || slot < s.first || slot >= s.n)
#pragma unroll
                        for (int q = 0; q < SETS; ++q) x[q][r] = -INFINITY;
                }
            }
            uint2 p[SETS][kTiles][kParts<T>];  // operand B of each part
#pragma unroll
            for (int q = 0; q < SETS; ++q) {
                if (srow[q]) {
#pragma unroll
                    for (int r = 0; r < kX; ++r) {
                        const int slot = slot0 + 2 * t + (r & 1) + 8 * (r >> 1);
                        if (slot >= s.first && slot < s.n) srow[q][slot] = x[q][r];
                    }
                }
                float top = x[q][0];
#pragma unroll
                for (int r = 1; r < kX; ++r) top = fmaxf(top, x[q][r]);
                top = quad_max(top);
                if (__any_sync(0xffffffffu, top > m[q] + kSlack<T>)) {
                    const float up = fmaxf(m[q], top), f = up == -INFINITY ? 1.0f : ex2(m[q] - up);
                    const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j) {
                        acc[q][j][0] *= f0;
                        acc[q][j][1] *= f1;
                        acc[q][j][2] *= f0;
                        acc[q][j][3] *= f1;
                    }
                    l[q] *= f;
                    lc[q] *= f;
                    m[q] = up;
                }
                const float zero = m[q] == -INFINITY ? 0.0f : m[q] - kWeightBias<T>;
                float sum = 0.0f;
#pragma unroll
                for (int r = 0; r < kX; ++r) {
                    x[q][r] = ex2(x[q][r] - zero);
                    sum += x[q][r];
                }
                // the rounding error of the sum is carried along: many small weights beside a large one count
                lc[q] += sum;
                const float l2 = l[q] + lc[q];
                lc[q] -= l2 - l[q];
                l[q] = l2;
#pragma unroll
                for (int u = 0; u < kTiles; ++u) {
                    if constexpr (sizeof(T) == 4) {
                        float f0[2], f1[2];
                        split<T>(x[q][2 * u], f0);
                        split<T>(x[q][2 * u + 1], f1);
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            p[q][u][e] = make_uint2(__float_as_uint(f0[e]), __float_as_uint(f1[e]));
                    } else {
                        uint32_t f0[kParts<T>], f1[kParts<T>];
                        split2<T>(x[q][4 * u], x[q][4 * u + 1], f0);
                        split2<T>(x[q][4 * u + 2], x[q][4 * u + 3], f1);
#pragma unroll
                        for (int e = 0; e < kParts<T>; ++e) p[q][u][e] = make_uint2(f0[e], f1[e]);
                    }
                }
            }
            copy_wait<1>();
            __syncwarp();  // every lane has read K's unit
            issue(i + 1, pages, a.kv.v, at, true);
            seen = pages;
            pages = after;
            src = v_src + at_v * S::kUnit;
#pragma unroll
            for (int u = 0; u < kTiles; ++u)
#pragma unroll
                for (int j = 0; j < S::kLines; ++j) {
                    uint4 v[S::kVRows];
#pragma unroll
                    for (int r = 0; r < S::kVRows; ++r)
                        v[r] = lds16(src + (u * kTile + (r & 1) + 8 * (r >> 1)) * S::kRow + j * 128);
                    const uint32_t v0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, v1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
                    if constexpr (sizeof(T) == 4) {
                        // high V with both parts of P, low V with the high one: the rest is below 2^-22
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float f[4][2];
                            split<T>(__uint_as_float(v0[2 * e]), f[0]);
                            split<T>(__uint_as_float(v0[2 * e + 1]), f[1]);
                            split<T>(__uint_as_float(v1[2 * e]), f[2]);
                            split<T>(__uint_as_float(v1[2 * e + 1]), f[3]);
                            const uint4 vh = make_uint4(__float_as_uint(f[0][0]), __float_as_uint(f[1][0]),
                                                        __float_as_uint(f[2][0]), __float_as_uint(f[3][0]));
                            const uint4 vl = make_uint4(__float_as_uint(f[0][1]), __float_as_uint(f[1][1]),
                                                        __float_as_uint(f[2][1]), __float_as_uint(f[3][1]));
#pragma unroll
                            for (int q = 0; q < SETS; ++q) {
                                float c[4];
                                float(&d)[4] = S::kFresh ? c : acc[q][j * 2 + e];
                                if (S::kFresh) c[0] = c[1] = c[2] = c[3] = 0.0f;
                                mma<T>(d, vl, p[q][u][0].x, p[q][u][0].y);
                                mma<T>(d, vh, p[q][u][1].x, p[q][u][1].y);
                                mma<T>(d, vh, p[q][u][0].x, p[q][u][0].y);
                                if (S::kFresh)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) acc[q][j * 2 + e][i] += c[i];
                            }
                        }
                    } else {
                        const uint32_t v2[4] = {v[2].x, v[2].y, v[2].z, v[2].w};
                        const uint32_t v3[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint4 vv = make_uint4(__byte_perm(v0[e], v1[e], 0x5410),
                                                        __byte_perm(v0[e], v1[e], 0x7632),
                                                        __byte_perm(v2[e], v3[e], 0x5410),
                                                        __byte_perm(v2[e], v3[e], 0x7632));
#pragma unroll
                            for (int q = 0; q < SETS; ++q) {
                                float c[4];
                                float(&d)[4] = S::kFresh ? c : acc[q][j * 4 + e];
                                if (S::kFresh) c[0] = c[1] = c[2] = c[3] = 0.0f;
#pragma unroll
                                for (int f = kParts<T> - 1; f >= 0; --f) mma<T>(d, vv, p[q][u][f].x, p[q][u][f].y);
                                if (S::kFresh)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) acc[q][j * 4 + e][i] += c[i];
                            }
                        }
                    }
                }
            at = spare;
        }
        copy_wait<0>();

        // the warps' results, each in its own ring: heads 2 t, 2 t + 1 of a set, the columns of the lane's V units
        float* mine_s = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int q = 0; q < SETS; ++q) {
#pragma unroll
            for (int j = 0; j < S::kLines; ++j)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = 0; e < kElems; e += 4) {
                        const int i = (j * kElems + e) / 2;
                        *reinterpret_cast<float4*>(mine_s + (8 * q + 2 * t + half) * S::kAccRow + (j * 8 + g) * kElems +
                                                   e) = make_float4(acc[q][i][half], acc[q][i][2 + half],
                                                                    acc[q][i + 1][half], acc[q][i + 1][2 + half]);
                    }
            const float sum = quad_sum(l[q] + lc[q]);
            if (t == 0) ml_s[warp * S::kHeads + 8 * q + g] = make_float2(m[q], sum);
        }
        __syncthreads();
        const bool begins = tile == 0, ends = tile + count == s.tiles;
        const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
        struct Sums {
            float M, L;
            float4 o;
        };
        auto sums_of = [&](int j, int d) {  // of the warps, at four columns of a head
            Sums r = {-INFINITY, 0.0f, make_float4(0, 0, 0, 0)};
#pragma unroll
            for (int w = 0; w < W; ++w) r.M = fmaxf(r.M, ml_s[w * S::kHeads + j].x);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float2 ml = ml_s[w * S::kHeads + j];
                const float f = piece_factor(ml.x, r.M);
                r.L += ml.y * f;
                const float4 p = *reinterpret_cast<const float4*>(
                    reinterpret_cast<const float*>(smem + w * S::kUnits * S::kUnit) + j * S::kAccRow + d);
                r.o.x += p.x * f;
                r.o.y += p.y * f;
                r.o.z += p.z * f;
                r.o.w += p.w * f;
            }
            return r;
        };
        auto store = [&](int j, int d, const Sums& r) {
            if (begins && ends) {
                const float inv = r.L > 0.0f ? 1.0f / r.L : 0.0f;
                *reinterpret_cast<float4*>(a.out + ((int64_t)b * a.nq + head0 + j) * HD + d) =
                    make_float4(r.o.x * inv, r.o.y * inv, r.o.z * inv, r.o.w * inv);
                if (sc.whole && d == 0) sc.whole[(int64_t)b * a.nq + head0 + j] = make_float2(r.M, r.L);
            } else {
                *reinterpret_cast<float4*>(sc.acc + ((int64_t)slot * S::kHeads + j) * HD + d) = r.o;
                if (d == 0) sc.ml[slot * S::kHeads + j] = make_float2(r.M, r.L);
            }
        };
        auto finite = [](const Sums& r) {
            return r.L < INFINITY && fabsf((r.o.x + r.o.y) + (r.o.z + r.o.w)) < INFINITY;
        };
        bool bad = false;
        for (int i = threadIdx.x; i < nh * (HD / 4); i += W * 32) {
            const int j = i / (HD / 4), d = 4 * (i - j * (HD / 4));
            const Sums r = sums_of(j, d);
            bad = bad || !finite(r);
            store(j, d, r);
        }
        if (__any_sync(0xffffffffu, bad)) {  // the warp takes its own columns again, head by head
            for (int i0 = warp * 32; i0 < nh * (HD / 4); i0 += W * 32) {
                const int i = min(i0 + lane, nh * (HD / 4) - 1), j = i / (HD / 4), d = 4 * (i - j * (HD / 4));
                Sums r = sums_of(j, d);
                unsigned left = __ballot_sync(0xffffffffu, !finite(r));
                while (left) {
                    const int head = __shfl_sync(0xffffffffu, j, __ffs(left) - 1);
                    left &= ~__ballot_sync(0xffffffffu, j == head);
                    PlainPiece<T> plain;
                    plain.q = a.q + b * a.ldq + (int64_t)(head0 + head) * HD;
                    plain.k = static_cast<const T*>(a.kv.k) + kvh * a.kv.head_stride;
                    plain.v_cols = static_cast<const T*>(a.kv.v) + kvh * a.kv.head_stride + d;
                    plain.table = table;
                    plain.page_stride = a.kv.page_stride;
                    plain.slot_stride = a.kv.slot_stride;
                    plain.page_shift = a.kv.page_shift;
                    plain.n_pages = (int)a.kv.n_pages;
                    plain.first = max(s.first, (s.tile0 + tile) * kSlots);
                    plain.last = min(s.n, (s.tile0 + tile + count) * kSlots);
                    plain.scale = a.scale * kLog2e;
                    plain.scores =
                        sc.scores ? sc.scores + ((int64_t)b * a.nq + head0 + head) * a.kv.capacity() : nullptr;
                    const int owner = __ffs(__ballot_sync(0xffffffffu, j == head)) - 1;
                    float M = __shfl_sync(0xffffffffu, r.M, owner), L = __shfl_sync(0xffffffffu, r.L, owner);
                    const bool known = L < INFINITY;
                    const float4 v = plain_piece<T, HD>(plain, known, M, L);
                    if (j != head) continue;
                    if (!known || !(fabsf(r.o.x) < INFINITY)) r.o.x = v.x;
                    if (!known || !(fabsf(r.o.y) < INFINITY)) r.o.y = v.y;
                    if (!known || !(fabsf(r.o.z) < INFINITY)) r.o.z = v.z;
                    if (!known || !(fabsf(r.o.w) < INFINITY)) r.o.w = v.w;
                    r.M = M;
                    r.L = L;
                    store(j, d, r);
                }
            }
        }
        base += s.tiles + S::kSetup;
        if (base >= end) return;
        if (++h == heads) {
            h = 0;
            do {
                if (++b == a.kv.n_seqs) return;
                s = slots_of<kSlots, true>(a, b);
            } while (s.tiles == 0);
        }
        __syncthreads();  // the rings and Q are rewritten
    }
}

// Joins the pieces of divided (sequence, head tile)s in the order of the CTAs
// that left them, and writes the zeros of sequences without slots. Few head tiles
// with many pieces: a CTA per head (kHeads 1). Many head tiles: a CTA per CTA of
// attend_kernel, for the one head tile at most that it begins and does not end,
// eight heads at once. A thread sums four columns of a head over every kGroups-th
// piece.
// It is on the way of every small call, so it is launched early (programmatic
// dependent launch, once attend_kernel's own wait is over), finds the pieces from
// the lengths before it waits for attend_kernel, and has one round of loads after
// it.
// With weights, the CTAs from join_blocks on add the slots' weights.
template <int HD, int kHeads>
struct JoinShape {
    static constexpr int kCols = HD / 4;
    static constexpr int kThreads = kHeads * kCols < 256 ? 256 : kHeads * kCols;
    static constexpr int kGroups = kThreads / (kHeads * kCols);
    static constexpr int kAhead = 4;        // pieces a thread loads before their factors are known
    static constexpr int kHeadsAtOnce = 32;  // of a weights CTA
};

// weights_out[b][kvh][t] = weights[b][kvh][t] + sum over the kv head's query
// heads of e^(s_t - m) / sum e^(s - m), four slots a thread.
template <typename T, typename S, int kThreads, int kHeadsAtOnce>
__device__ __forceinline__ void add_weights(const AttendArgs& a, const Scratch& sc, int64_t block) {
    __shared__ float2 zero_inv[kHeadsAtOnce];  // what to subtract from a score, what to multiply its power with
    const int64_t cap = a.kv.capacity();
    const int64_t blocks = (cap / 4 + kThreads - 1) / kThreads;  // of a (sequence, kv head)
    const int64_t row = block / blocks;
    const int b = (int)(row / a.kv.nkv), kvh = (int)(row - (int64_t)b * a.kv.nkv);
    const int64_t t = ((block - row * blocks) * kThreads + threadIdx.x) * 4;
    __shared__ Place place_s;
    if (threadIdx.x < 32) {
        const Place p = place_of<S>(a, sc, b);
        if (threadIdx.x == 0) place_s = p;
    }
    __syncthreads();
    const Place place = place_s;
    const Slots s = slots_of<S::kSlots>(a, b);
    const int64_t at = row * cap + t;
    const bool mine = t < cap && t < s.n && t + 4 > s.first;
    const bool copy = t < cap && !mine && a.weights_out != a.weights;
    float4 w = make_float4(0, 0, 0, 0);
    if (mine || copy) w = __ldcg(reinterpret_cast<const float4*>(a.weights + at));
    if (copy) *reinterpret_cast<float4*>(a.weights_out + at) = w;
    pdl_wait();
    if (s.tiles == 0) return;
    const int group = a.nq / a.kv.nkv;
    const int64_t head0 = (int64_t)b * a.nq + kvh * group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float p[4] = {0, 0, 0, 0};
    for (int g0 = 0; g0 < group; g0 += kHeadsAtOnce) {
        const int heads = min(kHeadsAtOnce, group - g0);
        if (g0) __syncthreads();
        for (int i = warp; i < heads; i += kThreads / 32) {
            const int j = g0 + i;
            const Pieces pc = place.pieces<S>(kvh * sc.head_tiles + j / S::kHeads);
            float M = -INFINITY, L = 0.0f;
            if (pc.count == 1) {
                const float2 ml = sc.whole[head0 + j];
                M = ml.x;
                L = ml.y;
            } else {
                for (int q = lane; q < pc.count; q += 32) M = fmaxf(M, sc.ml[pc.slot(q) * S::kHeads + j % S::kHeads].x);
                M = warp_max(M);
                for (int q = lane; q < pc.count; q += 32) {
                    const float2 ml = sc.ml[pc.slot(q) * S::kHeads + j % S::kHeads];
                    L += ml.y * piece_factor(ml.x, M);
                }
                L = warp_sum(L);
            }
            if (lane == 0) zero_inv[i] = L > 0.0f ? make_float2(M - kWeightBias<T>, 1.0f / L) : make_float2(0.0f, 0.0f);
        }
        __syncthreads();
        if (mine) {
#pragma unroll 4
            for (int i = 0; i < heads; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(sc.scores + (head0 + g0 + i) * cap + t);
                const float2 z = zero_inv[i];
                if (z.y > 0.0f) {
                    p[0] += ex2(x.x - z.x) * z.y;
                    p[1] += ex2(x.y - z.x) * z.y;
                    p[2] += ex2(x.z - z.x) * z.y;
                    p[3] += ex2(x.w - z.x) * z.y;
                }
            }
        }
    }
    if (!mine) return;
    auto in = [&](int i) { return t + i >= s.first && t + i < s.n; };  // scores elsewhere were not written
    if (in(0)) w.x += p[0];
    if (in(1)) w.y += p[1];
    if (in(2)) w.z += p[2];
    if (in(3)) w.w += p[3];
    *reinterpret_cast<float4*>(a.weights_out + at) = w;
}

template <typename T, int HD, int SETS, int kHeads>
__global__ void __launch_bounds__(JoinShape<HD, kHeads>::kThreads)
    join_kernel(const AttendArgs a, const Scratch sc, unsigned join_blocks) {
    using S = Shape<T, HD, SETS>;
    using J = JoinShape<HD, kHeads>;
    constexpr int kCols = J::kCols, kGroups = J::kGroups, kWarps = J::kThreads / 32, kAhead = J::kAhead;
    extern __shared__ float factors[];  // [kHeads][grid]
    __shared__ float4 part[kGroups][kHeads][kCols];
    __shared__ float inv_s[kHeads];
    pdl_launch_dependents();
    if (blockIdx.x >= join_blocks) {
        if (blockIdx.y == 0) add_weights<T, S, J::kThreads, J::kHeadsAtOnce>(a, sc, blockIdx.x - join_blocks);
        else pdl_wait();
        return;
    }
    const int group = a.nq / a.kv.nkv;
    const int unit = threadIdx.x / kCols, col = threadIdx.x - unit * kCols;
    const int grp = unit / kHeads, j = unit - grp * kHeads;
    __shared__ Found found_s;
    __shared__ bool divided_s;
    if (threadIdx.x < 32) {
        Found f;
        bool divided;
        if constexpr (kHeads == 1) {
            const int heads = a.kv.nkv * sc.head_tiles;
            f.b = blockIdx.x / (unsigned)heads;
            f.h = blockIdx.x - f.b * (unsigned)heads;
            const Place place = place_of<S>(a, sc, f.b);
            f.s = slots_of<S::kSlots>(a, f.b);
            f.share = place.share;
            f.base = place.start + (int64_t)f.h * (f.s.tiles + S::kSetup) + S::kSetup;
            divided = f.s.tiles > 0 && place.pieces<S>(f.h).count > 1;
        } else {  // that of the last unit of CTA c's share
            f = find<S, false>(a, sc, (int64_t)blockIdx.x + 1, -1);
            const int64_t bound = f.share * (blockIdx.x + 1);
            divided = f.b >= 0 && f.base < bound && f.base + f.s.tiles > bound && f.base / f.share == blockIdx.x;
        }
        if (threadIdx.x == 0) found_s = f, divided_s = divided;
    }
    __syncthreads();
    const Found f = found_s;
    const bool divided = divided_s;
    pdl_wait();
    for (int b = blockIdx.x; b < a.kv.n_seqs; b += join_blocks)
        if (blockIdx.y == 0 && slots_of<S::kSlots>(a, b).tiles == 0) {
            float4* out = reinterpret_cast<float4*>(a.out + (int64_t)b * a.nq * HD);
            for (int i = threadIdx.x; i < a.nq * (HD / 4); i += J::kThreads) out[i] = make_float4(0, 0, 0, 0);
        }
    if (!divided) return;
    const Pieces pc = pieces_of(f.base, f.s.tiles, f.share);
    const int kvh = f.h / sc.head_tiles, q0 = (f.h - kvh * sc.head_tiles) * S::kHeads;
    const int j0 = blockIdx.y * kHeads, nh = min(kHeads, min(S::kHeads, group - q0) - j0);
    if (nh <= 0) return;
    const int64_t head0 = (int64_t)f.b * a.nq + kvh * group + q0 + j0;
    float4* out = reinterpret_cast<float4*>(a.out + (head0 + j) * HD) + col;
    const bool mine = grp < kGroups && j < nh;
    auto load = [&](int p) {
        return reinterpret_cast<const float4*>(sc.acc + (pc.slot(p) * S::kHeads + j0 + j) * HD)[col];
    };
    float4 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (mine && grp + i * kGroups < pc.count) ahead[i] = load(grp + i * kGroups);
    // a warp per head: the factors e^(m - M) and the sum
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = warp; i < nh; i += kWarps) {
        const float2* ml = sc.ml + j0 + i;
        float2 first = lane < pc.count ? ml[pc.slot(lane) * S::kHeads] : make_float2(-INFINITY, 0.0f);
        float M = first.x, L = 0.0f;
        for (int p = lane + 32; p < pc.count; p += 32) M = fmaxf(M, ml[pc.slot(p) * S::kHeads].x);
        M = warp_max(M);
        for (int p = lane; p < pc.count; p += 32) {
            const float2 v = p == lane ? first : ml[pc.slot(p) * S::kHeads];
            const float f = piece_factor(v.x, M);
            factors[i * sc.grid + p] = f;
            L += v.y * f;
        }
        L = warp_sum(L);
        if (lane == 0) inv_s[i] = L > 0.0f ? 1.0f / L : 0.0f;
    }
    __syncthreads();
    float4 o = make_float4(0, 0, 0, 0);
    if (mine) {
        const float* f = factors + j * sc.grid;
        auto add = [&](const float4& v, int p) {
            o.x += v.x * f[p];
            o.y += v.y * f[p];
            o.z += v.z * f[p];
            o.w += v.w * f[p];
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (grp + i * kGroups < pc.count) add(ahead[i], grp + i * kGroups);
#pragma unroll 8
        for (int p = grp + kAhead * kGroups; p < pc.count; p += kGroups) add(load(p), p);
        part[grp][j][col] = o;
    }
    if constexpr (kGroups > 1) __syncthreads();
    if (grp > 0 || j >= nh) return;
#pragma unroll
    for (int q = 1; q < kGroups; ++q) {
        const float4 v = part[q][j][col];
        o.x += v.x;
        o.y += v.y;
        o.z += v.z;
        o.w += v.w;
    }
    const float inv = inv_s[j];
    *out = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

template <typename T, int HD, int SETS, int kHeads>
cudaError_t launch_join(AttendArgs a, Scratch sc, int grid_y, cudaStream_t st) {
    using J = JoinShape<HD, kHeads>;
    int64_t blocks = kHeads == 1 ? (int64_t)a.kv.n_seqs * a.kv.nkv * sc.head_tiles : sc.grid;
    unsigned join_blocks = (unsigned)blocks;
    if (a.weights)
        blocks += (int64_t)a.kv.n_seqs * a.kv.nkv * ((a.kv.capacity() / 4 + J::kThreads - 1) / J::kThreads);
    if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
    void* args[] = {&a, &sc, &join_blocks};
    return launch_pdl_kernel((const void*)join_kernel<T, HD, SETS, kHeads>, dim3((unsigned)blocks, grid_y),
                             dim3(J::kThreads), kHeads * sc.grid * sizeof(float), st, args);
}

template <typename T, int HD, int SETS>
cudaError_t launch(const AttendArgs& a, Scratch sc, int sms, cudaStream_t st) {
    using S = Shape<T, HD, SETS>;
    cudaError_t e = ensure_dynamic_smem((const void*)attend_kernel<T, HD, SETS>, S::kSmem);
    if (e != cudaSuccess) return e;
    sc.grid = sms * S::kCtas;
    AttendArgs aa = a;
    void* args[] = {&aa, &sc};
    e = launch_pdl_kernel((const void*)attend_kernel<T, HD, SETS>, dim3(sc.grid), dim3(S::kWarps * 32), S::kSmem, st,
                          args);
    if (e != cudaSuccess) return e;
    const int64_t tiles = (int64_t)a.kv.n_seqs * a.kv.nkv * sc.head_tiles;
    const int heads = a.nq / a.kv.nkv < S::kHeads ? a.nq / a.kv.nkv : S::kHeads;
    // Few heads: side by side, each by a CTA; from about two of those per SM on, the CTAs that find nothing to
    // join cost more (a CTA per head, one per share boundary: 64 heads in pieces of 131071 slots 91.2, 94.1 us;
    // 256 with a window of 512 15.4, 15.5; 512 heads of 2000 slots 16.4, 16.4; 768 of 300 17.1, 14.5; 1152 of
    // 1000 22.2, 19.0; 2048 of 1000 39.0, 31.1).
    if (tiles * heads <= 2 * sms) return launch_join<T, HD, SETS, 1>(a, sc, heads, st);
    return launch_join<T, HD, SETS, 8>(a, sc, SETS, st);
}

template <typename T, int HD>
cudaError_t launch_sets(const AttendArgs& a, const Scratch& sc, int sms, cudaStream_t st) {
    return pass_heads(a.kv, a.nq) == 8 ? launch<T, HD, 1>(a, sc, sms, st) : launch<T, HD, 2>(a, sc, sms, st);
}

template <typename T>
cudaError_t launch_hd(const AttendArgs& a, const Scratch& sc, int sms, cudaStream_t st) {
    switch (a.kv.hd) {
        case 64: return launch_sets<T, 64>(a, sc, sms, st);
        case 128: return launch_sets<T, 128>(a, sc, sms, st);
        case 192: return launch_sets<T, 192>(a, sc, sms, st);
        case 256: return launch_sets<T, 256>(a, sc, sms, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

}  // namespace qmm
