// Eviction from a paged key/value cache by accumulated attention weight
// (sm_100a). Per (sequence, kv head) with more than `budget` cached slots the
// kept slots are, in this order of preference: those of the last `recent`
// positions, then those with the most accumulated weight (equal weights: the
// lowest slot first; NaN ranks with -infinity). Kept slots at or above
// `budget` move into the evicted slots below it, the r-th of the former into
// the r-th of the latter: attention does not depend on the order of the
// slots (each keeps its own position), a move reads slots that no move
// writes, and no more rows are moved than have to be.
//
// Two launches: select_kernel finds the kept slots of a row (a (sequence, kv
// head)) with one CTA, or a cluster of up to eight for long rows, and lists the
// holes and the movers; move_kernel copies K and V rows with the whole GPU.
// Few or short rows are bound by select_kernel's chain of passes and barriers,
// many moved rows by HBM (each is read and written once).
#include "qmm_common.cuh"
#include "qmm_gemv_xsmem.cuh"
#include "qmm_kernels.cuh"
#include "qmm_paged.cuh"

namespace qmm {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kPer = 8;                    // consecutive slots of a thread in a round
constexpr int kRound = kSelectThreads * kPer;    // slots a CTA takes in a round
constexpr int kMaxCluster = 8;             // the portable size
constexpr int kDigits = 256;
constexpr int kCopies = 8;                 // of a histogram: neighbouring lanes count in different ones

// Unsigned order of the preference: a total order on the floats, protected
// slots above all of them. w + 0 turns -0 into +0, its equal.
__device__ __forceinline__ uint32_t slot_key(float w, bool is_recent) {
    if (is_recent) return 0xffffffffu;
    if (w != w) w = -INFINITY;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int warp_scan(int v) {  // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}
// Exclusive prefix of v over the CTA's threads; *total is the CTA's sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = warp_scan(v);
    __syncthreads();  // warp_sums is reused between calls
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    const int all = warp_scan(warp_sums[lane]);
    *total = __shfl_sync(0xffffffffu, all, 31);
    const int before = __shfl_sync(0xffffffffu, all, (warp + 31) & 31);
    return (warp ? before : 0) + s - v;
}
__device__ __forceinline__ int ld_cluster_s32(const int* local, uint32_t rank) {
    return __float_as_int(ld_cluster_f32(reinterpret_cast<const float*>(local), rank));
}

// What select_kernel leaves for move_kernel. list[row][slot range of a CTA]:
// its holes from the range's start, its movers from the range's start or the
// budget, whichever is later (the holes end before); counts per row and CTA.
struct Lists {
    int* list;     // [rows][capacity]
    int2* counts;  // [rows][kMaxCluster]: holes, movers
    int ctas;      // per row
    int range;     // slots of a CTA, a multiple of kPer
};

struct Row {
    int64_t base;  // of the row in weights and positions
    int n, kept;
    int64_t limit;  // positions from here on are protected
};
__device__ __forceinline__ Row row_of(const EvictArgs& a, int row) {
    const int b = row / a.kv.nkv;
    const int64_t cap = a.kv.capacity();
    Row r;
    r.base = row * cap;
    const int n = a.lengths[b];
    r.n = n < 0 ? 0 : (n > cap ? (int)cap : n);
    r.kept = r.n < a.budget ? r.n : a.budget;
    r.limit = (int64_t)a.next_positions[b] - a.recent;
    return r;
}

// The threshold by four rounds of counting 8-bit digits, from the top: after
// each, the digit of the budget-th preferred key among those that match the
// digits so far. kCluster: the CTAs of a row count their ranges and add up each
// other's counts through distributed shared memory.
template <bool kCluster>
__global__ void __launch_bounds__(kSelectThreads) select_kernel(const EvictArgs a, const Lists ls) {
    __shared__ int hist[kCopies][kDigits + 4];
    __shared__ int counts[4][kDigits];  // of this CTA, per digit round
    __shared__ int warp_sums[32];
    __shared__ int s_digit, s_left;
    const int row = blockIdx.y, rank = kCluster ? (int)blockIdx.x : 0;
    const Row r = row_of(a, row);
    const int64_t cap = a.kv.capacity();
    const int begin = rank * ls.range, end = (int)min((int64_t)begin + ls.range, cap);
    const int live = min(end, r.n);  // slots of mine that are cached: [begin, live)
    const float* w = a.weights + r.base;
    const int* pos = a.positions + r.base;
    float* w_out = a.weights_out + r.base;
    int* pos_out = a.positions_out + r.base;
    if (rank == 0 && row % a.kv.nkv == 0 && threadIdx.x == 0) a.lengths_out[row / a.kv.nkv] = r.kept;
    const int tid8 = threadIdx.x * kPer;

    struct Slots8 {
        float w[kPer];
        int p[kPer];
    };
    auto load = [&](int t) {
        Slots8 s;
        *reinterpret_cast<float4*>(s.w) = *reinterpret_cast<const float4*>(w + t);
        *reinterpret_cast<float4*>(s.w + 4) = *reinterpret_cast<const float4*>(w + t + 4);
        *reinterpret_cast<int4*>(s.p) = *reinterpret_cast<const int4*>(pos + t);
        *reinterpret_cast<int4*>(s.p + 4) = *reinterpret_cast<const int4*>(pos + t + 4);
        return s;
    };
    auto store = [&](int t, const Slots8& s) {
        *reinterpret_cast<float4*>(w_out + t) = *reinterpret_cast<const float4*>(s.w);
        *reinterpret_cast<float4*>(w_out + t + 4) = *reinterpret_cast<const float4*>(s.w + 4);
        *reinterpret_cast<int4*>(pos_out + t) = *reinterpret_cast<const int4*>(s.p);
        *reinterpret_cast<int4*>(pos_out + t + 4) = *reinterpret_cast<const int4*>(s.p + 4);
    };
    // what lies beyond the kept slots, and all of a row that is short enough
    const bool full = r.n > a.budget;
    for (int t = begin + tid8; t < end; t += kRound) {
        if (full && t < r.kept) continue;
        Slots8 s;
        if (t < r.kept) s = load(t);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (t + i >= r.kept) s.w[i] = 0.0f, s.p[i] = -1;
        if (!full || t >= r.kept) store(t, s);
    }
    if (!full) {
        if (threadIdx.x == 0) ls.counts[(int64_t)row * kMaxCluster + rank] = make_int2(0, 0);
        return;
    }

    uint32_t prefix = 0;
    int need = a.budget;  // slots still to take among those that match the prefix
#pragma unroll 1
    for (int round = 0; round < 4; ++round) {
        const int shift = 24 - 8 * round;
        for (int i = threadIdx.x; i < kCopies * (kDigits + 4); i += kSelectThreads) (&hist[0][0])[i] = 0;
        __syncthreads();
        int* mine = hist[threadIdx.x & (kCopies - 1)];
        for (int t = begin + tid8; t < live; t += kRound) {
            const Slots8 s = load(t);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const uint32_t key = slot_key(s.w[i], s.p[i] >= r.limit);
                if (t + i < live && (round == 0 || ((key ^ prefix) >> (shift + 8)) == 0))
                    atomicAdd(&mine[(key >> shift) & (kDigits - 1)], 1);
            }
        }
        __syncthreads();
        if (threadIdx.x < kDigits) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) c += hist[i][threadIdx.x];
            counts[round][threadIdx.x] = c;
        }
        if constexpr (kCluster) cluster_sync();
        else __syncthreads();
        // thread i has digit 255 - i: the first whose running count reaches `need`
        const int d = kDigits - 1 - (int)threadIdx.x;
        int c = 0;
        if (threadIdx.x < kDigits) {
            if constexpr (kCluster) {
#pragma unroll
                for (int q = 0; q < kMaxCluster; ++q)
                    if (q < ls.ctas) c += ld_cluster_s32(&counts[round][d], q);
            } else {
                c = counts[round][d];
            }
        }
        int total;
        const int above = block_scan(c, warp_sums, &total);
        if (threadIdx.x < kDigits && above < need && above + c >= need) {
            s_digit = d;
            s_left = need - above;
        }
        __syncthreads();
        prefix |= (uint32_t)s_digit << shift;
        need = s_left;
    }
    // `need` of the keys equal to prefix are kept, those of the lowest slots
    int ties = 0;  // of the CTAs before me
    if constexpr (kCluster) {
        for (int q = 0; q < rank; ++q) ties += ld_cluster_s32(&counts[3][prefix & (kDigits - 1)], q);
        cluster_sync();  // nobody reads my counts any more
    }
    int* list = ls.list + r.base;
    const int first_mover = max(begin, a.budget);
    int holes = 0, movers = 0;
    for (int t0 = begin; t0 < live; t0 += kRound) {
        const int t = t0 + tid8;
        Slots8 s;
        uint32_t tie = 0, keep = 0, in = 0;  // bit per slot
        if (t < live) {
            s = load(t);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const uint32_t key = slot_key(s.w[i], s.p[i] >= r.limit);
                if (t + i < live) {
                    in |= 1u << i;
                    if (key > prefix) keep |= 1u << i;
                    if (key == prefix) tie |= 1u << i;
                }
            }
        }
        int total;
        int seen = ties + block_scan(__popc(tie), warp_sums, &total);
        ties += total;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if ((tie >> i) & 1) {
                if (seen < need) keep |= 1u << i;
                ++seen;
            }
        uint32_t hole = 0, mover = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (t + i < a.budget) hole |= in & ~keep & (1u << i);
            else mover |= keep & (1u << i);
        }
        const int at = block_scan(__popc(hole) | (__popc(mover) << 16), warp_sums, &total);
        int h = holes + (at & 0xffff), m = movers + (at >> 16);
        holes += total & 0xffff;
        movers += total >> 16;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if ((hole >> i) & 1) list[begin + h++] = t + i;
            if ((mover >> i) & 1) list[first_mover + m++] = t + i;
            if (t < r.kept && t + i >= r.kept) s.w[i] = 0.0f, s.p[i] = -1;
        }
        // the holes' entries are move_kernel's: what is written to them here comes before
        if (t < live && t < r.kept) store(t, s);
    }
    if (threadIdx.x == 0) ls.counts[(int64_t)row * kMaxCluster + rank] = make_int2(holes, movers);
}

// A warp takes kBatch moves at a time: their slots and rows first, then all the
// 16-byte units of their K and V rows, eight loads of a lane in flight.
constexpr int kMoveThreads = 256;
constexpr int kBatch = 8;
constexpr int kLoads = 8;
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const EvictArgs a, const Lists ls, int units) {
    const int row = blockIdx.x, lane = threadIdx.x & 31;
    pdl_wait();
    const int2* counts = ls.counts + (int64_t)row * kMaxCluster;
    int2 c = lane < ls.ctas ? counts[lane] : make_int2(0, 0);
    const int2 through = make_int2(warp_scan(c.x), warp_scan(c.y));  // up to and with CTA `lane`
    const int moves = __shfl_sync(0xffffffffu, through.x, 31);
    const int b = row / a.kv.nkv, h = row - b * a.kv.nkv;
    const int64_t base = row * a.kv.capacity();
    const int warps = gridDim.y * (kMoveThreads / 32);
    const int size16 = 2 * units;  // 16-byte units of a move: K's, then V's
    const int bytes = units * 16 / a.kv.hd;
    for (int i0 = (blockIdx.y * (kMoveThreads / 32) + (threadIdx.x >> 5)) * kBatch; i0 < moves; i0 += warps * kBatch) {
        const int count = min(kBatch, moves - i0);
        int64_t dst = -1, src = -1;
        const int i = i0 + lane;
        // the CTAs whose lists hold hole i and mover i
        int qh = 0, qm = 0, before_h = 0, before_m = 0;
        for (int q = 0; q < ls.ctas; ++q) {
            const int th = __shfl_sync(0xffffffffu, through.x, q), tm = __shfl_sync(0xffffffffu, through.y, q);
            if (i >= th) qh = q + 1, before_h = th;
            if (i >= tm) qm = q + 1, before_m = tm;
        }
        if (lane < count) {
            const int to = ls.list[base + (int64_t)qh * ls.range + i - before_h];
            const int of = ls.list[base + max(qm * ls.range, a.budget) + i - before_m];
            a.weights_out[base + to] = a.weights[base + of];
            a.positions_out[base + to] = a.positions[base + of];
            dst = a.kv.row(b, h, to);
            src = a.kv.row(b, h, of);
            if (dst < 0 || src < 0) dst = src = -1;  // a slot without a page has no row
        }
        const int all = count * size16;
        for (int u0 = 0; u0 < all; u0 += 32 * kLoads) {
            uint4 v[kLoads];
            char* to[kLoads];
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int u = u0 + j * 32 + lane;
                const int m = u < all ? u / size16 : 0;
                const int64_t d = __shfl_sync(0xffffffffu, dst, m), s = __shfl_sync(0xffffffffu, src, m);
                to[j] = nullptr;
                if (u < all && d >= 0) {
                    int part = u - m * size16;
                    const bool is_v = part >= units;
                    if (is_v) part -= units;
                    char* pool = static_cast<char*>(is_v ? a.kv.v : a.kv.k) + part * 16;
                    v[j] = *reinterpret_cast<const uint4*>(pool + s * bytes);
                    to[j] = pool + d * bytes;
                }
            }
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
                if (to[j]) *reinterpret_cast<uint4*>(to[j]) = v[j];
        }
    }
}

// CTAs per row (a cluster) and their ranges: a round each until the cluster is
// full, more rounds for longer rows.
void divide(const PagedKv& kv, Lists* ls) {
    const int64_t cap = kv.capacity();
    int64_t ctas = (cap + kRound - 1) / kRound;
    if (ctas > kMaxCluster) ctas = kMaxCluster;
    ls->ctas = (int)ctas;
    ls->range = (int)((cap + ctas * kPer - 1) / (ctas * kPer) * kPer);
}

size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

size_t paged_evict_workspace(const PagedKv& kv, int) {
    const size_t rows = (size_t)kv.n_seqs * kv.nkv;
    return aligned(rows * kMaxCluster * sizeof(int2)) + rows * kv.capacity() * sizeof(int);
}

cudaError_t launch_paged_evict(const EvictArgs& a0, void* ws, cudaStream_t st) {
    const int64_t rows = (int64_t)a0.kv.n_seqs * a0.kv.nkv;
    if (rows <= 0) return cudaSuccess;
    if (rows > 65535) return cudaErrorInvalidConfiguration;
    EvictArgs a = a0;
    const int64_t cap = a.kv.capacity();
    if (a.budget > cap) a.budget = (int)cap;  // no sequence is longer
    Lists ls;
    divide(a.kv, &ls);
    ls.counts = static_cast<int2*>(ws);
    ls.list = reinterpret_cast<int*>(static_cast<uint8_t*>(ws) + aligned(rows * kMaxCluster * sizeof(int2)));

    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ls.ctas, (unsigned)rows);
    cfg.blockDim = dim3(kSelectThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ls.ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ls.ctas > 1 ? 1 : 0;
    cudaError_t e = ls.ctas > 1 ? cudaLaunchKernelEx(&cfg, select_kernel<true>, a, ls)
                                : cudaLaunchKernelEx(&cfg, select_kernel<false>, a, ls);
    note_launch();
    if (e != cudaSuccess) return e;

    // enough warps for every move of every row, up to 8 CTAs per SM
    int64_t most = a.budget < cap - a.budget ? a.budget : cap - a.budget;
    const int64_t per_cta = kMoveThreads / 32 * kBatch;
    int64_t y = (most + per_cta - 1) / per_cta;
    const int64_t enough = (148 * 8 + rows - 1) / rows;
    if (y > enough) y = enough;
    if (y < 1) y = 1;
    int units = a.kv.hd * kv_type_size(a.kv.dtype) / 16;
    void* args[] = {&a, &ls, &units};
    return launch_pdl_kernel((const void*)move_kernel, dim3((unsigned)rows, (unsigned)y), dim3(kMoveThreads), 0, st, args);
}

}  // namespace qmm
