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
constexpr int kPer = 8;                        // consecutive slots of a thread in a round
constexpr int kRound = kSelectThreads * kPer;  // slots a CTA takes in a round
constexpr int kMaxCluster = 8;                 // the portable size
constexpr int kDigits = 256;
constexpr int kCopies = 8;  // of a histogram: neighbouring lanes count in different ones

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
    int2* counts;  // [rows][ctas]: holes, movers
    int rows;
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
// other's counts through distributed shared memory. kHeld: a CTA's range is one
// round, whose slots stay in registers; longer ranges are read again (from L1 and
// L2) each time.
template <bool kCluster, bool kHeld>
__global__ void __launch_bounds__(kSelectThreads) select_kernel(const EvictArgs a, const Lists ls) {
    __shared__ __align__(16) int hist[2][kCopies][kDigits + 4];  // of this round and the next
    __shared__ __align__(16) int counts[4][kDigits];             // of this CTA, per digit round
    __shared__ int warp_sums[32];
    __shared__ int s_digit, s_left;
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.y, rank = kCluster ? (int)blockIdx.x : 0;
    const int64_t cap = a.kv.capacity(), base = row * cap;
    const int begin = rank * ls.range, end = (int)min((int64_t)begin + ls.range, cap);
    const float* w = a.weights + base;
    const int* pos = a.positions + base;
    float* w_out = a.weights_out + base;
    int* pos_out = a.positions_out + base;
    const int tid8 = threadIdx.x * kPer, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

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
    Slots8 held = {};
    if (kHeld && begin + tid8 < end) held = load(begin + tid8);  // beside the loads of row_of
    auto slots = [&](int t) { return kHeld ? held : load(t); };
    for (int i = threadIdx.x; i < kCopies * (kDigits + 4); i += kSelectThreads) (&hist[0][0][0])[i] = 0;

    const Row r = row_of(a, row);
    const int live = min(end, r.n);  // slots of mine that are cached: [begin, live)
    if (rank == 0 && row % a.kv.nkv == 0 && threadIdx.x == 0) a.lengths_out[row / a.kv.nkv] = r.kept;
    // what lies beyond the kept slots, and all of a row that is short enough
    const bool full = r.n > a.budget;
    for (int t = begin + tid8; t < end; t += kRound) {
        if (full && t < r.kept) continue;
        Slots8 s = {};
        if (t < r.kept) s = slots(t);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (t + i >= r.kept) s.w[i] = 0.0f, s.p[i] = -1;
        store(t, s);
    }
    int2* my_counts = ls.counts + (int64_t)row * ls.ctas + rank;
    if (!full) {
        if (threadIdx.x == 0) *my_counts = make_int2(0, 0);
        return;
    }
    __syncthreads();

    uint32_t prefix = 0;
    int need = a.budget;  // slots still to take among those that match the prefix
#pragma unroll 1
    for (int round = 0; round < 4; ++round) {
        const int shift = 24 - 8 * round;
        int* mine = hist[round & 1][threadIdx.x & (kCopies - 1)];
        for (int t = begin + tid8; t < live; t += kRound) {
            const Slots8 s = slots(t);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const uint32_t key = slot_key(s.w[i], s.p[i] >= r.limit);
                if (t + i < live && (round == 0 || ((key ^ prefix) >> (shift + 8)) == 0))
                    atomicAdd(&mine[(key >> shift) & (kDigits - 1)], 1);
            }
        }
        __syncthreads();
        if constexpr (kCluster) {
            if (threadIdx.x < kDigits) {
                int c = 0;
#pragma unroll
                for (int i = 0; i < kCopies; ++i) c += hist[round & 1][i][threadIdx.x];
                counts[round][threadIdx.x] = c;
            }
            cluster_sync();
        }
        // the first warp finds the digit (lane l has digits 255 - 8 l down), the others clear for the next round
        if (warp == 0) {
            int c[8] = {};
            const int d0 = kDigits - 8 - 8 * lane;
            if constexpr (kCluster) {
                for (int q = 0; q < ls.ctas; ++q)
#pragma unroll
                    for (int i = 0; i < 8; ++i) c[i] += ld_cluster_s32(&counts[round][d0 + i], q);
            } else {
#pragma unroll
                for (int q = 0; q < kCopies; ++q) {
                    const int4 lo = *reinterpret_cast<const int4*>(&hist[round & 1][q][d0]);
                    const int4 hi = *reinterpret_cast<const int4*>(&hist[round & 1][q][d0 + 4]);
                    c[0] += lo.x, c[1] += lo.y, c[2] += lo.z, c[3] += lo.w;
                    c[4] += hi.x, c[5] += hi.y, c[6] += hi.z, c[7] += hi.w;
                }
            }
            int sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += c[i];
            int above = warp_scan(sum) - sum;
            if (above < need && above + sum >= need) {  // one lane
                int d = 7;
#pragma unroll
                for (int i = 7; i >= 0; --i)
                    if (d == i && above + c[i] < need) above += c[i], d = i - 1;
                s_digit = d0 + d;
                s_left = need - above;
            }
        } else {
            for (int i = threadIdx.x - 32; i < kCopies * (kDigits + 4); i += kSelectThreads - 32)
                (&hist[(round + 1) & 1][0][0])[i] = 0;
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
    int* list = ls.list + base;
    const int first_mover = max(begin, a.budget);
    int holes = 0, movers = 0;
    for (int t0 = begin; t0 < live; t0 += kRound) {
        const int t = t0 + tid8;
        Slots8 s = {};
        uint32_t tie = 0, keep = 0, in = 0;  // bit per slot
        if (t < live) {
            s = slots(t);
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
    if (threadIdx.x == 0) *my_counts = make_int2(holes, movers);
}

// The moves of all rows are dealt out in batches, warp by warp: a lane finds the
// slots and rows of a move, then all lanes copy the 16-byte units of the batch's K
// and V rows, eight loads of a lane in flight. The chain of loads before the copy
// is paid once a batch, so there are no more batches than warps as long as a
// batch is at most 32 moves (with batches of four, 16 sequences of 1500 to 8192
// slots, 8 kv heads of 128, took 51 us instead of 23).
constexpr int kMoveThreads = 256;
constexpr int kMoveCtas = 3;  // per SM: one wave
// kSteps: 16-byte units of a move (its K row, then its V row) per lane.
template <int kSteps>
__global__ void __launch_bounds__(kMoveThreads, kMoveCtas) move_kernel(const EvictArgs a, const Lists ls, int units) {
    constexpr int kMoves = 8 / kSteps;  // with their loads in flight together
    const int lane = threadIdx.x & 31;
    const int64_t cap = a.kv.capacity();
    pdl_launch_dependents();
    pdl_wait();
    // each lane adds up a run of rows
    const int per = (ls.rows + 31) / 32, r0 = lane * per, r1 = min(ls.rows, r0 + per);
    auto holes_of = [&](int row) {
        int n = 0;
        for (int q = 0; q < ls.ctas; ++q) n += ls.counts[(int64_t)row * ls.ctas + q].x;
        return n;
    };
    const int64_t warps = (int64_t)gridDim.x * (kMoveThreads / 32);
    int64_t mine = 0;
    for (int row = r0; row < r1; ++row) mine += holes_of(row);
    int64_t all_moves = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all_moves += __shfl_xor_sync(0xffffffffu, all_moves, o);
    // of a batch: rows end with part of one, and a second batch for some warps would double the time
    const int64_t deal = warps > 2 * ls.rows ? warps - ls.rows : warps;
    const int size = (int)max((int64_t)1, min((all_moves + deal - 1) / deal, (int64_t)32));
    mine = 0;
    for (int row = r0; row < r1; ++row) mine += (holes_of(row) + size - 1) / size;
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    const int64_t batches = __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    const int bytes = units * 16 / a.kv.hd;  // of an element
    char* unit_at[kSteps];                    // this lane's units of row 0; null: none
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int u = lane + 32 * i;
        unit_at[i] = u < units ? static_cast<char*>(a.kv.k) + u * 16
                               : (u < 2 * units ? static_cast<char*>(a.kv.v) + (u - units) * 16 : nullptr);
    }
    for (int64_t k = (int64_t)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); k < batches; k += warps) {
        const int owner = __ffs(__ballot_sync(0xffffffffu, k >= before && k < before + mine)) - 1;
        int64_t batch = k - __shfl_sync(0xffffffffu, before, owner);
        int row = owner * per, moves = holes_of(row);
        while (batch >= (moves + size - 1) / size) {
            batch -= (moves + size - 1) / size;
            moves = holes_of(++row);
        }
        const int count = min(size, moves - (int)batch * size);
        const int b = row / a.kv.nkv, h = row - b * a.kv.nkv;
        const int64_t base = row * cap;
        int64_t dst = -1, src = -1;
        if (lane < count) {
            const int i = (int)batch * size + lane;
            // the CTAs whose lists hold hole i and mover i
            int hole = 0, mover = 0, holes = 0, movers = 0;
            for (int q = 0; q < ls.ctas; ++q) {
                const int2 c = ls.counts[(int64_t)row * ls.ctas + q];
                if (i >= holes && i < holes + c.x) hole = q * ls.range + i - holes;
                if (i >= movers && i < movers + c.y) mover = max(q * ls.range, a.budget) + i - movers;
                holes += c.x;
                movers += c.y;
            }
            const int to = ls.list[base + hole], of = ls.list[base + mover];
            a.weights_out[base + to] = a.weights[base + of];
            a.positions_out[base + to] = a.positions[base + of];
            dst = a.kv.row(b, h, to);
            src = a.kv.row(b, h, of);
            if (dst < 0 || src < 0) dst = src = -1;  // a slot without a page has no row
        }
        for (int m0 = 0; m0 < count; m0 += kMoves) {
            uint4 v[kMoves][kSteps];
#pragma unroll
            for (int m = 0; m < kMoves; ++m) {
                const int64_t from = __shfl_sync(0xffffffffu, src, (m0 + m) & 31) * bytes;
                if (m0 + m < count && from >= 0)
#pragma unroll
                    for (int i = 0; i < kSteps; ++i)
                        if (unit_at[i]) v[m][i] = *reinterpret_cast<const uint4*>(unit_at[i] + from);
            }
#pragma unroll
            for (int m = 0; m < kMoves; ++m) {
                const int64_t to = __shfl_sync(0xffffffffu, dst, (m0 + m) & 31) * bytes;
                if (m0 + m < count && to >= 0)
#pragma unroll
                    for (int i = 0; i < kSteps; ++i)
                        if (unit_at[i]) *reinterpret_cast<uint4*>(unit_at[i] + to) = v[m][i];
            }
        }
    }
}

// CTAs per row (a cluster) and their ranges: a round each until the cluster is
// full, more rounds for longer rows. Shorter ranges pay more in cluster barriers and
// remote counts than they save in loads: with ranges of 4096 and 2048 slots 4 rows of
// 4161 take 16.8 and 18.8 us for 14.7, 128 rows of up to 8192 69 and 115 us for 53, a
// row of 32768 39.8 us for 30.6 (both launches).
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
    ls.rows = (int)rows;
    ls.counts = static_cast<int2*>(ws);
    ls.list = reinterpret_cast<int*>(static_cast<uint8_t*>(ws) + aligned(rows * kMaxCluster * sizeof(int2)));

    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ls.ctas, (unsigned)rows);
    cfg.blockDim = dim3(kSelectThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ls.ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ls.ctas > 1 ? 2 : 1;
    cudaError_t e;
    if (ls.ctas == 1) e = cudaLaunchKernelEx(&cfg, select_kernel<false, true>, a, ls);
    else if (ls.range <= kRound) e = cudaLaunchKernelEx(&cfg, select_kernel<true, true>, a, ls);
    else e = cudaLaunchKernelEx(&cfg, select_kernel<true, false>, a, ls);
    note_launch();
    if (e != cudaSuccess) return e;

    // a warp for every move there can be, one wave at most
    const int64_t most = rows * (a.budget < cap - a.budget ? a.budget : cap - a.budget) + 1;
    int64_t grid = (most + kMoveThreads / 32 - 1) / (kMoveThreads / 32);
    const int64_t wave = (int64_t)paged_sm_count() * kMoveCtas;
    if (grid > wave) grid = wave;
    int units = a.kv.hd * kv_type_size(a.kv.dtype) / 16;
    void* args[] = {&a, &ls, &units};
    const void* fn[] = {(const void*)move_kernel<1>, (const void*)move_kernel<2>, (const void*)move_kernel<4>,
                        (const void*)move_kernel<4>};
    return launch_pdl_kernel(fn[(2 * units + 31) / 32 - 1], dim3((unsigned)grid), dim3(kMoveThreads), 0, st, args);
}

}  // namespace qmm
