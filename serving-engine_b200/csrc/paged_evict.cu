// paged_evict.cu -- eviction from a paged K/V cache by accumulated attention
// weight (operator API paged_kv_evict).
//
// Per (sequence, kv head): n = min(length, budget) positions stay -- the first
// `sinks`, the last `recent`, and the best scores between them -- and move, in
// order, to positions 0 .. n-1.  The bytes are the scores once, and the kept
// rows read and written (8 D bytes each): HBM bounds it, the choice is latency.
//
// Two launches.  The choice is one CTA per (sequence, kv head): its scores in
// shared memory, the n-th best found 8 bits of its ordered key at a time from
// a histogram, then every kept position's place from ballots and one scan, ties
// going to the lowest positions.  (A cluster of 8 CTAs per choice, histograms
// added through distributed shared memory, took 20 us a cluster for 4096
// scores: each of its exchanges costs more than the reading it saves.)
// The move is spread over the GPU.
//
// Moving in place is safe without a second copy because kept position j comes
// from kept[j] >= j and kept rises: a CTA takes rows in order of j in batches,
// reading a batch whole before it writes it.  Rows that a later batch reads lie
// at or above that batch's own start, where no earlier batch has written.  So
// in place the CTAs of a (sequence, kv head) split the columns of the rows
// (whole 32-byte sectors where a row has them), each taking all rows in order;
// into other blocks they split the rows.
#include "paged.cuh"

namespace b2 {

constexpr int kEvThreads = 1024;   // of a choice
constexpr int kEvCached = 49152;   // scores of a choice kept in shared memory; the rest are read again
constexpr int kMvThreads = 256;    // of a move
constexpr int kMvBatch = 4;        // 16-byte pieces in flight per thread
constexpr int kMvRows = 128;       // rows of a CTA that moves into other blocks
constexpr int kMvSlices = 8;       // column slices in place

struct EvictArgs {
    b2_paged_kv kv;
    float* scores;
    const int* dst;
    int dst_blocks;
    int nkv, D, budget, sinks, recent;
    int* kept;
    int* new_lens;
    int cached;  // floats of shared memory for scores
};

// The order scores are ranked in, as unsigned keys: NaN above everything,
// -0 equal to +0.
__device__ __forceinline__ uint32_t rank_key(float f) {
    if (f != f) return 0xffffffffu;
    return float_key(f + 0.f);
}

__global__ void __launch_bounds__(kEvThreads, 1) evict_choose_kernel(const EvictArgs a) {
    extern __shared__ float s_sc[];
    __shared__ int s_hist[2][256];
    __shared__ int s_pick[2];  // the bin that holds the n-th best, positions above it
    __shared__ int2 s_warp[kEvThreads / 32];
    const int kvh = blockIdx.x, b = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int bs = a.kv.block_size;
    griddep_wait();
    griddep_launch_dependents();
    const int L = paged_len(a.kv, b), n = min(L, a.budget);
    const int* bt = a.kv.block_tables + (int64_t)b * a.kv.max_blocks;
    int* kept = a.kept + ((int64_t)b * a.nkv + kvh) * a.budget;
    if (L <= a.budget) {
        for (int j = t; j < a.budget; j += kEvThreads) kept[j] = j < n ? j : -1;
        return;
    }
    const int m0 = a.sinks, m1 = L - a.recent;  // the positions that compete
    auto load = [&](int i) -> float {
        const int blk = bt[(unsigned)i / (unsigned)bs];
        if ((unsigned)blk >= (unsigned)a.kv.num_blocks) return -INFINITY;
        return a.scores[((int64_t)blk * a.nkv + kvh) * bs + (unsigned)i % (unsigned)bs];
    };
    const int cached = min(L, a.cached);
    if (t < 256) s_hist[0][t] = 0;
#pragma unroll 8
    for (int i = t; i < cached; i += kEvThreads) s_sc[i] = load(i);
    auto key = [&](int i) { return rank_key(i < cached ? s_sc[i] : load(i)); };
    int need = n - a.sinks - a.recent;  // of the competing ones that stay
    uint32_t thr = need > 0 ? 0u : 0xffffffffu;
    if (need > 0) {
        for (int pass = 0; pass < 4; ++pass) {
            const int shift = 24 - 8 * pass;
            int* hist = s_hist[pass & 1];
            __syncthreads();
            for (int i = m0 + t; i < m1; i += kEvThreads) {
                const uint32_t k = key(i);
                if (pass == 0 || (k ^ thr) >> (shift + 8) == 0) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (warp == 0) {  // lane l: bins 8 l .. 8 l + 7, counted from the top
                int h[8], mine = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[e] = hist[lane * 8 + e];
                    mine += h[e];
                }
                int above = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_down_sync(~0u, above, o);
                    if (lane + o < 32) above += v;
                }
                above -= mine;
#pragma unroll
                for (int e = 7; e >= 0; --e) {
                    if (above < need && need <= above + h[e]) {
                        s_pick[0] = lane * 8 + e;
                        s_pick[1] = above;
                    }
                    above += h[e];
                }
            } else if (warp <= 8) {
                s_hist[(pass + 1) & 1][t - 32] = 0;
            }
            __syncthreads();
            thr |= (uint32_t)s_pick[0] << shift;
            need -= s_pick[1];
        }
    }
    __syncthreads();
    // need is now how many positions with key == thr stay.  A position's place: the forced and better ones before
    // it, and the equal ones before it as far as they stay.  A warp takes a stretch of positions, 32 at a time.
    const int q = ((L + kEvThreads - 1) / kEvThreads) * 32, q0 = min(L, warp * q), q1 = min(L, q0 + q);
    auto kind = [&](int i) -> int {  // 1: stays, 2: equal, 0: goes
        if (i >= q1) return 0;
        if (i < m0 || i >= m1) return 1;
        const uint32_t k = key(i);
        return k > thr ? 1 : k == thr ? 2 : 0;
    };
    int2 before = make_int2(0, 0);
    for (int i = q0; i < q1; i += 32) {
        const int k = kind(i + lane);
        before.x += __popc(__ballot_sync(~0u, k == 1));
        before.y += __popc(__ballot_sync(~0u, k == 2));
    }
    if (lane == 0) s_warp[warp] = before;
    __syncthreads();
    before = s_warp[lane];
    if (lane >= warp) before = make_int2(0, 0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before.x += __shfl_xor_sync(~0u, before.x, o);
        before.y += __shfl_xor_sync(~0u, before.y, o);
    }
    const unsigned under = (1u << lane) - 1;
    for (int i = q0; i < q1; i += 32) {
        const int k = kind(i + lane);
        const unsigned in = __ballot_sync(~0u, k == 1), eq = __ballot_sync(~0u, k == 2);
        const int e = before.y + __popc(eq & under);
        if (k == 1 || (k == 2 && e < need)) kept[before.x + __popc(in & under) + min(e, need)] = i + lane;
        before.x += __popc(in);
        before.y += __popc(eq);
    }
}

// grid (row ranges, or column slices in place; kv heads; sequences)
__global__ void __launch_bounds__(kMvThreads, 4) evict_move_kernel(const EvictArgs a) {
    const int kvh = blockIdx.y, b = blockIdx.z, rank = blockIdx.x, cs = gridDim.x, t = threadIdx.x;
    const int bs = a.kv.block_size;
    griddep_wait();
    griddep_launch_dependents();
    // (new_lens may be the lengths themselves: the minimum below is the same before and after)
    const int L = paged_len(a.kv, b), n = min(L, a.budget);
    if (kvh == 0 && rank == 0 && t == 0) a.new_lens[b] = n;
    const int* bt = a.kv.block_tables + (int64_t)b * a.kv.max_blocks;
    const int* kept = a.kept + ((int64_t)b * a.nkv + kvh) * a.budget;
    const int* dt = a.dst ? a.dst + (int64_t)b * a.dst_blocks : bt;
    const int chunks = a.D / 8;  // 16-byte pieces of a row, K's then V's
    int j0 = 0, j1 = n, first = 0, width = 2 * chunks;
    if (a.dst) {
        j0 = min(n, rank * kMvRows);
        j1 = min(n, j0 + kMvRows);
    } else {
        width = (2 * chunks + cs - 1) / cs;
        first = rank * width;
        width = min(width, 2 * chunks - first);
    }
    
    if (width > 0) {
        const int rows = kMvThreads / width, r = t / width, piece = first + t - r * width;
        uint4* base = static_cast<uint4*>(piece < chunks ? a.kv.k : a.kv.v);
        const int64_t col = (int64_t)kvh * a.kv.stride_head + (piece < chunks ? piece : piece - chunks) * 8;
        auto at = [&](const int* tab, int pos) -> int64_t {
            const int blk = tab[(unsigned)pos / (unsigned)bs];
            if ((unsigned)blk >= (unsigned)a.kv.num_blocks) return -1;
            return (int64_t)blk * a.kv.stride_block + (int64_t)((unsigned)pos % (unsigned)bs) * a.kv.stride_slot + col;
        };
        for (int jb = j0; jb < j1; jb += rows * kMvBatch) {
            int src[kMvBatch];
            int64_t from[kMvBatch], to[kMvBatch];
            uint4 v[kMvBatch];
#pragma unroll
            for (int e = 0; e < kMvBatch; ++e) {
                const int j = jb + e * rows + r;
                src[e] = r < rows && j < j1 ? __ldcg(kept + j) : -1;
            }
#pragma unroll
            for (int e = 0; e < kMvBatch; ++e) {
                const int j = jb + e * rows + r;
                from[e] = -1;
                if (src[e] < 0 || (!a.dst && src[e] == j)) continue;
                from[e] = at(bt, src[e]);
                to[e] = at(dt, j);
                if (to[e] < 0) from[e] = -1;
            }
#pragma unroll
            for (int e = 0; e < kMvBatch; ++e)
                if (from[e] >= 0) v[e] = base[from[e] >> 3];
            if (!a.dst) __syncthreads();
#pragma unroll
            for (int e = 0; e < kMvBatch; ++e)
                if (from[e] >= 0) base[to[e] >> 3] = v[e];
        }
    }
    if (a.dst || rank == 0) {
        auto at = [&](const int* tab, int pos) -> int64_t {
            const int blk = tab[(unsigned)pos / (unsigned)bs];
            if ((unsigned)blk >= (unsigned)a.kv.num_blocks) return -1;
            return ((int64_t)blk * a.nkv + kvh) * bs + (unsigned)pos % (unsigned)bs;
        };
        for (int jb = j0; jb < j1; jb += kMvThreads) {
            const int j = jb + t;
            int64_t from = -1, to = -1;
            float v = 0.f;
            if (j < j1) {
                from = at(bt, __ldcg(kept + j));
                to = at(dt, j);
                if (from >= 0) v = a.scores[from];
            }
            if (!a.dst) __syncthreads();
            if (from >= 0 && to >= 0) a.scores[to] = v;
        }
    }
}

}  // namespace b2

extern "C" int b2_paged_kv_evict(const b2_paged_kv* kv, float* scores, const int* dst_tables, int max_dst_blocks,
                                 int batch, int nkv, int D, int budget, int sinks, int recent, int* kept,
                                 int* new_lens, void* stream) {
    using namespace b2;
    if (batch <= 0) return B2_OK;
    B2_REQUIRE(kv && scores && kept && new_lens && budget > 0 && sinks >= 0 && recent >= 0 &&
               (int64_t)sinks + recent <= budget);
    const int rc = check_paged(kv, nkv, D);
    if (rc != B2_OK) return rc;
    B2_REQUIRE(!dst_tables || (int64_t)max_dst_blocks * kv->block_size >= budget);
    if (batch > 65535 || nkv > 65535) return B2_ERR_UNSUPPORTED;
    EvictArgs a = {};
    a.kv = *kv;
    a.scores = scores;
    a.dst = dst_tables;
    a.dst_blocks = max_dst_blocks;
    a.nkv = nkv;
    a.D = D;
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    a.kept = kept;
    a.new_lens = new_lens;
    const int64_t span = (int64_t)kv->max_blocks * kv->block_size;
    a.cached = (int)(span < kEvCached ? span : kEvCached);
    cudaStream_t s = as_stream(stream);
    B2_TRY(cudaFuncSetAttribute(evict_choose_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvCached * 4));
    B2_TRY(launch(evict_choose_kernel, dim3(nkv, batch), dim3(kEvThreads), (size_t)a.cached * sizeof(float), s, true, a));
    const int64_t parts = dst_tables ? ((int64_t)budget + kMvRows - 1) / kMvRows : kMvSlices;
    B2_TRY(launch(evict_move_kernel, dim3((unsigned)parts, nkv, batch), dim3(kMvThreads), 0, s, true, a));
    return B2_OK;
}
