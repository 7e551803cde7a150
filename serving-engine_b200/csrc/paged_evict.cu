// paged_evict.cu -- eviction from a paged K/V cache by accumulated attention
// weight (operator API paged_kv_evict).
//
// Per (sequence, kv head): n = min(length, budget) positions stay -- the first
// `sinks`, the last `recent`, and the best scores between them -- and move, in
// order, to positions 0 .. n-1.  The bytes are the scores once, and the kept
// rows read and written (8 D bytes each): HBM bounds it, the choice is latency.
//
// One launch.  A thread-block cluster per (sequence, kv head): each CTA keeps
// its share of the scores in shared memory; the n-th best is found 8 bits of
// its ordered key at a time from histograms that the CTAs add up through
// distributed shared memory; one scan of (better, equal) counts per CTA and
// one exchange of their totals give every kept position its place, ties going
// to the lowest positions.  Then the CTAs move the rows.
//
// Moving in place is safe without a second copy because kept position j comes
// from kept[j] >= j and kept rises: a CTA takes rows in order of j in batches,
// reading a batch whole before it writes it.  Rows that a later batch reads lie
// at or above that batch's own start, where no earlier batch has written.  So
// in place the CTAs of a cluster split the columns of the rows (whole 32-byte
// sectors where a row has them), each taking all rows in order; into other
// blocks they split the rows.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace b2 {

constexpr int kEvThreads = 512;
constexpr int kEvCluster = 8;
constexpr int kEvCached = 16384;  // scores a CTA keeps in shared memory
constexpr int kEvBatch = 4;       // 16-byte pieces in flight per thread

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

__global__ void __launch_bounds__(kEvThreads, 2) evict_kernel(const EvictArgs a) {
    extern __shared__ float s_sc[];
    __shared__ int s_hist[2][256];
    __shared__ int s_sum[256];
    __shared__ int s_pick[2];              // the bin that holds the n-th best, positions above it
    __shared__ int2 s_warp[kEvThreads / 32];
    __shared__ int2 s_total;               // (better, equal) of this CTA
    __shared__ int2 s_before;              // of the CTAs before it
    cg::cluster_group cl = cg::this_cluster();
    const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int kvh = blockIdx.x / cs, b = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int bs = a.kv.block_size;
    griddep_wait();
    const int L = paged_len(a.kv, b), n = min(L, a.budget);
    const int* bt = a.kv.block_tables + (int64_t)b * a.kv.max_blocks;
    int* kept = a.kept + ((int64_t)b * a.nkv + kvh) * a.budget;
    if (kvh == 0 && rank == 0 && t == 0 && a.new_lens != a.kv.seq_lens) a.new_lens[b] = n;

    const bool all = L <= a.budget;
    if (all) {
        for (int j = rank * kEvThreads + t; j < a.budget; j += cs * kEvThreads) kept[j] = j < n ? j : -1;
        if (!a.dst) return;
    } else {
        const int share = (L + cs - 1) / cs, p0 = min(L, rank * share), p1 = min(L, p0 + share);
        const int m0 = a.sinks, m1 = L - a.recent;  // the positions that compete
        auto load = [&](int i) -> float {
            const int blk = bt[(unsigned)i / (unsigned)bs];
            if ((unsigned)blk >= (unsigned)a.kv.num_blocks) return -INFINITY;
            return a.scores[((int64_t)blk * a.nkv + kvh) * bs + (unsigned)i % (unsigned)bs];
        };
        const bool cached = share <= a.cached;
        if (cached) {
#pragma unroll 4
            for (int i = p0 + t; i < p1; i += kEvThreads) s_sc[i - p0] = load(i);
        }
        auto key = [&](int i) { return rank_key(cached ? s_sc[i - p0] : load(i)); };
        const int c0 = max(p0, m0), c1 = min(p1, m1);
        int need = n - a.sinks - a.recent;  // of the competing ones that stay
        uint32_t thr = need > 0 ? 0u : 0xffffffffu;
        if (t < 256) s_hist[0][t] = 0;
        if (need > 0) {  // (the same for the whole cluster)
            for (int pass = 0; pass < 4; ++pass) {
                const int shift = 24 - 8 * pass;
                int* hist = s_hist[pass & 1];
                __syncthreads();
                for (int i0 = c0; i0 < c1; i0 += kEvThreads) {
                    const int i = i0 + t;
                    int bin = -1;
                    if (i < c1) {
                        const uint32_t k = key(i);
                        if (pass == 0 || (k ^ thr) >> (shift + 8) == 0) bin = (k >> shift) & 255;
                    }
                    // equal bins of a warp add once: scores share their exponents
                    const unsigned same = __match_any_sync(~0u, bin);
                    if (bin >= 0 && lane == __ffs(same) - 1) atomicAdd(&hist[bin], __popc(same));
                }
                cl.sync();
                if (t < 256) {
                    int v = 0;
                    for (int r = 0; r < cs; ++r) v += *cl.map_shared_rank(&hist[t], r);
                    s_sum[t] = v;
                    s_hist[(pass + 1) & 1][t] = 0;  // every CTA has read the pass before
                }
                __syncthreads();
                if (warp == 0) {  // lane l: bins 8 l .. 8 l + 7, counted from the top
                    int mine = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) mine += s_sum[lane * 8 + e];
                    int above = mine;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int v = __shfl_down_sync(~0u, above, o);
                        if (lane + o < 32) above += v;
                    }
                    above -= mine;
                    if (above < need && need <= above + mine) {
                        int e = 7;
                        while (above + s_sum[lane * 8 + e] < need) above += s_sum[lane * 8 + e--];
                        s_pick[0] = lane * 8 + e;
                        s_pick[1] = above;
                    }
                }
                __syncthreads();
                thr |= (uint32_t)s_pick[0] << shift;
                need -= s_pick[1];
            }
        }
        // need is now how many positions with key == thr stay.  Every position's place: the better and forced ones
        // before it, and the equal ones before it as far as they stay
        const int q = (share + kEvThreads - 1) / kEvThreads, q0 = min(p1, p0 + t * q), q1 = min(p1, q0 + q);
        auto kind = [&](int i) -> int {  // 1: stays, 2: equal, 0: goes
            if (i < m0 || i >= m1) return 1;
            const uint32_t k = key(i);
            return k > thr ? 1 : k == thr ? 2 : 0;
        };
        int2 mine = make_int2(0, 0);
        for (int i = q0; i < q1; ++i) {
            const int k = kind(i);
            mine.x += k & 1;
            mine.y += k >> 1;
        }
        int2 before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, before.x, o), y = __shfl_up_sync(~0u, before.y, o);
            if (lane >= o) {
                before.x += x;
                before.y += y;
            }
        }
        if (lane == 31) s_warp[warp] = before;
        __syncthreads();
        before.x -= mine.x;
        before.y -= mine.y;
        int2 total = make_int2(0, 0);
#pragma unroll
        for (int w = 0; w < kEvThreads / 32; ++w) {
            if (w < warp) {
                before.x += s_warp[w].x;
                before.y += s_warp[w].y;
            }
            total.x += s_warp[w].x;
            total.y += s_warp[w].y;
        }
        if (t == 0) s_total = total;
        cl.sync();
        if (t == 0) {
            int2 v = make_int2(0, 0);
            for (int r = 0; r < rank; ++r) {
                const int2 x = *cl.map_shared_rank(&s_total, r);
                v.x += x.x;
                v.y += x.y;
            }
            s_before = v;
        }
        __syncthreads();
        before.x += s_before.x;
        before.y += s_before.y;
        for (int i = q0; i < q1; ++i) {
            const int k = kind(i);
            if (k == 1 || (k == 2 && before.y < need)) kept[before.x + min(before.y, need)] = i;
            before.x += k & 1;
            before.y += k >> 1;
        }
        cl.sync();  // the list is whole, every score has been read, and no CTA's shared memory is needed any more
    }

    // ---- move
    const int* dt = a.dst ? a.dst + (int64_t)b * a.dst_blocks : bt;
    const int chunks = a.D / 8;  // 16-byte pieces of a row, K's then V's
    int j0 = 0, j1 = n, first = 0, width = 2 * chunks;
    if (a.dst) {
        const int part = (n + cs - 1) / cs;
        j0 = min(n, rank * part);
        j1 = min(n, j0 + part);
    } else {
        width = (2 * chunks + cs - 1) / cs;
        first = rank * width;
        width = min(width, 2 * chunks - first);
    }
    auto source = [&](int j) { return all ? j : __ldcg(kept + j); };
    if (width > 0) {
        const int rows = kEvThreads / width, r = t / width, piece = first + t - r * width;
        uint4* base = static_cast<uint4*>(piece < chunks ? a.kv.k : a.kv.v);
        const int64_t col = (int64_t)kvh * a.kv.stride_head + (piece < chunks ? piece : piece - chunks) * 8;
        auto at = [&](const int* tab, int pos) -> int64_t {
            const int blk = tab[(unsigned)pos / (unsigned)bs];
            if ((unsigned)blk >= (unsigned)a.kv.num_blocks) return -1;
            return (int64_t)blk * a.kv.stride_block + (int64_t)((unsigned)pos % (unsigned)bs) * a.kv.stride_slot + col;
        };
        for (int jb = j0; jb < j1; jb += rows * kEvBatch) {
            int src[kEvBatch];
            int64_t from[kEvBatch], to[kEvBatch];
            uint4 v[kEvBatch];
#pragma unroll
            for (int e = 0; e < kEvBatch; ++e) {
                const int j = jb + e * rows + r;
                src[e] = r < rows && j < j1 ? source(j) : -1;
            }
#pragma unroll
            for (int e = 0; e < kEvBatch; ++e) {
                const int j = jb + e * rows + r;
                from[e] = -1;
                if (src[e] < 0 || (!a.dst && src[e] == j)) continue;
                from[e] = at(bt, src[e]);
                to[e] = at(dt, j);
                if (to[e] < 0) from[e] = -1;
            }
#pragma unroll
            for (int e = 0; e < kEvBatch; ++e)
                if (from[e] >= 0) v[e] = base[from[e] >> 3];
            if (!a.dst) __syncthreads();
#pragma unroll
            for (int e = 0; e < kEvBatch; ++e)
                if (from[e] >= 0) base[to[e] >> 3] = v[e];
        }
    }
    if (a.dst || rank == 0) {
        auto at = [&](const int* tab, int pos) -> int64_t {
            const int blk = tab[(unsigned)pos / (unsigned)bs];
            if ((unsigned)blk >= (unsigned)a.kv.num_blocks) return -1;
            return ((int64_t)blk * a.nkv + kvh) * bs + (unsigned)pos % (unsigned)bs;
        };
        for (int jb = j0; jb < j1; jb += kEvThreads) {
            const int j = jb + t;
            int64_t from = -1, to = -1;
            float v = 0.f;
            if (j < j1) {
                from = at(bt, source(j));
                to = at(dt, j);
                if (from >= 0) v = a.scores[from];
            }
            if (!a.dst) __syncthreads();
            if (from >= 0 && to >= 0) a.scores[to] = v;
        }
    }
}

// New lengths written over the old ones: only once every cluster has read them.
__global__ void evict_lens_kernel(const EvictArgs a, int batch) {
    griddep_wait();
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b < batch) a.new_lens[b] = min(a.budget, paged_len(a.kv, b));
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
    if (batch > 65535 || nkv > (1 << 24)) return B2_ERR_UNSUPPORTED;
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
    const int cs = kEvCluster;
    const int64_t share = (span + cs - 1) / cs;
    a.cached = (int)(share < kEvCached ? share : kEvCached);
    const size_t smem = (size_t)a.cached * sizeof(float);
    B2_TRY(cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvCached * 4));
    B2_TRY(launch_cluster(evict_kernel, dim3((unsigned)(nkv * cs), batch), dim3(kEvThreads), smem, as_stream(stream),
                          true, cs, a));
    if (new_lens == kv->seq_lens)
        B2_TRY(launch(evict_lens_kernel, dim3((batch + 255) / 256), dim3(256), 0, as_stream(stream), true, a, batch));
    return B2_OK;
}
