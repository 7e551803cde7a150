// paged_evict.cu -- eviction from a paged K/V cache by accumulated attention
// weight (operator API paged_kv_evict).
//
// Per (sequence, kv head): n = min(length, budget) positions stay -- the first
// `sinks`, the last `recent`, and the best scores between them -- and move, in
// order, to positions 0 .. n-1.  The bytes are the scores once (those past the
// 45056 that a CTA keeps in shared memory five times, one table entry and one
// score at a time), and the kept rows read and written (8 D bytes each): HBM
// bounds it, the choice is latency.
//
// The choice is one CTA per (sequence, kv head): the positions' ordered keys
// in shared memory, the n-th best found 11 bits at a time from a histogram,
// then every kept position's place by one scan, ties going to the lowest
// positions.  Latency bounds it: the scores are a small part of the bytes.  (A
// cluster of 8 CTAs per choice, histograms added through distributed shared
// memory, took 20 us a cluster for 4096 scores, this 10: each of its exchanges
// costs more than the reading it saves.)  The move is a second launch spread
// over the GPU, or, where few bytes stay, the choosing CTA's own.  Measured: 16
// x 32768 to 8192 (8 heads of 128, half): 201 us, the move 177 of them at 5.9
// TB/s (92 % of the measured copy); 8 x up to 4096 to 1024: 20 us.  Few long
// sequences leave most SMs idle in the choice: 1 x 32768 to 8192 40 us, 1 x
// 131072 230 (events around single calls, some 4 us above calls in a row).
//
// Moving in place is safe without a second copy because kept position j comes
// from kept[j] >= j and kept rises: a CTA takes rows in order of j in batches,
// reading a batch whole before it writes it.  Rows that a later batch reads lie
// at or above that batch's own start, where no earlier batch has written.  So
// in place the CTAs of a (sequence, kv head) split the columns of the rows
// (whole 32-byte sectors where a row has them), each taking all rows in order;
// into other blocks they split the rows.  In place, timed singly: 16 x
// 32768 to 8192 321 us, 8 x 4096 to 1024 30, 1 x 32768 to 8192 128 (8 CTAs per
// sequence and head, each through all rows with a barrier per batch).
#include "paged.cuh"

namespace b2 {

constexpr int kEvThreads = 1024;   // of a choice
constexpr int kEvCached = 45056;   // keys of a choice kept in shared memory; the rest are read again
constexpr int kMvThreads = 256;    // of a move
constexpr int kMvBatch = 4;        // 16-byte pieces in flight per thread
constexpr int kMvRows = 128;       // rows looked up together; those of a CTA that moves into other blocks
constexpr int kMvSlices = 8;       // column slices in place
constexpr int64_t kFusedBytes = 128 << 10;

struct EvictArgs {
    b2_paged_kv kv;
    float* scores;
    const int* dst;
    int dst_blocks;
    int nkv, D, budget, sinks, recent;
    int* kept;
    int* new_lens;
    BlockDiv div;
    int quads;   // 4 consecutive positions (from a multiple of 4) lie in one block, their scores 16-byte aligned
    int cached;  // keys that the choice's shared memory holds
};

// What positions are ranked by: positions that stay in any case above
// everything, then NaN, then the scores, -0 equal to +0.
constexpr uint32_t kEvStays = 0xffffffffu, kEvNan = 0xfffffffeu;
__device__ __forceinline__ uint32_t rank_key(float f) { return f != f ? kEvNan : float_key(f + 0.f); }

// Moves rows j0 .. j1 - 1 of one (sequence, kv head), pieces first .. first +
// width - 1 of each (16 bytes; K's, then V's), and their scores if `scores`.
// The whole CTA of THREADS calls it.  One thread per row looks up where it
// comes from and goes; the copies then take a few instructions per 16 bytes
// (looking up per copy bounded the kernel by its arithmetic: 5.0 TB/s).
template <int ROWS>
struct MoveLists {
    int64_t from[ROWS], to[ROWS];  // of the rows looked up together, in elements; from -1: nothing to move
};
template <int THREADS, int ROWS>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int kvh, int b, int j0, int j1, int first, int width,
                                          bool scores, MoveLists<ROWS>& list) {
    const int t = threadIdx.x;
    const int* bt = a.kv.block_tables + (int64_t)b * a.kv.max_blocks;
    const int* dt = a.dst ? a.dst + (int64_t)b * a.dst_blocks : bt;
    const int* kept = a.kept + ((int64_t)b * a.nkv + kvh) * a.budget;
    const int chunks = a.D / 8;
    // thread t: piece first + t % width of rows t / width, t / width + rows, ..
    const int rows = width > 0 ? THREADS / width : 0, r = width > 0 ? t / width : 0, piece = first + t - r * width;
    uint4* base = static_cast<uint4*>(piece < chunks ? a.kv.k : a.kv.v) + (piece < chunks ? piece : piece - chunks);
    for (int jb = j0; jb < j1; jb += ROWS) {
        const int m = min(ROWS, j1 - jb);
        int64_t sf = -1, st = -1;
        float sv = 0.f;
        if (t < m) {
            const int j = jb + t, i = __ldcg(kept + j), ib = a.div.block(i), jb2 = a.div.block(j);
            const int sb = bt[ib], db = dt[jb2];
            const bool go = (unsigned)sb < (unsigned)a.kv.num_blocks && (unsigned)db < (unsigned)a.kv.num_blocks &&
                            (a.dst || i != j);
            const int ss = a.div.slot(i, ib), ds = a.div.slot(j, jb2);
            list.from[t] = go ? sb * a.kv.stride_block + ss * a.kv.stride_slot + kvh * a.kv.stride_head : -1;
            list.to[t] = db * a.kv.stride_block + ds * a.kv.stride_slot + kvh * a.kv.stride_head;
            if (go && scores) {
                sf = ((int64_t)sb * a.nkv + kvh) * a.kv.block_size + ss;
                st = ((int64_t)db * a.nkv + kvh) * a.kv.block_size + ds;
                sv = a.scores[sf];
            }
        }
        __syncthreads();  // (in place it also parts the batch's score reads from its writes)
        if (sf >= 0) a.scores[st] = sv;
        for (int k0 = 0; k0 < m; k0 += rows * kMvBatch) {
            if (rows == 0) break;
            int64_t from[kMvBatch];
            uint4 v[kMvBatch];
#pragma unroll
            for (int e = 0; e < kMvBatch; ++e) {
                const int k = k0 + e * rows + r;
                from[e] = r < rows && k < m ? list.from[k] : -1;
                if (from[e] >= 0) v[e] = __ldcs(base + (from[e] >> 3));
            }
            if (!a.dst) __syncthreads();
#pragma unroll
            for (int e = 0; e < kMvBatch; ++e)
                if (from[e] >= 0) __stcs(base + (list.to[k0 + e * rows + r] >> 3), v[e]);
        }
        __syncthreads();
    }
}

// Fills kept for (kvh, b) of a sequence of L positions; the whole CTA of kEvThreads calls it.
__device__ __forceinline__ void choose(const EvictArgs& a, int kvh, int b, int L) {
    extern __shared__ __align__(16) uint32_t s_key[];
    __shared__ int s_hist[2][2048];
    __shared__ int s_pick[2];  // the bin that holds the n-th best, positions above it
    __shared__ int s_sum[kEvThreads / 32];
    __shared__ int2 s_warp[kEvThreads / 32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int bs = a.kv.block_size, n = min(L, a.budget);
    const int* bt = a.kv.block_tables + (int64_t)b * a.kv.max_blocks;
    int* kept = a.kept + ((int64_t)b * a.nkv + kvh) * a.budget;
    if (L <= a.budget) {
        for (int j = t; j < a.budget; j += kEvThreads) kept[j] = j < n ? j : -1;
        return;
    }
    auto load = [&](int i) -> uint32_t {
        if (i < a.sinks || i >= L - a.recent) return kEvStays;
        const int blk = bt[a.div.block(i)];
        if ((unsigned)blk >= (unsigned)a.kv.num_blocks) return rank_key(-INFINITY);
        return rank_key(a.scores[((int64_t)blk * a.nkv + kvh) * bs + a.div.slot(i, a.div.block(i))]);
    };
    const int cached = min(L, a.cached) & ~3;
    s_hist[0][t] = 0;
    s_hist[0][t + kEvThreads] = 0;
    if (a.quads) {
        // 4 consecutive positions of a block at a time, four such per thread on their way
        constexpr int kOn = 4;
        for (int i0 = 4 * t; i0 < cached; i0 += kOn * 4 * kEvThreads) {
            int blk[kOn];
            float4 f[kOn];
#pragma unroll
            for (int e = 0; e < kOn; ++e) {
                const int i = i0 + e * 4 * kEvThreads;
                blk[e] = i < cached ? bt[a.div.block(i)] : -1;
            }
#pragma unroll
            for (int e = 0; e < kOn; ++e) {
                const int i = i0 + e * 4 * kEvThreads;
                f[e] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if ((unsigned)blk[e] < (unsigned)a.kv.num_blocks)
                    f[e] = *reinterpret_cast<const float4*>(a.scores + ((int64_t)blk[e] * a.nkv + kvh) * bs +
                                                            a.div.slot(i, a.div.block(i)));
            }
#pragma unroll
            for (int e = 0; e < kOn; ++e) {
                const int i = i0 + e * 4 * kEvThreads;
                if (i >= cached) continue;
                uint4 k = make_uint4(rank_key(f[e].x), rank_key(f[e].y), rank_key(f[e].z), rank_key(f[e].w));
                if (i < a.sinks || i + 4 > L - a.recent) {
                    auto stays = [&](int x) { return x < a.sinks || x >= L - a.recent; };
                    if (stays(i)) k.x = kEvStays;
                    if (stays(i + 1)) k.y = kEvStays;
                    if (stays(i + 2)) k.z = kEvStays;
                    if (stays(i + 3)) k.w = kEvStays;
                }
                *reinterpret_cast<uint4*>(s_key + i) = k;
            }
        }
    } else {
#pragma unroll 2
        for (int i = t; i < cached; i += kEvThreads) s_key[i] = load(i);
    }
    // keys of positions i .. i + 3 (i a multiple of 4); past the end a key no position of this choice has
    auto keys = [&](int i) -> uint4 {
        if (i < cached) return *reinterpret_cast<const uint4*>(s_key + i);
        return make_uint4(load(i), i + 1 < L ? load(i + 1) : 0u, i + 2 < L ? load(i + 2) : 0u, i + 3 < L ? load(i + 3) : 0u);
    };
    int need = n;
    uint32_t thr = 0;
    for (int pass = 0; pass < 3; ++pass) {  // bits 31 .. 21, 20 .. 10, 9 .. 0
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
        int* hist = s_hist[pass & 1];
        __syncthreads();
        const int up = shift + width;
        auto add = [&](uint32_t k) {
            if (pass == 0 || (k ^ thr) >> up == 0) atomicAdd(&hist[(k >> shift) & ((1 << width) - 1)], 1);
        };
#pragma unroll 2
        for (int i = 4 * t; i < cached; i += 4 * kEvThreads) {
            const uint4 v = *reinterpret_cast<const uint4*>(s_key + i);
            add(v.x);
            add(v.y);
            add(v.z);
            add(v.w);
        }
        for (int i = cached + t; i < L; i += kEvThreads) add(load(i));
        __syncthreads();
        // thread t: bins 2 t and 2 t + 1, counted from the top
        const int2 h = reinterpret_cast<const int2*>(hist)[t];
        int above = h.x + h.y;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_down_sync(~0u, above, o);
            if (lane + o < 32) above += v;
        }
        if (lane == 0) s_sum[warp] = above;
        s_hist[(pass + 1) & 1][t] = 0;
        s_hist[(pass + 1) & 1][t + kEvThreads] = 0;
        __syncthreads();
        int v = s_sum[lane];
        if (lane <= warp) v = 0;
        above += __reduce_add_sync(~0u, v) - h.x - h.y;
        if (above < need && need <= above + h.x + h.y) {
            const bool top = need <= above + h.y;
            s_pick[0] = 2 * t + (top ? 1 : 0);
            s_pick[1] = top ? above : above + h.y;
        }
        __syncthreads();
        thr |= (uint32_t)s_pick[0] << shift;
        need -= s_pick[1];
    }
    // need is now how many positions with key == thr stay.  A position's place: the better ones before it, and the
    // equal ones before it as far as they stay.  A warp takes a stretch of positions, 4 of them a lane at a time.
    const int q = (L + 128 * 32 - 1) / (128 * 32) * 128, q0 = min(L, warp * q), q1 = min(L, q0 + q);
    auto kinds = [&](int i) -> int {  // better ones of the 4 in bits 0 .. 3, equal ones in bits 16 .. 19
        if (i >= q1) return 0;
        const uint4 v = keys(i);
        int r = (v.x > thr) | (v.y > thr) << 1 | (v.z > thr) << 2 | (v.w > thr) << 3 | (v.x == thr) << 16 |
                (v.y == thr) << 17 | (v.z == thr) << 18 | (v.w == thr) << 19;
        if (q1 - i < 4) r &= ((1 << (q1 - i)) - 1) * 0x10001;
        return r;
    };
    auto count = [](int r) { return __popc(r & 0xf) | __popc(r & 0xf0000) << 16; };
    int2 before = make_int2(0, 0);
#pragma unroll 2
    for (int i = q0; i < q1; i += 128) {
        const int c = count(kinds(i + 4 * lane));
        before.x += c & 0xffff;
        before.y += c >> 16;
    }
    before.x = __reduce_add_sync(~0u, before.x);
    before.y = __reduce_add_sync(~0u, before.y);
    if (lane == 0) s_warp[warp] = before;
    __syncthreads();
    before = s_warp[lane];
    if (lane >= warp) before = make_int2(0, 0);
    before.x = __reduce_add_sync(~0u, before.x);
    before.y = __reduce_add_sync(~0u, before.y);
#pragma unroll 2
    for (int i = q0; i < q1; i += 128) {
        const int r = kinds(i + 4 * lane), c = count(r);
        int incl = c;  // at most 128 of each: the halves do not meet
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, incl, o);
            if (lane >= o) incl += v;
        }
        int in = before.x + ((incl - c) & 0xffff), eq = before.y + ((incl - c) >> 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (r >> e & 1) kept[in++ + min(eq, need)] = i + 4 * lane + e;
            if (r >> (16 + e) & 1) {
                if (eq < need) kept[in + eq] = i + 4 * lane + e;
                ++eq;
            }
        }
        incl = __shfl_sync(~0u, incl, 31);
        before.x += incl & 0xffff;
        before.y += incl >> 16;
    }
}

// grid (kv heads, sequences).  FUSED: the CTA moves the rows as well.
template <bool FUSED>
__global__ void __launch_bounds__(kEvThreads, 1) evict_choose_kernel(const EvictArgs a) {
    const int kvh = blockIdx.x, b = blockIdx.y;
    griddep_wait();
    griddep_launch_dependents();
    const int L = paged_len(a.kv, b);
    choose(a, kvh, b, L);
    if constexpr (FUSED) {
        __shared__ MoveLists<kEvThreads> list;
        const int n = min(L, a.budget);
        if (kvh == 0 && threadIdx.x == 0) a.new_lens[b] = n;
        __syncthreads();  // the list is whole
        move_rows<kEvThreads, kEvThreads>(a, kvh, b, 0, n, 0, a.D / 4, true, list);
    }
}

// grid (kv heads; row ranges, or column slices in place; sequences): the heads
// of one range run together, so that their rows' DRAM pages do.
__global__ void __launch_bounds__(kMvThreads, 4) evict_move_kernel(const EvictArgs a) {
    __shared__ MoveLists<kMvRows> list;
    const int kvh = blockIdx.x, b = blockIdx.z, rank = blockIdx.y, parts = gridDim.y, t = threadIdx.x;
    griddep_wait();
    griddep_launch_dependents();
    // (new_lens may be the lengths themselves: the minimum below is the same before and after)
    const int L = paged_len(a.kv, b), n = min(L, a.budget);
    if (kvh == 0 && rank == 0 && t == 0) a.new_lens[b] = n;
    const int pieces = a.D / 4;  // 16-byte pieces of a K and a V row
    int j0 = 0, j1 = n, first = 0, width = pieces;
    bool scores = true;
    if (a.dst) {
        j0 = min(n, rank * kMvRows);
        j1 = min(n, j0 + kMvRows);
    } else {
        width = (pieces + parts - 1) / parts;
        first = min(pieces, rank * width);
        width = min(width, pieces - first);
        scores = rank == 0;
    }
    move_rows<kMvThreads, kMvRows>(a, kvh, b, j0, j1, first, width, scores, list);
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
    a.div = block_div(kv->block_size);
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
    a.cached = (int)(span < kEvCached ? (span + 3) & ~int64_t(3) : kEvCached);
    const int64_t rows = budget < span ? budget : span;
    const int64_t parts = dst_tables ? (rows + kMvRows - 1) / kMvRows : kMvSlices;
    if (parts > 65535) return B2_ERR_UNSUPPORTED;
    a.quads = kv->block_size % 4 == 0 && aligned16(scores);
    cudaStream_t s = as_stream(stream);
    const size_t smem = (size_t)a.cached * sizeof(uint32_t);
    // One launch or two, by the bytes a (sequence, kv head) keeps.  At 64 KB (256 rows of 64, 2 heads) one launch takes
    // 8.5 us on the device and 3.9 on the host, two take 7.9 and 6.3; at 128 KB 9.9 against 8.5 for 2 pairs, but 11.6
    // against 14.4 for 128; at 256 KB (512 rows of 128, 8 pairs) 12.7 against 8.9.  Lengths written over the old ones
    // need the second launch: other heads' CTAs still read them.
    if (rows * 4 * D <= kFusedBytes && new_lens != kv->seq_lens) {
        static bool fused[64];
        B2_TRY(allow_smem(evict_choose_kernel<true>, kEvCached * 4, fused));
        B2_TRY(launch(evict_choose_kernel<true>, dim3(nkv, batch), dim3(kEvThreads), smem, s, true, a));
        return B2_OK;
    }
    static bool done[64];
    B2_TRY(allow_smem(evict_choose_kernel<false>, kEvCached * 4, done));
    B2_TRY(launch(evict_choose_kernel<false>, dim3(nkv, batch), dim3(kEvThreads), smem, s, true, a));
    B2_TRY(launch(evict_move_kernel, dim3(nkv, (unsigned)parts, batch), dim3(kMvThreads), 0, s, true, a));
    return B2_OK;
}
