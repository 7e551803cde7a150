// paged_evict.cu -- eviction from a paged K/V cache by accumulated attention
// weight (operator API paged_kv_evict).
//
// Per (sequence, kv head): n = min(length, budget) positions stay -- the first
// `sinks`, the last `recent`, and the best scores between them -- and move, in
// order, to positions 0 .. n-1.  Kept position j comes from kept[j] >= j, so
// moving rows in order of j never overwrites a row that is still to be read.
#include "paged.cuh"

namespace b2 {

struct EvictArgs {
    b2_paged_kv kv;
    float* scores;
    const int* dst;
    int dst_blocks;
    int nkv, D, budget, sinks, recent;
    int* kept;
    int* new_lens;
};

// The order scores are ranked in, as unsigned keys: NaN above everything,
// -0 equal to +0.
__device__ __forceinline__ uint32_t rank_key(float f) {
    if (f != f) return 0xffffffffu;
    return float_key(f + 0.f);
}

// One CTA per (kv head, sequence).  The threshold key -- the n-th best of the
// positions that compete -- one bit at a time, then the kept positions in
// order by a running count.
__global__ void __launch_bounds__(1024) evict_simple_select(const EvictArgs a) {
    __shared__ float redf[32];
    __shared__ int cnt[32];
    griddep_wait();
    const int kvh = blockIdx.x, b = blockIdx.y, bs = a.kv.block_size, t = threadIdx.x;
    const int lane = t & 31, warp = t >> 5;
    const int L = paged_len(a.kv, b);
    const int* bt = a.kv.block_tables + (int64_t)b * a.kv.max_blocks;
    int* kept = a.kept + ((int64_t)b * a.nkv + kvh) * a.budget;
    const int n = min(L, a.budget);
    for (int j = t; j < a.budget; j += 1024) kept[j] = j < n && L <= a.budget ? j : -1;
    if (L <= a.budget) return;
    const int m0 = a.sinks, m1 = L - a.recent, need = n - a.sinks - a.recent;
    auto key = [&](int i) -> uint32_t {
        const int blk = bt[i / bs];
        if (blk < 0 || blk >= a.kv.num_blocks) return 0;
        return rank_key(a.scores[((int64_t)blk * a.nkv + kvh) * bs + i % bs]);
    };
    auto count = [&](uint32_t thr) -> int {  // positions of the middle with key >= thr
        float c = 0.f;
        for (int i = m0 + t; i < m1; i += 1024) c += key(i) >= thr ? 1.f : 0.f;
        return (int)block_sum(c, redf);
    };
    uint32_t thr = 0;
    for (int bit = 31; bit >= 0; --bit)
        if (count(thr | (1u << bit)) >= need) thr |= 1u << bit;
    const int above = thr == 0xffffffffu ? 0 : count(thr + 1);
    int ties = need - above, base = 0;  // ties still to give out, kept so far
    for (int i0 = 0; i0 < L; i0 += 1024) {
        const int i = i0 + t;
        const uint32_t k = i < L && i >= m0 && i < m1 ? key(i) : 0;
        const bool mid = i >= m0 && i < m1;
        // tie rank inside this stretch
        const unsigned eq = __ballot_sync(~0u, mid && k == thr);
        __syncthreads();
        if (lane == 0) cnt[warp] = __popc(eq);
        __syncthreads();
        int before = __popc(eq & ((1u << lane) - 1)), tot = 0;
        for (int w = 0; w < 32; ++w) {
            before += w < warp ? cnt[w] : 0;
            tot += cnt[w];
        }
        const bool keep = i < L && (!mid || k > thr || (k == thr && before < ties));
        ties = max(0, ties - tot);
        const unsigned kb = __ballot_sync(~0u, keep);
        __syncthreads();
        if (lane == 0) cnt[warp] = __popc(kb);
        __syncthreads();
        int at = base + __popc(kb & ((1u << lane) - 1)), all = 0;
        for (int w = 0; w < 32; ++w) {
            at += w < warp ? cnt[w] : 0;
            all += cnt[w];
        }
        base += all;
        if (keep) kept[at] = i;
    }
}

// One CTA per (kv head, sequence) moves the kept rows one after another.
__global__ void __launch_bounds__(128) evict_simple_move(const EvictArgs a) {
    griddep_wait();
    const int kvh = blockIdx.x, b = blockIdx.y, bs = a.kv.block_size, t = threadIdx.x;
    const int n = min(a.budget, paged_len(a.kv, b));
    const int* bt = a.kv.block_tables + (int64_t)b * a.kv.max_blocks;
    const int* dt = a.dst ? a.dst + (int64_t)b * a.dst_blocks : bt;
    const int* kept = a.kept + ((int64_t)b * a.nkv + kvh) * a.budget;
    uint16_t *K = static_cast<uint16_t*>(a.kv.k), *V = static_cast<uint16_t*>(a.kv.v);
    for (int j = 0; j < n; ++j) {
        const int i = kept[j], sb = bt[i / bs], db = dt[j / bs];
        if (sb < 0 || sb >= a.kv.num_blocks || db < 0 || db >= a.kv.num_blocks) continue;
        const int64_t s = sb * a.kv.stride_block + (i % bs) * a.kv.stride_slot + kvh * a.kv.stride_head;
        const int64_t d = db * a.kv.stride_block + (j % bs) * a.kv.stride_slot + kvh * a.kv.stride_head;
        for (int e = t; e < a.D; e += 128) {
            K[d + e] = K[s + e];
            V[d + e] = V[s + e];
        }
        if (t == 0) a.scores[((int64_t)db * a.nkv + kvh) * bs + j % bs] = a.scores[((int64_t)sb * a.nkv + kvh) * bs + i % bs];
    }
    if (kvh == 0 && t == 0) a.new_lens[b] = n;
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
    B2_TRY(launch(evict_simple_select, dim3(nkv, batch), dim3(1024), 0, as_stream(stream), true, a));
    B2_TRY(launch(evict_simple_move, dim3(nkv, batch), dim3(128), 0, as_stream(stream), true, a));
    return B2_OK;
}
