// paged.cuh -- argument checks and element access shared by the operators on a
// caller's paged K/V cache (paged_attn.cu, paged_evict.cu).
#pragma once

#include "common.cuh"

namespace b2 {

// Host checks of a cache description: no device access.
inline int check_paged(const b2_paged_kv* kv, int nkv, int D) {
    if (!kv || !kv->k || !kv->v || !kv->block_tables || !kv->seq_lens || kv->num_blocks <= 0 || kv->block_size <= 0 ||
        kv->max_blocks <= 0 || nkv <= 0 || D <= 0)
        return B2_ERR_INVALID;
    if (D > 256 || (D & 7) || (int64_t)kv->max_blocks * kv->block_size > (1 << 30) || !aligned16(kv->k) ||
        !aligned16(kv->v) || (kv->stride_block & 7) || (kv->stride_slot & 7) || (kv->stride_head & 7))
        return B2_ERR_UNSUPPORTED;
    return B2_OK;
}

// Division of positions (below 2^30) by the block size: one wide multiply
// instead of a divide.  m = floor(2^(30 + s) / d) + 1 with 2^s >= d gives
// floor(x / d) for every x < 2^30: the excess x (m d - 2^(30+s)) / (d 2^(30+s))
// is below 2^30 d / (d 2^(30+s)) <= 1 / d.
struct BlockDiv {
    uint32_t m;
    int shift, d;
    __device__ __forceinline__ int block(int pos) const { return (int)(((uint64_t)(uint32_t)pos * m) >> shift); }
    __device__ __forceinline__ int slot(int pos, int block) const { return pos - block * d; }
};
inline BlockDiv block_div(int d) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    return BlockDiv{(uint32_t)((1ull << (30 + s)) / (unsigned)d + 1), 30 + s, d};
}

// Length of sequence b, cut to what its table row can hold.
__device__ __forceinline__ int paged_len(const b2_paged_kv& kv, int b) {
    return max(0, min(kv.seq_lens[b], kv.max_blocks * kv.block_size));
}

}  // namespace b2
