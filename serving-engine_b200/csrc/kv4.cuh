// kv4.cuh -- the paged K/V cache of 4-bit rows: its layout and host checks.
//
// A row (K or V of one token and kv head) is held in groups of 64 channels,
// each as m + u s with codes u in 0 .. 15 and halves s, m: 72 bytes for 128
// channels.  16 consecutive positions of a kv head are a tile, K and V together
// and contiguous, in the order in which the lanes of a warp use them as
// fragments of m16n8k16 products (lane l, r = l / 4, c = l % 4), so that a tile
// is copied in one piece and read in whole words:
//   K codes  row p at p DP / 2.  Word j (channels 8 j .. 8 j + 7, channel 8 j +
//            e at bits 4 e) stands at (j % 4) (DP / 32) + j / 4: lane (r, c)
//            reads DP / 32 words of rows r and r + 8, word i of channels 32 i.
//   V codes  at 8 DP.  16 bits hold channels 32 x + 4 r + i (i at bits 4 i) of a
//            position; lane (r, c) reads 8 bytes per x, positions 2 c, 2 c + 1,
//            2 c + 8 and 2 c + 9.
//   scales   K's at 16 DP, V's 64 NG further: (s, m) of group g of position p
//            at (slot(p) NG + g) 4, slot in the order above, so that lane (r,
//            c) reads those of its four positions as one run.
// Blocks are [kv head][block_size / 16][tile].  Channels head_dim .. DP - 1 are
// padding: code 0.
#pragma once

#include "paged.cuh"

namespace b2 {

constexpr int kv4_dp(int D) { return D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256; }
constexpr int kv4_groups(int DP) { return (DP + 63) / 64; }
constexpr int kv4_tile(int DP) { return 16 * DP + 128 * kv4_groups(DP); }
// Place of position p of a tile among the scales.
__host__ __device__ constexpr int kv4_slot(int p) { return (p & 7) / 2 * 4 + p / 8 * 2 + (p & 1); }

// Host checks of a cache description: no device access.
inline int check_paged4(const b2_paged_kv4* kv, int nkv, int D) {
    if (!kv || !kv->pool || !kv->block_tables || !kv->seq_lens || kv->num_blocks <= 0 || kv->block_size <= 0 ||
        kv->max_blocks <= 0 || nkv <= 0 || D <= 0)
        return B2_ERR_INVALID;
    if (D > 256 || (D & 7) || (kv->block_size & 15) || (int64_t)kv->max_blocks * kv->block_size > (1 << 30) ||
        !aligned16(kv->pool) || (kv->stride_block & 15))
        return B2_ERR_UNSUPPORTED;
    const int64_t block = (int64_t)nkv * (kv->block_size / 16) * kv4_tile(kv4_dp(D));
    if (kv->num_blocks > 1 && kv->stride_block < block) return B2_ERR_INVALID;  // blocks would overlap
    return B2_OK;
}

}  // namespace b2
