// block_select.cu -- which blocks of a long paged cache a new token looks at
// (operator API paged_block_bounds and paged_block_select).
//
// Bounds.  For each block and kv head, lo_d <= k_d <= hi_d over the keys that
// the block holds, in 8 bits: whole multiples of one power of two per (block,
// head), the least that 127 multiples of cover the largest |k|, lo rounded down
// and hi up.  The bytes are the keys once; a CTA takes a (block, kv head), its
// warps every fourth row or group of rows, a lane 8 channels.
//
// Choice.  No query head h of a group has a logit above sum_d max(q_hd lo_d,
// q_hd hi_d) in a block.  Summed over the group's heads that is
//   score = sum_d hi_d P_d + lo_d N_d,  P_d, N_d = sums of the positive and of
//   the negative q_hd,
// one product of 2 D terms for any number of heads.  P and N are rounded to 16
// bits (one power of two for all), so that the sum is one of whole numbers,
// exact in 32 bits whatever its order (256 * 2 * 127 * 32767 < 2^31), and blocks
// rank the same in every implementation: as two products of bytes, P and N
// being 256 times their upper byte and their lower one.  The sum as a 32-bit
// float times the block's power of two is what blocks are ranked by.  A block
// that holds a NaN or an infinity ranks first, so that it shows.
//
// The bytes are 2 D + 4 per (block, kv head).  Scores go to the workspace; a
// second launch, a CTA per (sequence, kv head), finds the n-th best by its
// ordered key, 11 bits of the range still open at a time until 32 are left, and
// lists what is above it and the first of those equal to it, in order.  (In one
// launch, the last CTA of each pair choosing and every CTA working out P and N:
// 54 us for 32 x 2048 blocks of 8 heads of 128, instead of 27 and 7.)
//
// Measured, cold: bounds of 32768 tokens of 8 heads of 128 in 16 bits 15 us (4.5
// TB/s: a block's loads leave together, 112 KB per SM, then its warp works them off
// before it looks up the next one), of the newest block of 8 sequences 6.3 us, a chain of three loads; scores of 32 x up to
// 2048 blocks of 8 heads 28 us (117 MB, 4.3 TB/s with its start), of 4094 blocks
// 11 us, five loads one after the other; the choice among 2048 blocks 6.6 us (8.5
// of 256 pairs), among 8188 9.5 us (14 us with 512 threads and keys in shared
// memory): its barriers, six and five a further 11 bits, and the keys' atomics.
#include <cmath>

#include "kv4.cuh"
#include "mma.cuh"
#include "workspace.cuh"

namespace b2 {

// ---------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------

constexpr int kBdWarps = 4;
constexpr int kBdThreads = 32 * kBdWarps;

struct BoundsArgs {
    const uint16_t* k;    // 16-bit rows, or
    const uint8_t* pool;  // 4-bit ones
    int64_t stride_block, stride_slot, stride_head;  // elements; 4-bit: block bytes, -, head bytes
    const int *block_tables, *seq_lens, *newest;
    int num_blocks, block_size, max_blocks, batch, nkv, D, bf16;
    int8_t* codes;
    float* scale;
};

// The smaller, or a NaN if one is.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The same, and the larger, of two 16-bit numbers each.
template <bool BF16>
__device__ __forceinline__ uint32_t least2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (BF16)
        asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
        asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t most2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (BF16)
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

template <bool KV4, bool BF16>
__global__ void __launch_bounds__(kBdThreads, 7) bounds_kernel(const BoundsArgs a) {
    __shared__ __align__(16) float s_lo[kBdWarps - 1][256], s_hi[kBdWarps - 1][256];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
    griddep_wait();
    griddep_launch_dependents();
    // a lane has 8 channels, 8, 16 or 32 lanes a row
    const int DP = kv4_dp(a.D), NG = kv4_groups(DP), wide = DP == 64 ? 3 : DP <= 128 ? 4 : 5;
    const int sub = lane >> wide, own_c = (lane & ((1 << wide) - 1)) * 8;
    const bool in = own_c < a.D;
    const int c = in ? own_c : 0;  // (lanes past the row read its first channels and keep them to themselves)
    int base = 0;  // blocks of the sequences before b0
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
        // every warp by itself: lane b for the blocks that sequence b0 + b's newest positions lie in
        int n = 0, len = 0;
        if (b0 + lane < a.batch) {
            len = max(0, min(a.seq_lens[b0 + lane], a.max_blocks * a.block_size));
            const int since = a.newest ? len - max(0, min(len, a.newest[b0 + lane])) : 0;
            if (since < len) n = (len - 1) / a.block_size - since / a.block_size + 1;
        }
        int end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, end, o);
            if (lane >= o) end += v;
        }
        // more blocks than CTAs: a warp for each, else all warps of a CTA together
        const int all = __shfl_sync(~0u, end, 31), team = all > (int)gridDim.x ? 1 : kBdWarps;
        const int grid = (int)gridDim.x * (kBdWarps / team), own = team == 1 ? warp : 0;
        const int r0 = (team == 1 ? 0 : warp * (32 >> wide)) + sub, step = team * (32 >> wide);
        int i = (int)blockIdx.x + own * (int)gridDim.x;
        if (i < base) i += (base - i + grid - 1) / grid * grid;
        for (; i < base + all; i += grid) {
            const int b = __ffs(__ballot_sync(~0u, end > i - base)) - 1;
            const int from_end = __shfl_sync(~0u, end, b) - 1 - (i - base), L = __shfl_sync(~0u, len, b);
            const int blk = (L - 1) / a.block_size - from_end, rows = min(a.block_size, L - blk * a.block_size);
            const int id = a.block_tables[(int64_t)(b0 + b) * a.max_blocks + blk];
            if ((unsigned)id >= (unsigned)a.num_blocks) continue;
            float lo[8], hi[8];
            constexpr int ON = 8;  // rows on their way
            if constexpr (KV4) {
#pragma unroll
                for (int e = 0; e < 8; ++e) lo[e] = INFINITY, hi[e] = -INFINITY;
                const uint8_t* at = a.pool + (int64_t)id * a.stride_block + h * a.stride_head;
                const int j = c >> 3, word = ((j & 3) * (DP / 32) + (j >> 2)) * 4, meta = 16 * DP + (c >> 6) * 4;
                for (int r = 0; r < rows; r += ON * step) {
                    uint32_t w[ON], m[ON];
#pragma unroll
                    for (int k = 0; k < ON; ++k) {
                        const int rr = min(r + r0 + k * step, rows - 1);  // (the last row once more changes nothing)
                        const uint8_t* tile = at + (int64_t)(rr >> 4) * kv4_tile(DP);
                        w[k] = *reinterpret_cast<const uint32_t*>(tile + (rr & 15) * (DP / 2) + word);
                        m[k] = *reinterpret_cast<const uint32_t*>(tile + meta + kv4_slot(rr & 15) * NG * 4);
                    }
#pragma unroll
                    for (int k = 0; k < ON; ++k) {
                        const float2 sm = h2_to_f2(m[k]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float f = fmaf((float)((w[k] >> (4 * e)) & 15), sm.x, sm.y);
                            lo[e] = min_nan(lo[e], f);
                            hi[e] = max_nan(hi[e], f);
                        }
                    }
                }
            } else {
                // (of 16-bit numbers the least and the largest are such numbers: two at a time, a NaN staying one)
                uint32_t l[4], u[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) l[e] = BF16 ? 0x7f807f80u : 0x7c007c00u, u[e] = l[e] | 0x80008000u;
                const uint16_t* const at = a.k + (int64_t)id * a.stride_block + (int64_t)h * a.stride_head + c;
                for (int r = 0; r < rows; r += ON * step) {
                    uint4 w[ON];
#pragma unroll
                    for (int k = 0; k < ON; ++k)  // (the last row once more changes nothing)
                        w[k] = *reinterpret_cast<const uint4*>(at + min(r + r0 + k * step, rows - 1) * a.stride_slot);
#pragma unroll
                    for (int k = 0; k < ON; ++k) {
                        const uint32_t x[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) l[e] = least2<BF16>(l[e], x[e]), u[e] = most2<BF16>(u[e], x[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = BF16 ? make_float2(__uint_as_float(l[e] << 16), __uint_as_float(l[e] & 0xffff0000u)) : h2_to_f2(l[e]);
                    const float2 y = BF16 ? make_float2(__uint_as_float(u[e] << 16), __uint_as_float(u[e] & 0xffff0000u)) : h2_to_f2(u[e]);
                    lo[2 * e] = x.x, lo[2 * e + 1] = x.y;
                    hi[2 * e] = y.x, hi[2 * e + 1] = y.y;
                }
            }
            for (int o = 1 << wide; o < 32; o <<= 1)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    lo[e] = min_nan(lo[e], __shfl_xor_sync(~0u, lo[e], o));
                    hi[e] = max_nan(hi[e], __shfl_xor_sync(~0u, hi[e], o));
                }
            if (team > 1) {  // the first warp goes on alone
                if (warp > 0 && sub == 0 && in) {
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        *reinterpret_cast<float4*>(&s_lo[warp - 1][c + e]) = make_float4(lo[e], lo[e + 1], lo[e + 2], lo[e + 3]);
                        *reinterpret_cast<float4*>(&s_hi[warp - 1][c + e]) = make_float4(hi[e], hi[e + 1], hi[e + 2], hi[e + 3]);
                    }
                }
                __syncthreads();
                if (warp == 0 && in) {
#pragma unroll
                    for (int v = 0; v < kBdWarps - 1; ++v)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            lo[e] = min_nan(lo[e], s_lo[v][c + e]);
                            hi[e] = max_nan(hi[e], s_hi[v][c + e]);
                        }
                }
                __syncthreads();
                if (warp > 0) continue;
            }
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = in ? max_nan(top, max_nan(fabsf(lo[e]), fabsf(hi[e]))) : top;
            for (int o = 1; o < (1 << wide); o <<= 1) top = max_nan(top, __shfl_xor_sync(~0u, top, o));
            const bool fine = top < INFINITY;
            // the least e with top <= 127 * 2^e: top is f 2^x with f from 1 to 2, 127 is 127/64 2^6
            const uint32_t bits = __float_as_uint(top);
            const int e = top == 0.f ? 0 : max(-126, (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) > 0x7e0000u ? 5 : 6));
            if (sub == 0 && in) {
                const float back = fine ? pow2(-e) : 0.f;
                // (a product that vanishes still is on its side of zero)
                uint32_t d[2] = {0, 0}, u[2] = {0, 0};
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float x = lo[k], y = hi[k];
                    const int dn = fine ? (int)fminf(floorf(x * back), x < 0.f ? -1.f : 127.f) : 0;
                    const int up = fine ? (int)fmaxf(ceilf(y * back), y > 0.f ? 1.f : -127.f) : 0;
                    d[k / 4] |= (uint32_t)(dn & 255) << (8 * (k & 3));
                    u[k / 4] |= (uint32_t)(up & 255) << (8 * (k & 3));
                }
                int8_t* out = a.codes + ((int64_t)id * a.nkv + h) * 2 * a.D + c;
                *reinterpret_cast<uint2*>(out) = make_uint2(d[0], d[1]);
                *reinterpret_cast<uint2*>(out + a.D) = make_uint2(u[0], u[1]);
                if (lane == 0) a.scale[(int64_t)id * a.nkv + h] = fine ? pow2(e) : INFINITY;
            }
        }
        base += all;
    }
}

static int bounds_launch(const BoundsArgs& a, bool kv4, cudaStream_t s) {
    // the blocks of a head are dealt out in turn to as many CTAs as fill the GPU once
    const int64_t most = (int64_t)a.batch * a.max_blocks;
    int64_t grid = 7 * sm_count() / a.nkv;
    grid = grid < 1 ? 1 : grid > most ? most : grid;
    const dim3 g((unsigned)grid, (unsigned)a.nkv);
    if (kv4)
        B2_TRY(launch(bounds_kernel<true, false>, g, dim3(kBdThreads), 0, s, true, a));
    else if (a.bf16)
        B2_TRY(launch(bounds_kernel<false, true>, g, dim3(kBdThreads), 0, s, true, a));
    else
        B2_TRY(launch(bounds_kernel<false, false>, g, dim3(kBdThreads), 0, s, true, a));
    return B2_OK;
}

// ---------------------------------------------------------------------------
// choice
// ---------------------------------------------------------------------------

constexpr int kScThreads = 256;  // of the scores
constexpr int kScWarps = kScThreads / 32;
constexpr int kSlKeys = 8;  // keys that a thread keeps
constexpr int kSlBins = 2048;
constexpr uint32_t kSlStays = 0xffffffffu;  // blocks that are chosen in any case

struct SelectArgs {
    const void* q;
    int64_t ldq;
    const int *block_tables, *seq_lens;
    int num_blocks, block_size, max_blocks;
    const int8_t* codes;
    const float* scale;
    int* out;
    int nq, nkv, D, group, bf16, n, first, last;
    int chunk, heads, team;  // blocks and kv heads per CTA of the scores, warps per head
    uint32_t* keys;          // [batch][nkv][max_blocks]
};

__device__ __forceinline__ int dp4_su(uint32_t s, uint32_t u, int c) {
    int d;
    asm("dp4a.s32.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(s), "r"(u), "r"(c));
    return d;
}
__device__ __forceinline__ int dp4_ss(uint32_t s, uint32_t u, int c) {
    int d;
    asm("dp4a.s32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(s), "r"(u), "r"(c));
    return d;
}

// P: 16-byte pieces of a bounds row (2 D bytes) that each of 4 lanes takes.
// A warp has the bounds of one kv head (a team of warps where there are fewer
// than 8): P and N are worked out by every warp for itself, without a barrier,
// while the first bounds are on their way.
template <int P>
__global__ void __launch_bounds__(kScThreads, 2) score_kernel(const SelectArgs a) {
    __shared__ __align__(16) uint8_t s_q[kScWarps][2][512];  // upper and lower bytes of N, P
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.z, h = blockIdx.y * a.heads + warp / a.team;
    griddep_wait();
    griddep_launch_dependents();
    const int len = max(0, min(a.seq_lens[b], a.max_blocks * a.block_size));
    const int nb = (len + a.block_size - 1) / a.block_size;
    const int c0 = blockIdx.x * a.chunk, c1 = min(nb, c0 + a.chunk);
    if (nb <= a.n || c0 >= nb || warp / a.team >= a.heads || h >= a.nkv) return;  // (a warp's own business: no barrier here)
    constexpr int ON = P <= 4 ? 2 : 1;  // blocks of a lane at a time
    const int part = lane & 3, pieces = a.D / 8, step = 8 * a.team, first = c0 + (warp % a.team) * 8 + (lane >> 2);
    const int* bt = a.block_tables + (int64_t)b * a.max_blocks;
    // (where there is no block, or no piece, the first one's is read and comes to nothing)
    int shift[P];
#pragma unroll
    for (int p = 0; p < P; ++p) shift[p] = part + 4 * p < pieces ? part + 4 * p : 0;
    const uint4* const codes = reinterpret_cast<const uint4*>(a.codes) + (int64_t)h * pieces;
    const float* const scales = a.scale + h;
    uint4 w[ON][P];
    float sc[ON];
    int id[ON];        // of the blocks that are fetched next
    bool there[ON], next[ON];
    auto look = [&](int j0) {
#pragma unroll
        for (int n = 0; n < ON; ++n) id[n] = j0 + n * step < c1 ? bt[j0 + n * step] : -1;
    };
    auto fetch = [&]() {
#pragma unroll
        for (int n = 0; n < ON; ++n) {
            next[n] = (unsigned)id[n] < (unsigned)a.num_blocks;
            const int64_t row = (next[n] ? id[n] : 0) * (int64_t)a.nkv;
            const uint4* src = codes + row * pieces;
#pragma unroll
            for (int p = 0; p < P; ++p) w[n][p] = src[shift[p]];
            sc[n] = scales[row];
        }
    };
    look(first);
    fetch();
    look(first + ON * step);

    // ---- P and N in 16 bits: N first, as lo stands before hi
    constexpr int CH = P;  // channels of a lane: D <= 32 P
    double neg[CH], pos[CH];
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.ldq + (int64_t)h * a.group * a.D;
#pragma unroll
    for (int k = 0; k < CH; ++k) neg[k] = pos[k] = 0.0;
#pragma unroll 4
    for (int g = 0; g < a.group; ++g)
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const int c = k * 32 + lane;
            if (c < a.D) {
                const uint32_t u = q[(int64_t)g * a.D + c];
                const float f = a.bf16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half((uint16_t)u));
                pos[k] += f <= 0.f ? 0.0 : (double)f;  // (a NaN to both)
                neg[k] += f >= 0.f ? 0.0 : (double)f;
            }
        }
    // the largest of them by its bits, which rank like the numbers (a NaN above all)
    unsigned long long big = 0;
    auto bits = [](double y) { return (unsigned long long)__double_as_longlong(y) & ~(1ull << 63); };
#pragma unroll
    for (int k = 0; k < CH; ++k) big = max(big, max(bits(neg[k]), bits(pos[k])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(~0u, big, o));
    const bool fine = big < 0x7ff0000000000000ull;
    // the least e with it <= 32767 * 2^e: it is f 2^x with f from 1 to 2, 32767 is 32767/16384 2^14 (doubles of sums of
    // halves and bf16 are normal, or zero)
    const int x = (int)(big >> 52) - 1023, e = x - ((big & 0xfffffffffffffull) > 0xfffc000000000ull ? 13 : 14);
    const double back = fine && big ? __longlong_as_double((long long)(1023 - e) << 52) : 0.0;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        const int c = k * 32 + lane;
        if (c < a.D) {
            const int n = fine ? __double2int_rn(neg[k] * back) : 0, p = fine ? __double2int_rn(pos[k] * back) : 0;
            s_q[warp][0][c] = (uint8_t)(n >> 8), s_q[warp][1][c] = (uint8_t)n;
            s_q[warp][0][a.D + c] = (uint8_t)(p >> 8), s_q[warp][1][a.D + c] = (uint8_t)p;
        }
    }
    __syncwarp();

    // ---- scores, 4 lanes a block
    uint32_t* keys = a.keys + ((int64_t)b * a.nkv + h) * a.max_blocks;
    uint4 qh[P], ql[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int at = part + 4 * p;
        qh[p] = at < pieces ? *reinterpret_cast<const uint4*>(s_q[warp][0] + 16 * at) : make_uint4(0, 0, 0, 0);
        ql[p] = at < pieces ? *reinterpret_cast<const uint4*>(s_q[warp][1] + 16 * at) : make_uint4(0, 0, 0, 0);
    }
    for (int j0 = first; j0 - (lane >> 2) < c1; j0 += ON * step) {
        int sum[ON];
        float s[ON];
#pragma unroll
        for (int n = 0; n < ON; ++n) there[n] = next[n];
#pragma unroll
        for (int n = 0; n < ON; ++n) {
            int hi = 0, lo = 0;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                hi = dp4_ss(w[n][p].x, qh[p].x, hi), lo = dp4_su(w[n][p].x, ql[p].x, lo);
                hi = dp4_ss(w[n][p].y, qh[p].y, hi), lo = dp4_su(w[n][p].y, ql[p].y, lo);
                hi = dp4_ss(w[n][p].z, qh[p].z, hi), lo = dp4_su(w[n][p].z, ql[p].z, lo);
                hi = dp4_ss(w[n][p].w, qh[p].w, hi), lo = dp4_su(w[n][p].w, ql[p].w, lo);
            }
            sum[n] = hi * 256 + lo;
            s[n] = sc[n];
        }
        fetch();
        look(j0 + 2 * ON * step);
#pragma unroll
        for (int n = 0; n < ON; ++n) {
            sum[n] += __shfl_xor_sync(~0u, sum[n], 1);
            sum[n] += __shfl_xor_sync(~0u, sum[n], 2);
            const int j = j0 + n * step;
            if (part == 0 && j < c1) {
                const float score = s[n] == INFINITY ? INFINITY : (float)sum[n] * s[n];
                // (a NaN, as of a scale never written, ranks first but is not one of the blocks that stay)
                keys[j] = j < a.first || j >= nb - a.last ? kSlStays
                                                          : there[n] ? min(float_key(score + 0.f), kSlStays - 2) : 0u;
            }
        }
    }
}

// One CTA per (sequence, kv head).  Keys stay in registers (up to 8 of a thread;
// of longer sequences they are read again from the workspace).
template <int THREADS>
__global__ void __launch_bounds__(THREADS) choose_kernel(const SelectArgs a) {
    constexpr int WARPS = THREADS / 32;
    __shared__ uint32_t s_few32[32];
    __shared__ int s_hist[kSlBins];
    __shared__ int s_sum[WARPS];
    __shared__ uint32_t s_count[kSlKeys][WARPS];  // keys above the border, and equal to it << 16
    __shared__ int s_bin, s_above, s_in, s_few;
    __shared__ uint32_t s_range[2][WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.x, b = blockIdx.y;
    constexpr int PER = kSlBins / THREADS;
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < PER; ++i) s_hist[i * THREADS + tid] = 0;
    };
    clear();
    if (tid == 0) s_bin = s_above = s_in = s_few = 0;
    griddep_wait();
    griddep_launch_dependents();
    const int len = max(0, min(a.seq_lens[b], a.max_blocks * a.block_size));
    const int nb = (len + a.block_size - 1) / a.block_size;
    const int64_t pair = (int64_t)b * a.nkv + h;
    int* out = a.out + pair * a.n;
    if (nb <= a.n) {  // every block
        for (int i = tid; i < a.n; i += THREADS) out[i] = i < nb ? i : -1;
        return;
    }
    const uint32_t* keys = a.keys + pair * a.max_blocks;
    constexpr int ROUND = kSlKeys * THREADS;  // keys at a time
    uint32_t key[kSlKeys];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int j = 0; j < kSlKeys; ++j) {
            const int i = i0 + j * THREADS + tid;
            key[j] = i < nb ? __ldcg(keys + i) : kSlStays;  // (what stays is left out of the ranking)
        }
    };
    // f(key) for all of this thread's
    auto each = [&](auto f) {
        for (int i0 = 0; i0 < nb; i0 += ROUND) {
            if (nb > ROUND) fetch(i0);
#pragma unroll
            for (int j = 0; j < kSlKeys; ++j)
                if (i0 + j * THREADS < nb) f(key[j]);
        }
    };
    if (nb <= ROUND) fetch(0);
    uint32_t lowest = ~0u, highest = 0u;
    each([&](uint32_t k) {
        if (k != kSlStays) lowest = min(lowest, k), highest = max(highest, k);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lowest = min(lowest, __shfl_xor_sync(~0u, lowest, o));
        highest = max(highest, __shfl_xor_sync(~0u, highest, o));
    }
    if (lane == 0) s_range[0][warp] = lowest, s_range[1][warp] = highest;
    __syncthreads();
    lowest = s_range[0][lane % WARPS], highest = s_range[1][lane % WARPS];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lowest = min(lowest, __shfl_xor_sync(~0u, lowest, o));
        highest = max(highest, __shfl_xor_sync(~0u, highest, o));
    }
    // want: how many of the keys lowest .. highest are chosen; all above are
    int want = a.n - a.first - a.last;
    while (want > 0 && lowest < highest) {
        const uint32_t range = highest - lowest;
        const int shift = max(0, 21 - __clz(range));  // range >> shift below 2048
        each([&](uint32_t k) {
            k -= lowest;
            if (k <= range) atomicAdd(&s_hist[k >> shift], 1);
        });
        __syncthreads();
        // the bin of the want-th best: thread t sums the bins PER t' .. PER t' + PER - 1, t' counting from the top
        const int top_bin = kSlBins - 1 - tid * PER;
        int mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine += s_hist[top_bin - i];
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        int before = lane < warp ? s_sum[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(~0u, before, o);
        incl += before;
        if (incl >= want && incl - mine < want) {
            int above = incl - mine, bin = top_bin;
            while (above + s_hist[bin] < want) above += s_hist[bin--];
            s_bin = bin;
            s_above = above;
            s_in = s_hist[bin];
            s_few = 0;
        }
        __syncthreads();
        want -= s_above;
        lowest += (uint32_t)s_bin << shift;
        highest = lowest + min(highest - lowest, (1u << shift) - 1);  // (the end of a bin near the top is past 32 bits)
        clear();
        const int in = s_in;
        if (in <= 32 && lowest < highest) {  // few enough to be ranked side by side in every warp
            each([&](uint32_t k) {
                if (k - lowest <= highest - lowest) {
                    const int at = atomicAdd(&s_few, 1);
                    if (at < 32) s_few32[at] = k;  // (more only if the keys change under way: a workspace used twice at once)
                }
            });
            __syncthreads();
            const uint32_t k = lane < in ? s_few32[lane] : 0u;
            int more = 0, same = 0;  // candidates above this lane's, and equal to it
            for (int i = 0; i < in; ++i) {
                const uint32_t o = __shfl_sync(~0u, k, i);
                more += o > k;
                same += o == k;
            }
            const int who = __ffs(__ballot_sync(~0u, lane < in && more < want && more + same >= want)) - 1;
            lowest = highest = __shfl_sync(~0u, k, who);
            want -= __shfl_sync(~0u, more, who);
        }
        __syncthreads();
    }
    // ---- what is above, and the first `want` that equal it, in order (want 0: nothing below the blocks that stay)
    const uint32_t border = want > 0 ? lowest : kSlStays - 1;
    const uint32_t below = (1u << lane) - 1;
    int above = 0, equal = 0;  // before the keys of this round
    for (int i0 = 0; i0 < nb; i0 += ROUND) {
        if (nb > ROUND) {
            fetch(i0);
            __syncthreads();
        }
        const int rows = min(kSlKeys, (nb - i0 + THREADS - 1) / THREADS);
#pragma unroll
        for (int j = 0; j < kSlKeys; ++j) {
            if (j >= rows) break;
            const bool there = i0 + j * THREADS + tid < nb;
            const uint32_t up = __ballot_sync(~0u, there && key[j] > border), eq = __ballot_sync(~0u, there && key[j] == border);
            if (lane == 0) s_count[j][warp] = __popc(up) | __popc(eq) << 16;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kSlKeys; ++j) {
            if (j >= rows) break;
            const int i = i0 + j * THREADS + tid;
            const bool there = i < nb, over = there && key[j] > border, same = there && key[j] == border;
            const uint32_t up = __ballot_sync(~0u, over), eq = __ballot_sync(~0u, same);
            uint32_t sum = lane < WARPS ? s_count[j][lane] : 0u;  // of warps 0 .. lane
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(~0u, sum, o);
                if (lane >= o) sum += v;
            }
            const uint32_t all = __shfl_sync(~0u, sum, 31), prior = __shfl_sync(~0u, sum, warp - 1 & 31);
            const uint32_t before = warp > 0 ? prior : 0u;
            const int e = equal + (int)(before >> 16) + __popc(eq & below);
            const int at = above + (int)(before & 0xffffu) + __popc(up & below) + min(e, want);
            if ((over || (same && e < want)) && at < a.n) out[at] = i;
            above += (int)(all & 0xffffu);
            equal += (int)(all >> 16);
        }
    }
}

template <int P>
static int select_launch(const SelectArgs& a, int batch, cudaStream_t s) {
    const dim3 grid((unsigned)((a.max_blocks + a.chunk - 1) / a.chunk), (unsigned)((a.nkv + a.heads - 1) / a.heads), (unsigned)batch);
    B2_TRY(launch(score_kernel<P>, grid, dim3(kScThreads), 0, s, true, a));
    // as many threads as keep all keys in registers (2048 blocks of 256 pairs: 8.5 us with 512, 11 with 1024, 8.9 with 256;
    // 4094 blocks of 8 pairs: 7.4 with 512, 7.5 with 1024)
    const dim3 pairs((unsigned)a.nkv, (unsigned)batch);
    if (a.max_blocks <= 512 * kSlKeys)
        B2_TRY(launch(choose_kernel<512>, pairs, dim3(512), 0, s, true, a));
    else
        B2_TRY(launch(choose_kernel<1024>, pairs, dim3(1024), 0, s, true, a));
    return B2_OK;
}

}  // namespace b2

static int bounds_check(const void* codes, const void* scale, int batch, int nkv, int max_blocks) {
    B2_REQUIRE(codes && scale);
    if (!b2::aligned16(codes)) return B2_ERR_UNSUPPORTED;
    // blocks of all sequences are counted in 32 bits
    if ((int64_t)batch * max_blocks > (1ll << 30) || nkv > 65535) return B2_ERR_UNSUPPORTED;
    return B2_OK;
}

extern "C" int b2_paged_block_bounds(const b2_paged_kv* kv, const int* newest, void* codes, float* scale, int batch,
                                     int nkv, int D, void* stream) {
    using namespace b2;
    if (batch <= 0) return B2_OK;
    int rc = check_paged(kv, nkv, D);
    if (rc == B2_OK) rc = bounds_check(codes, scale, batch, nkv, kv->max_blocks);
    if (rc != B2_OK) return rc;
    BoundsArgs a = {};
    a.k = static_cast<const uint16_t*>(kv->k);
    a.stride_block = kv->stride_block;
    a.stride_slot = kv->stride_slot;
    a.stride_head = kv->stride_head;
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.newest = newest;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.batch = batch;
    a.nkv = nkv;
    a.D = D;
    a.bf16 = kv->bf16;
    a.codes = static_cast<int8_t*>(codes);
    a.scale = scale;
    return bounds_launch(a, false, as_stream(stream));
}

extern "C" int b2_paged_kv4_block_bounds(const b2_paged_kv4* kv, const int* newest, void* codes, float* scale,
                                         int batch, int nkv, int D, void* stream) {
    using namespace b2;
    if (batch <= 0) return B2_OK;
    int rc = check_paged4(kv, nkv, D);
    if (rc == B2_OK) rc = bounds_check(codes, scale, batch, nkv, kv->max_blocks);
    if (rc != B2_OK) return rc;
    BoundsArgs a = {};
    a.pool = static_cast<const uint8_t*>(kv->pool);
    a.stride_block = kv->stride_block;
    a.stride_head = (int64_t)(kv->block_size / 16) * kv4_tile(kv4_dp(D));
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.newest = newest;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.batch = batch;
    a.nkv = nkv;
    a.D = D;
    a.codes = static_cast<int8_t*>(codes);
    a.scale = scale;
    return bounds_launch(a, true, as_stream(stream));
}

extern "C" size_t b2_paged_block_select_workspace_bytes(int batch, int nkv, int max_blocks) {
    if (batch <= 0 || nkv <= 0 || max_blocks <= 0) return 0;
    return (size_t)batch * nkv * max_blocks * sizeof(uint32_t);
}

extern "C" int b2_paged_block_select(const b2_block_select* r, b2_workspace* ws, void* stream) {
    using namespace b2;
    B2_REQUIRE(r);
    const int batch = r->batch, nq = r->num_q_heads, nkv = r->num_kv_heads, D = r->head_dim, max_blocks = r->max_blocks;
    if (batch <= 0) return B2_OK;
    B2_REQUIRE(r->q && r->block_tables && r->seq_lens && r->blocks && r->num_blocks > 0 && r->block_size > 0 && max_blocks > 0 &&
               r->n > 0 && r->first >= 0 && r->last >= 0 && (int64_t)r->first + r->last <= r->n && nq > 0 && nkv > 0 &&
               nq % nkv == 0 && D > 0);
    const int rc = bounds_check(r->codes, r->scale, batch, nkv, max_blocks);
    if (rc != B2_OK) return rc;
    if (D > 256 || (D & 7) || (int64_t)max_blocks * r->block_size > (1 << 30) || batch > 65535 || nkv > 65535)
        return B2_ERR_UNSUPPORTED;
    if (!ws || ws->bytes < b2_paged_block_select_workspace_bytes(batch, nkv, max_blocks)) return B2_ERR_WORKSPACE;
    SelectArgs a = {};
    a.q = r->q;
    a.ldq = r->ldq;
    a.block_tables = r->block_tables;
    a.seq_lens = r->seq_lens;
    a.num_blocks = r->num_blocks;
    a.block_size = r->block_size;
    a.max_blocks = max_blocks;
    a.codes = static_cast<const int8_t*>(r->codes);
    a.scale = r->scale;
    a.out = r->blocks;
    a.nq = nq;
    a.nkv = nkv;
    a.D = D;
    a.group = nq / nkv;
    a.bf16 = r->bf16;
    a.n = r->n;
    a.first = r->first;
    a.last = r->last;
    a.keys = static_cast<uint32_t*>(ws->ptr);
    // up to 8 heads per CTA, and as many CTAs as an SM holds together where that leaves each a few steps
    a.heads = nkv < kScWarps ? nkv : kScWarps;
    a.team = kScWarps / a.heads;
    const int64_t groups = (nkv + a.heads - 1) / a.heads, step = 8 * a.team;
    int64_t chunk = (batch * groups * max_blocks + 2 * sm_count() - 1) / (2 * sm_count());
    chunk = chunk < 4 * step ? 4 * step : chunk > 32 * step ? 32 * step : (chunk + step - 1) / step * step;
    a.chunk = (int)chunk;
    cudaStream_t s = as_stream(stream);
    if (D <= 64) return select_launch<2>(a, batch, s);
    if (D <= 128) return select_launch<4>(a, batch, s);
    return select_launch<8>(a, batch, s);
}
