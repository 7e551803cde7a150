// block_select.cu -- which blocks of a long paged cache a new token looks at
// (operator API paged_block_bounds and paged_block_select).
//
// Bounds.  For each block and kv head, lo_d <= k_d <= hi_d over the keys that
// the block holds, in 8 bits: whole multiples of one power of two per (block,
// head), the least that 127 multiples of cover the largest |k|, lo rounded down
// and hi up.  The bytes are the keys once; a CTA takes a (block, kv head), its
// warps every fourth row, a lane 4 channels.
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
// The bytes are 2 D + 4 per (block, kv head).  Scores go to the workspace; the
// CTA that arrives last for its (sequence, kv head) finds the n-th best by its
// ordered key, 11 bits of the range still open at a time, and lists what is
// above it and the first of those equal to it, in order.
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

template <bool KV4>
__global__ void __launch_bounds__(kBdThreads) bounds_kernel(const BoundsArgs a) {
    __shared__ int s_end[kBdThreads];  // (block, head) pairs of the sequences up to each of the next kBdThreads
    __shared__ float s_lo[kBdWarps][256], s_hi[kBdWarps][256];
    __shared__ float s_top[kBdWarps];
    __shared__ int s_bad;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();
    griddep_launch_dependents();
    const int DP = kv4_dp(a.D), NG = kv4_groups(DP);
    int64_t base = 0;  // pairs of the sequences before b0
    for (int b0 = 0; b0 < a.batch; b0 += kBdThreads) {
        // the blocks that sequence b0 + tid's newest positions lie in
        int n = 0;
        if (b0 + tid < a.batch) {
            const int len = max(0, min(a.seq_lens[b0 + tid], a.max_blocks * a.block_size));
            const int since = a.newest ? len - max(0, min(len, a.newest[b0 + tid])) : 0;
            if (since < len) n = (len - 1) / a.block_size - since / a.block_size + 1;
        }
        __syncthreads();
        s_end[tid] = n;
        __syncthreads();
        for (int o = 1; o < kBdThreads; o <<= 1) {
            const int v = tid >= o ? s_end[tid - o] : 0;
            __syncthreads();
            s_end[tid] += v;
            __syncthreads();
        }
        const int64_t all = (int64_t)s_end[kBdThreads - 1] * a.nkv;
        int64_t i = base > blockIdx.x ? blockIdx.x + (base - blockIdx.x + gridDim.x - 1) / gridDim.x * gridDim.x : blockIdx.x;
        for (; i < base + all; i += gridDim.x) {
            const int pair = (int)((i - base) / a.nkv), h = (int)(i - base - (int64_t)pair * a.nkv);
            int lo = 0, up = kBdThreads - 1;  // the first sequence whose blocks end behind this one
            while (lo < up) {
                const int mid = (lo + up) / 2;
                if (s_end[mid] > pair)
                    up = mid;
                else
                    lo = mid + 1;
            }
            const int b = b0 + lo, from_end = s_end[lo] - 1 - pair;
            const int len = max(0, min(a.seq_lens[b], a.max_blocks * a.block_size));
            const int blk = (len - 1) / a.block_size - from_end, rows = min(a.block_size, len - blk * a.block_size);
            const int id = a.block_tables[(int64_t)b * a.max_blocks + blk];
            if ((unsigned)id >= (unsigned)a.num_blocks) continue;
            if (tid == 0) s_bad = 0;
            __syncthreads();
            bool bad = false;
            for (int c = lane * 4; c < a.D; c += 128) {
                float l[4], u[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) l[e] = INFINITY, u[e] = -INFINITY;
                auto take = [&](const float (&f)[4]) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        l[e] = fminf(l[e], f[e]);
                        u[e] = fmaxf(u[e], f[e]);
                        bad |= !(fabsf(f[e]) < INFINITY);
                    }
                };
                if constexpr (KV4) {
                    const uint8_t* at = a.pool + (int64_t)id * a.stride_block + h * a.stride_head;
                    const int j = c >> 3, in_row = ((j & 3) * (DP / 32) + (j >> 2)) * 4 + ((c >> 2) & 1) * 2;
#pragma unroll 4
                    for (int r = warp; r < rows; r += kBdWarps) {
                        const uint8_t* tile = at + (int64_t)(r >> 4) * kv4_tile(DP);
                        const uint32_t w = *reinterpret_cast<const uint16_t*>(tile + (r & 15) * (DP / 2) + in_row);
                        const float2 sm = h2_to_f2(
                            *reinterpret_cast<const uint32_t*>(tile + 16 * DP + (kv4_slot(r & 15) * NG + (c >> 6)) * 4));
                        float f[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[e] = fmaf((float)((w >> (4 * e)) & 15), sm.x, sm.y);
                        take(f);
                    }
                } else {
                    const uint16_t* at = a.k + (int64_t)id * a.stride_block + (int64_t)h * a.stride_head + c;
#pragma unroll 4
                    for (int r = warp; r < rows; r += kBdWarps) {
                        const uint2 w = *reinterpret_cast<const uint2*>(at + r * a.stride_slot);
                        float2 x, y;
                        if (a.bf16) {
                            x = make_float2(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u));
                            y = make_float2(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
                        } else {
                            x = h2_to_f2(w.x), y = h2_to_f2(w.y);
                        }
                        const float f[4] = {x.x, x.y, y.x, y.y};
                        take(f);
                    }
                }
                *reinterpret_cast<float4*>(&s_lo[warp][c]) = make_float4(l[0], l[1], l[2], l[3]);
                *reinterpret_cast<float4*>(&s_hi[warp][c]) = make_float4(u[0], u[1], u[2], u[3]);
            }
            if (__any_sync(~0u, bad) && lane == 0) s_bad = 1;
            __syncthreads();
            float top = 0.f;
            for (int c = tid; c < a.D; c += kBdThreads) {
                float l = s_lo[0][c], u = s_hi[0][c];
#pragma unroll
                for (int w = 1; w < kBdWarps; ++w) l = fminf(l, s_lo[w][c]), u = fmaxf(u, s_hi[w][c]);
                s_lo[0][c] = l;
                s_hi[0][c] = u;
                top = fmaxf(top, fmaxf(fabsf(l), fabsf(u)));
            }
            top = warp_max(top);
            if (lane == 0) s_top[warp] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kBdWarps; ++w) top = fmaxf(top, s_top[w]);
            // the least e with top <= 127 * 2^e
            int e;
            const float f = frexpf(top, &e);
            e = max(-126, f > 127.f / 128.f ? e - 6 : e - 7);
            if (top == 0.f) e = 0;
            const double back = ldexp(1.0, -e);
            int8_t* out = a.codes + ((int64_t)id * a.nkv + h) * 2 * a.D;
            const bool fine = s_bad == 0;
            for (int c = tid; c < a.D; c += kBdThreads) {
                out[c] = (int8_t)(fine ? (int)floor((double)s_lo[0][c] * back) : 0);
                out[a.D + c] = (int8_t)(fine ? (int)ceil((double)s_hi[0][c] * back) : 0);
            }
            if (tid == 0) a.scale[(int64_t)id * a.nkv + h] = fine ? ldexpf(1.f, e) : INFINITY;
            __syncthreads();
        }
        base += all;
    }
}

static int bounds_launch(const BoundsArgs& a, bool kv4, cudaStream_t s) {
    // pairs are dealt out in turn: 16 CTAs of 4 warps fill an SM
    const int64_t most = (int64_t)a.batch * a.nkv * a.max_blocks;
    const unsigned grid = (unsigned)(most < 16 * sm_count() ? most : 16 * sm_count());
    if (kv4)
        B2_TRY(launch(bounds_kernel<true>, dim3(grid), dim3(kBdThreads), 0, s, true, a));
    else
        B2_TRY(launch(bounds_kernel<false>, dim3(grid), dim3(kBdThreads), 0, s, true, a));
    return B2_OK;
}

// ---------------------------------------------------------------------------
// choice
// ---------------------------------------------------------------------------

constexpr int kSlThreads = 256;
constexpr int kSlWarps = kSlThreads / 32;
constexpr int kSlKeys = 8192;  // keys of a choice kept in shared memory; of longer ones they are read again
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
    int chunk;       // blocks per CTA
    uint32_t* keys;  // [batch][nkv][max_blocks]
    int* counters;
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
template <int P>
__global__ void __launch_bounds__(kSlThreads) select_kernel(const SelectArgs a) {
    __shared__ union {
        struct {
            double sum[2][256];
            __align__(16) uint8_t hi[512], lo[512];
        } q;
        struct {
            uint32_t keys[kSlKeys];
            int hist[kSlBins];
        } c;
    } sm;
    __shared__ double s_red[kSlWarps];
    __shared__ int s_wsum[kSlWarps][2];
    __shared__ int s_last, s_bin, s_above;
    __shared__ uint32_t s_range[2][kSlWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.y, b = blockIdx.z;
    griddep_wait();
    griddep_launch_dependents();
    const int len = max(0, min(a.seq_lens[b], a.max_blocks * a.block_size));
    const int nb = (len + a.block_size - 1) / a.block_size;
    const int64_t pair = (int64_t)b * a.nkv + h;
    int* out = a.out + pair * a.n;
    if (nb <= a.n) {  // every block
        if (blockIdx.x == 0)
            for (int i = tid; i < a.n; i += kSlThreads) out[i] = i < nb ? i : -1;
        return;
    }
    const int c0 = blockIdx.x * a.chunk, c1 = min(nb, c0 + a.chunk);
    if (c0 >= nb) return;

    // ---- P and N in 16 bits: N first, as lo stands before hi
    double top = 0.0;
    for (int c = tid; c < a.D; c += kSlThreads) {
        double neg = 0.0, pos = 0.0;
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.ldq + (int64_t)h * a.group * a.D + c;
#pragma unroll 4
        for (int g = 0; g < a.group; ++g) {
            const uint32_t w = q[(int64_t)g * a.D];
            const float f = a.bf16 ? __uint_as_float(w << 16) : __half2float(__ushort_as_half((uint16_t)w));
            if (!(f <= 0.f)) pos += (double)f;  // (a NaN to both)
            if (!(f >= 0.f)) neg += (double)f;
        }
        sm.q.sum[0][c] = neg;
        sm.q.sum[1][c] = pos;
        const double t = fmax(-neg, pos);
        top = t > top || !(t < INFINITY) ? t : top;
        if (!(neg > -INFINITY) || !(pos < INFINITY)) top = INFINITY;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(~0u, top, o));
    if (lane == 0) s_red[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSlWarps; ++w) top = fmax(top, s_red[w]);
    int e = 0;
    const double f = frexp(top < INFINITY && top > 0.0 ? top : 1.0, &e);
    e = f > 32767.0 / 32768.0 ? e - 14 : e - 15;  // the least with top <= 32767 * 2^e
    const double back = top < INFINITY ? ldexp(1.0, -e) : 0.0;
    for (int i = tid; i < 2 * a.D; i += kSlThreads) {
        const double x = sm.q.sum[i >= a.D][i >= a.D ? i - a.D : i];
        const int v = top < INFINITY ? (int)rint(x * back) : 0;
        sm.q.hi[i] = (uint8_t)(v >> 8);
        sm.q.lo[i] = (uint8_t)v;
    }
    __syncthreads();

    // ---- scores of this CTA's blocks: 4 lanes a block
    uint32_t* keys = a.keys + pair * a.max_blocks;
    const int part = lane & 3, pieces = a.D / 8;
    uint4 qh[P], ql[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int at = part + 4 * p;
        qh[p] = at < pieces ? *reinterpret_cast<const uint4*>(sm.q.hi + 16 * at) : make_uint4(0, 0, 0, 0);
        ql[p] = at < pieces ? *reinterpret_cast<const uint4*>(sm.q.lo + 16 * at) : make_uint4(0, 0, 0, 0);
    }
    constexpr int STEP = kSlThreads / 4;
    constexpr int ON = P <= 4 ? 4 : 2;  // blocks of a thread at a time
    const int* bt = a.block_tables + (int64_t)b * a.max_blocks;
    for (int j0 = c0 + (tid >> 2); j0 - (tid >> 2) < c1; j0 += ON * STEP) {
        int id[ON];
#pragma unroll
        for (int n = 0; n < ON; ++n) id[n] = j0 + n * STEP < c1 ? bt[j0 + n * STEP] : -1;
        uint4 w[ON][P];
        float sc[ON];
#pragma unroll
        for (int n = 0; n < ON; ++n) {
            const bool there = (unsigned)id[n] < (unsigned)a.num_blocks;
            const int64_t row = (int64_t)id[n] * a.nkv + h;
            const uint4* src = reinterpret_cast<const uint4*>(a.codes + row * 2 * a.D) + part;
#pragma unroll
            for (int p = 0; p < P; ++p)
                w[n][p] = there && part + 4 * p < pieces ? __ldg(src + 4 * p) : make_uint4(0, 0, 0, 0);
            sc[n] = there ? a.scale[row] : 0.f;
        }
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
            int sum = hi * 256 + lo;
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
            const int j = j0 + n * STEP;
            if (part == 0 && j < c1) {
                const bool there = (unsigned)id[n] < (unsigned)a.num_blocks;
                const float score = sc[n] == INFINITY ? INFINITY : (float)sum * sc[n];
                // (a NaN, as of a scale never written, ranks first but is not one of the blocks that stay)
                keys[j] = j < a.first || j >= nb - a.last ? kSlStays
                                                          : there ? min(float_key(score + 0.f), kSlStays - 2) : 0u;
            }
        }
    }

    // ---- the last CTA of this (sequence, kv head) chooses
    const int ctas = (nb + a.chunk - 1) / a.chunk;
    if (ctas > 1) {
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            s_last = atomicAdd(a.counters + pair, 1) == ctas - 1;
            __threadfence();
        }
        __syncthreads();
        if (!s_last) return;
        if (tid == 0) a.counters[pair] = 0;
    }
    __syncthreads();
    const bool fits = nb <= kSlKeys;
    uint32_t lowest = ~0u, highest = 0u;
    for (int i = tid; i < nb; i += kSlThreads) {
        const uint32_t k = __ldcg(keys + i);
        if (fits) sm.c.keys[i] = k;
        if (k != kSlStays) lowest = min(lowest, k), highest = max(highest, k);
    }
    auto key = [&](int i) -> uint32_t { return fits ? sm.c.keys[i] : __ldcg(keys + i); };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lowest = min(lowest, __shfl_xor_sync(~0u, lowest, o));
        highest = max(highest, __shfl_xor_sync(~0u, highest, o));
    }
    if (lane == 0) s_range[0][warp] = lowest, s_range[1][warp] = highest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSlWarps; ++w) lowest = min(lowest, s_range[0][w]), highest = max(highest, s_range[1][w]);
    // want: how many of the keys lowest .. highest are chosen; all above are
    int want = a.n - a.first - a.last;
    while (want > 0 && lowest < highest) {
        const uint32_t range = highest - lowest;
        const int shift = max(0, 21 - __clz(range));  // range >> shift below 2048
        for (int i = tid; i < kSlBins; i += kSlThreads) sm.c.hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < nb; i += kSlThreads) {
            const uint32_t k = key(i) - lowest;
            if (k <= range) atomicAdd(&sm.c.hist[k >> shift], 1);
        }
        __syncthreads();
        // the bin of the want-th best: thread t sums the bins 8 t' .. 8 t' + 7, t' counting from the top
        constexpr int PER = kSlBins / kSlThreads;
        const int top_bin = kSlBins - 1 - tid * PER;
        int mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine += sm.c.hist[top_bin - i];
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) s_wsum[warp][0] = incl;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kSlWarps; ++w)
            if (w < warp) incl += s_wsum[w][0];
        if (incl >= want && incl - mine < want) {
            int above = incl - mine, bin = top_bin;
            while (above + sm.c.hist[bin] < want) above += sm.c.hist[bin--];
            s_bin = bin;
            s_above = above;
        }
        __syncthreads();
        want -= s_above;
        lowest += (uint32_t)s_bin << shift;
        highest = min(highest, lowest + ((1u << shift) - 1));
        __syncthreads();
    }
    // ---- what is above, and the first `want` that equal it, in order (want 0: nothing below the blocks that stay)
    const uint32_t border = want > 0 ? lowest : kSlStays - 1;
    const int per = (nb + kSlThreads - 1) / kSlThreads, i0 = min(nb, tid * per), i1 = min(nb, i0 + per);
    int above = 0, equal = 0;
    for (int i = i0; i < i1; ++i) {
        const uint32_t k = key(i);
        above += k > border;
        equal += k == border;
    }
    int ia = above, ie = equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, ia, o), y = __shfl_up_sync(~0u, ie, o);
        if (lane >= o) ia += x, ie += y;
    }
    if (lane == 31) s_wsum[warp][0] = ia, s_wsum[warp][1] = ie;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSlWarps; ++w)
        if (w < warp) ia += s_wsum[w][0], ie += s_wsum[w][1];
    above = ia - above;  // before this thread's own
    equal = ie - equal;
    for (int i = i0; i < i1; ++i) {
        const uint32_t k = key(i);
        const bool eq = k == border && equal < want;
        if (k > border || eq) out[above + min(equal, want)] = i;
        above += k > border;
        equal += k == border;
    }
}

template <int P>
static int select_launch(const SelectArgs& a, int batch, cudaStream_t s) {
    const dim3 grid((unsigned)((a.max_blocks + a.chunk - 1) / a.chunk), (unsigned)a.nkv, (unsigned)batch);
    B2_TRY(launch(select_kernel<P>, grid, dim3(kSlThreads), 0, s, true, a));
    return B2_OK;
}

}  // namespace b2

static int bounds_check(const void* codes, const void* scale, int batch, int nkv, int max_blocks) {
    B2_REQUIRE(codes && scale);
    if (!b2::aligned16(codes)) return B2_ERR_UNSUPPORTED;
    // blocks of all sequences are counted in 32 bits
    if ((int64_t)batch * max_blocks > (1ll << 31) - 1) return B2_ERR_UNSUPPORTED;
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

extern "C" int b2_paged_block_select(const void* q, int64_t ldq, int bf16, const int* block_tables, const int* seq_lens,
                                     int num_blocks, int block_size, int max_blocks, const void* codes,
                                     const float* scale, int* blocks, int n, int first, int last, int batch, int nq,
                                     int nkv, int D, b2_workspace* ws, void* stream) {
    using namespace b2;
    if (batch <= 0) return B2_OK;
    B2_REQUIRE(q && block_tables && seq_lens && blocks && num_blocks > 0 && block_size > 0 && max_blocks > 0 && n > 0 &&
               first >= 0 && last >= 0 && (int64_t)first + last <= n && nq > 0 && nkv > 0 && nq % nkv == 0 && D > 0);
    const int rc = bounds_check(codes, scale, batch, nkv, max_blocks);
    if (rc != B2_OK) return rc;
    if (D > 256 || (D & 7) || (int64_t)max_blocks * block_size > (1 << 30) || batch > 65535 || nkv > 65535)
        return B2_ERR_UNSUPPORTED;
    if (!ws || ws->bytes < b2_paged_block_select_workspace_bytes(batch, nkv, max_blocks)) return B2_ERR_WORKSPACE;
    SelectArgs a = {};
    a.q = q;
    a.ldq = ldq;
    a.block_tables = block_tables;
    a.seq_lens = seq_lens;
    a.num_blocks = num_blocks;
    a.block_size = block_size;
    a.max_blocks = max_blocks;
    a.codes = static_cast<const int8_t*>(codes);
    a.scale = scale;
    a.out = blocks;
    a.nq = nq;
    a.nkv = nkv;
    a.D = D;
    a.group = nq / nkv;
    a.bf16 = bf16;
    a.n = n;
    a.first = first;
    a.last = last;
    a.keys = static_cast<uint32_t*>(ws->ptr);
    a.counters = ws->counters;
    // a few CTAs per SM in all; as many counters as there are, else one CTA per choice
    const int64_t pairs = (int64_t)batch * nkv;
    int64_t chunk = (pairs * max_blocks + 4 * sm_count() - 1) / (4 * sm_count());
    chunk = (chunk + 255) / 256 * 256;
    a.chunk = pairs > kWsCounters || chunk >= max_blocks ? max_blocks : (int)chunk;
    cudaStream_t s = as_stream(stream);
    if (D <= 64) return select_launch<2>(a, batch, s);
    if (D <= 128) return select_launch<4>(a, batch, s);
    return select_launch<8>(a, batch, s);
}
