// paged_append.cu -- the rows of new tokens into a paged K/V cache, the position
// rotation of their queries and keys on the way (operator API paged_kv_append),
// for caches of 16-bit and of 4-bit rows, and rows of a 4-bit cache back to 16
// bits (paged_kv_read).
//
//   x'_i = x_i cos a_i - x_{i + r/2} sin a_i, x'_{i + r/2} = x_{i + r/2} cos a_i
//   + x_i sin a_i for i < r/2 of the first r channels, a_i = position f_i
//   4-bit rows, per group of 64 channels: m = half(min x), s = half((max x - m)
//   / 15), u = (x - m) / s rounded to even and clamped to 0 .. 15
//
// One read of q, k and v and one write of q and the rows: HBM bounds long
// prompts, latency single tokens.  A CTA takes up to 8 consecutive tokens of a
// sequence (all heads, or a share of them where there are few tokens), so the
// angles are worked out once per token and not per head.  The angle is kept as
// turns: position times f / 2 pi in 64 bits, its whole part dropped, so that far
// positions lose nothing; sine and cosine then in 32 bits, for which rows of 16
// bits are too coarse to notice.
//
// 4-bit codes are decided exactly: a key near the border between two codes would
// otherwise fall either way by the rounding of whoever rotates it.  Keys are
// rotated in 64 bits (the B200 has a 64-bit multiply-add for every two 32-bit
// ones, so this stays below the memory time); the division is a 32-bit product
// wherever that cannot miss the border, which is checked, and settled in 64 bits
// where it can.
#include <cmath>

#include "kv4.cuh"
#include "mma.cuh"

namespace b2 {

constexpr int kApThreads = 256;
constexpr int kApTokens = 8;

struct AppendArgs {
    b2_kv_view q, k, v, q_out;
    b2_paged_kv kv;       // 16-bit rows
    uint8_t* pool;        // 4-bit rows
    int64_t pool_block, head_bytes;
    const int *block_tables, *seq_lens, *counts, *positions;
    int num_blocks, block_size, max_blocks;
    int S, nq, nkv, D, rot, tokens, shares, bf16;
    int per;              // items of a row
    BlockDiv by_item;
    double turns[128];    // f_i / 2 pi
};

template <int V>
struct Chunk {};
template <>
struct Chunk<8> {
    using T = uint4;
};
template <>
struct Chunk<4> {
    using T = uint2;
};
__device__ __forceinline__ float2 unpack2(uint32_t x, bool bf16) {
    return bf16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) : h2_to_f2(x);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf16) {
    return bf16 ? pack16<true>(a, b) : pack16<false>(a, b);
}

// How many new rows sequence b has, and where the first one goes.
__device__ __forceinline__ int2 new_rows(const int* seq_lens, const int* counts, int b, int S) {
    const int n = counts ? max(0, min(S, counts[b])) : S;
    return make_int2(n, seq_lens[b] - n);
}

// u of (x - m) / s: d = x - m, r = 32-bit 1 / s
__device__ __forceinline__ int code_of(double d, float df, double s, float r) {
    const float t = df * r;
    float u = rintf(t);
    if (fabsf(t - u) > 0.4998f && t < 16.f) {
        // (the product is off by less than 16 * 2^-22: elsewhere its rounding is right)
        const double left = d - (double)u * s;
        if (left > 0.5 * s || (left == 0.5 * s && ((int)u & 1))) u += 1.f;
        if (left < -0.5 * s || (left == -0.5 * s && ((int)u & 1))) u -= 1.f;
    }
    return (int)fminf(fmaxf(u, 0.f), 15.f);
}

// KV4: rows of 4 bits.  VEC: channels per load, 8, or 4 where half the rotated
// channels are no multiple of 8.
template <bool KV4, int VEC>
__global__ void __launch_bounds__(kApThreads) append_kernel(const __grid_constant__ AppendArgs a) {
    using Vec = typename Chunk<VEC>::T;
    __shared__ float2 s_cs[kApTokens][128];
    __shared__ double2 s_cs64[KV4 ? kApTokens : 1][128];
    __shared__ int64_t s_row[kApTokens];  // where a token's rows go: element offset of head 0, or byte offset of its tile
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.z, share = blockIdx.y, t0 = blockIdx.x * a.tokens;
    griddep_wait();
    griddep_launch_dependents();
    const int2 rows = new_rows(a.seq_lens, a.counts, b, a.S);
    const int nt = min(a.tokens, rows.x - t0);
    if (nt <= 0) return;
    if (tid < nt) {
        const int64_t pos = (int64_t)rows.y + t0 + tid;
        int64_t at = -1;
        if (pos >= 0 && pos < (int64_t)a.max_blocks * a.block_size) {
            const int blk = (int)pos / a.block_size, slot = (int)pos - blk * a.block_size;
            const int id = a.block_tables[(int64_t)b * a.max_blocks + blk];
            if ((unsigned)id < (unsigned)a.num_blocks) {
                if (KV4)
                    at = ((int64_t)id * a.pool_block + (int64_t)(slot >> 4) * kv4_tile(kv4_dp(a.D))) * 16 + (slot & 15);
                else
                    at = (int64_t)id * a.kv.stride_block + (int64_t)slot * a.kv.stride_slot;
            }
        }
        s_row[tid] = at;
    }
    const int half = a.rot / 2;
    const int64_t first = a.positions ? (int64_t)a.positions[b] + t0 : (int64_t)rows.y + t0;
    for (int i = tid; i < nt * half; i += kApThreads) {
        const int t = i / half, e = i - t * half;
        double turn = (double)(first + t) * a.turns[e];
        turn -= rint(turn);
        if (KV4) {
            double sn, cn;
            sincospi(2.0 * turn, &sn, &cn);
            s_cs64[t][e] = make_double2(cn, sn);
            s_cs[t][e] = make_float2((float)cn, (float)sn);
        } else {
            float sn, cn;
            sincospif((float)(2.0 * turn), &sn, &cn);
            s_cs[t][e] = make_float2(cn, sn);
        }
    }
    __syncthreads();

    const int q0 = a.nq * share / a.shares, q1 = a.nq * (share + 1) / a.shares;
    const int k0 = a.nkv * share / a.shares, k1 = a.nkv * (share + 1) / a.shares;
    const int heads = (a.q.data ? q1 - q0 : 0) + (KV4 ? 0 : 2 * (k1 - k0));
    // ---- rows of 16 bits: an item is two chunks of VEC channels that are rotated together, or two to be copied
    const int items = nt * heads * a.per;
    constexpr int ON = 4;
    for (int i0 = tid; i0 < items; i0 += ON * kApThreads) {
        Vec x[ON], y[ON];
        const uint16_t* src[ON];
        uint16_t* dst[ON];
        int c0[ON], c1[ON], tok[ON];  // channels of the two chunks; c1 < 0: none
        bool turn[ON];
#pragma unroll
        for (int n = 0; n < ON; ++n) {
            const int i = i0 + n * kApThreads;
            dst[n] = nullptr;
            if (i >= items) continue;
            const int r = a.by_item.block(i), e = a.by_item.slot(i, r);
            tok[n] = r / heads;
            int h = r - tok[n] * heads;
            const int s = t0 + tok[n];
            turn[n] = e < a.rot / (2 * VEC);
            c0[n] = turn[n] ? e * VEC : a.rot + (e - a.rot / (2 * VEC)) * 2 * VEC;
            c1[n] = turn[n] ? half + e * VEC : c0[n] + VEC;
            if (c1[n] >= a.D) c1[n] = -1;
            const int nqh = a.q.data ? q1 - q0 : 0;
            if (h < nqh) {
                h += q0;
                src[n] = static_cast<const uint16_t*>(a.q.data) + b * a.q.stride_b + s * a.q.stride_s + h * a.q.stride_h;
                dst[n] = static_cast<uint16_t*>(const_cast<void*>(a.q_out.data)) + b * a.q_out.stride_b +
                         s * a.q_out.stride_s + h * a.q_out.stride_h;
            } else {
                h -= nqh;
                const bool key = h < k1 - k0;
                h = k0 + (key ? h : h - (k1 - k0));
                const b2_kv_view& w = key ? a.k : a.v;
                src[n] = static_cast<const uint16_t*>(w.data) + b * w.stride_b + s * w.stride_s + h * w.stride_h;
                if (!key) turn[n] = false;
                if (s_row[tok[n]] >= 0)
                    dst[n] = static_cast<uint16_t*>(key ? a.kv.k : a.kv.v) + s_row[tok[n]] + (int64_t)h * a.kv.stride_head;
            }
            if (!dst[n]) continue;
            x[n] = *reinterpret_cast<const Vec*>(src[n] + c0[n]);
            if (c1[n] >= 0) y[n] = *reinterpret_cast<const Vec*>(src[n] + c1[n]);
        }
#pragma unroll
        for (int n = 0; n < ON; ++n) {
            if (!dst[n]) continue;
            if (turn[n]) {
                uint32_t* xs = reinterpret_cast<uint32_t*>(&x[n]);
                uint32_t* ys = reinterpret_cast<uint32_t*>(&y[n]);
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                    const float2 u = unpack2(xs[j], a.bf16), w = unpack2(ys[j], a.bf16);
                    const float2 t = s_cs[tok[n]][c0[n] + 2 * j], v = s_cs[tok[n]][c0[n] + 2 * j + 1];
                    xs[j] = pack2(u.x * t.x - w.x * t.y, u.y * v.x - w.y * v.y, a.bf16);
                    ys[j] = pack2(w.x * t.x + u.x * t.y, w.y * v.x + u.y * v.y, a.bf16);
                }
            }
            *reinterpret_cast<Vec*>(dst[n] + c0[n]) = x[n];
            if (c1[n] >= 0) *reinterpret_cast<Vec*>(dst[n] + c1[n]) = y[n];
        }
    }
    if (!KV4) return;

    // ---- rows of 4 bits: lane l holds channels 4 l .. 4 l + 3 of 128 at a time, 16 lanes a group; two rows at once
    // where a row has 64
    const int DP = kv4_dp(a.D), NG = kv4_groups(DP), kvh = k1 - k0;
    const bool twin = DP == 64;
    const int sub = twin ? lane >> 4 : 0, c4 = (twin ? lane & 15 : lane) * 4;
    const int nr = nt * kvh;  // rows of K, then of V
    for (int r0 = warp * (twin ? 2 : 1); r0 < 2 * nr; r0 += kApThreads / 32 * (twin ? 2 : 1)) {
        const int r = min(r0 + sub, 2 * nr - 1);
        const bool key = r < nr;
        const int rr = key ? r : r - nr, tok = rr / kvh, h = k0 + rr - tok * kvh;
        const int64_t at = s_row[tok];
        const b2_kv_view& w = key ? a.k : a.v;
        const uint16_t* src = static_cast<const uint16_t*>(w.data) + b * w.stride_b + (int64_t)(t0 + tok) * w.stride_s +
                              h * w.stride_h;
        const bool mine = at >= 0 && r0 + sub < 2 * nr;
        const int p = (int)(at & 15);
        uint8_t* tile = a.pool + (at >> 4) + h * a.head_bytes;
        for (int c = c4; c < (DP + 127) / 128 * 128; c += 128) {
            const bool in = c < a.D;
            double x[4] = {0, 0, 0, 0};
            float f[4] = {0.f, 0.f, 0.f, 0.f};
            if (in) {
                auto four = [&](int ch, float (&v)[4]) {
                    const uint2 u = *reinterpret_cast<const uint2*>(src + ch);
                    const float2 p0 = unpack2(u.x, a.bf16), p1 = unpack2(u.y, a.bf16);
                    v[0] = p0.x, v[1] = p0.y, v[2] = p1.x, v[3] = p1.y;
                };
                four(c, f);
                if (key && c < a.rot) {  // (half the rotated channels are a multiple of 4)
                    const bool low = c < half;
                    float g[4];
                    four(low ? c + half : c - half, g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const double2 t = s_cs64[tok][(low ? c : c - half) + i];
                        x[i] = fma((double)f[i], t.x, (low ? -(double)g[i] : (double)g[i]) * t.y);
                        f[i] = (float)x[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = f[i];
                }
            }
            // least and largest of the group; the least only as a half of its 32-bit value is needed
            float lo = INFINITY;
            double hi = -INFINITY;
            bool fine = true;
            if (in) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    lo = fminf(lo, f[i]);
                    hi = x[i] > hi ? x[i] : hi;
                    fine = fine && fabsf(f[i]) < INFINITY;
                }
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
                const double y = __shfl_xor_sync(~0u, hi, o);
                hi = y > hi ? y : hi;
            }
            const uint32_t odd = __ballot_sync(~0u, !fine);
            fine = ((odd >> (lane & 16)) & 0xffffu) == 0;
            __half m = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f));
            double span = (hi - (double)__half2float(m)) / 15.0;
            span = span > 65504.0 ? 65504.0 : span > 0.0 ? span : 0.0;
            __half s = __float2half_rn((float)span);
            if (!fine) m = s = __ushort_as_half(0x7fff);
            if (fine && hi < lo) m = s = __ushort_as_half(0);  // a group of padding alone
            const float sf = __half2float(s), mf = __half2float(m);
            uint32_t codes = 0;
            if (in && sf > 0.f) {
                const float rs = __frcp_rn(sf);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    codes |= code_of(x[i] - (double)mf, key ? (float)(x[i] - (double)mf) : f[i] - mf, (double)sf, rs) << (4 * i);
            }
            if (!mine || c >= DP) continue;
            const int j = c >> 3, x32 = c >> 5, r8 = (c & 31) >> 2;
            const int place = key ? p * (DP / 2) + ((j & 3) * (DP / 32) + (j >> 2)) * 4 + ((c >> 2) & 1) * 2
                                  : 8 * DP + ((x32 * 8 + r8) * 4 + ((p & 7) >> 1)) * 8 + (p >> 3) * 4 + (p & 1) * 2;
            *reinterpret_cast<uint16_t*>(tile + place) = (uint16_t)codes;
            if ((c & 63) == 0)
                *reinterpret_cast<__half2*>(tile + 16 * DP + (key ? 0 : 64 * NG) + (kv4_slot(p) * NG + (c >> 6)) * 4) =
                    __halves2half2(s, m);
        }
    }
}

struct ReadArgs {
    b2_kv_view k, v;
    const uint8_t* pool;
    int64_t pool_block, head_bytes;
    const int *block_tables, *seq_lens, *counts;
    int num_blocks, block_size, max_blocks, T, nkv, D, bf16;
};

// A warp per tile of 16 positions and kv head; its lanes read what they read in
// the attention's products (kv4.cuh) and write 16 bytes of K, 8 of V at a time.
template <int DP>
__global__ void __launch_bounds__(128) kv4_read_kernel(const ReadArgs a) {
    constexpr int W = DP / 32, NG = kv4_groups(DP);
    griddep_wait();
    griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lr = lane >> 2, lc = lane & 3;
    const int b = blockIdx.z, h = blockIdx.y;
    const int len = max(0, min(a.seq_lens[b], a.max_blocks * a.block_size));
    const int n = max(0, min(min(len, a.T), a.counts ? a.counts[b] : a.T));
    const int first = len - n;
    const int tile0 = (first >> 4) + blockIdx.x * 4 + warp, pos0 = tile0 * 16;
    if (pos0 >= len) return;
    const int blk = pos0 / a.block_size, slot = pos0 - blk * a.block_size;
    const int id = a.block_tables[(int64_t)b * a.max_blocks + blk];
    if ((unsigned)id >= (unsigned)a.num_blocks) return;
    const uint8_t* tile = a.pool + (int64_t)id * a.pool_block + h * a.head_bytes + (int64_t)(slot >> 4) * kv4_tile(DP);
    uint32_t kw[2][W], vw[W][2], km[2][NG], vm[4][NG];
#pragma unroll
    for (int pp = 0; pp < 2; ++pp) {
#pragma unroll
        for (int j = 0; j < W; ++j)
            kw[pp][j] = *reinterpret_cast<const uint32_t*>(tile + (lr + 8 * pp) * (DP / 2) + (lc * W + j) * 4);
#pragma unroll
        for (int g = 0; g < NG; ++g)
            km[pp][g] = *reinterpret_cast<const uint32_t*>(tile + 16 * DP + (kv4_slot(lr + 8 * pp) * NG + g) * 4);
    }
#pragma unroll
    for (int x = 0; x < W; ++x) {
        const uint2 u = *reinterpret_cast<const uint2*>(tile + 8 * DP + (x * 32 + lane) * 8);
        vw[x][0] = u.x, vw[x][1] = u.y;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < NG; ++g)
            vm[i][g] = *reinterpret_cast<const uint32_t*>(tile + 16 * DP + 64 * NG + ((lc * 4 + i) * NG + g) * 4);
    uint16_t* ko = static_cast<uint16_t*>(const_cast<void*>(a.k.data)) + b * a.k.stride_b + h * a.k.stride_h;
    uint16_t* vo = static_cast<uint16_t*>(const_cast<void*>(a.v.data)) + b * a.v.stride_b + h * a.v.stride_h;
#pragma unroll
    for (int pp = 0; pp < 2; ++pp) {
        const int pos = pos0 + lr + 8 * pp;
        if (pos < first || pos >= len) continue;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int c = 32 * j + 8 * lc;
            if (c >= a.D) continue;
            const float2 sm = h2_to_f2(km[pp][j / 2]);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = fmaf((float)((kw[pp][j] >> (4 * e)) & 15), sm.x, sm.y);
            *reinterpret_cast<uint4*>(ko + (int64_t)(pos - first) * a.k.stride_s + c) =
                make_uint4(pack2(f[0], f[1], a.bf16), pack2(f[2], f[3], a.bf16), pack2(f[4], f[5], a.bf16),
                           pack2(f[6], f[7], a.bf16));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // positions 2 lc, 2 lc + 1 and those + 8
        const int pos = pos0 + (i >> 1) * 8 + 2 * lc + (i & 1);
        if (pos < first || pos >= len) continue;
#pragma unroll
        for (int x = 0; x < W; ++x) {
            const int c = 32 * x + 4 * lr;
            if (c >= a.D) continue;
            const float2 sm = h2_to_f2(vm[i][x / 2]);
            const uint32_t u = vw[x][i >> 1] >> (16 * (i & 1));
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = fmaf((float)((u >> (4 * e)) & 15), sm.x, sm.y);
            *reinterpret_cast<uint2*>(vo + (int64_t)(pos - first) * a.v.stride_s + c) =
                make_uint2(pack2(f[0], f[1], a.bf16), pack2(f[2], f[3], a.bf16));
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

static bool rows_fit(const b2_kv_view& v) {
    return aligned16(v.data) && v.stride_d == 1 && !((v.stride_b | v.stride_h | v.stride_s) & 7);
}

// What both kinds of cache share: arguments checked and filled in but for the cache.
static int append_args(AppendArgs& a, const b2_kv_view* q, const b2_kv_view* q_out, b2_kv_view k, b2_kv_view v,
                       const double* inv_freq, int rot, const int* counts, const int* positions, int batch, int64_t S,
                       int nq, int nkv, int D) {
    B2_REQUIRE(k.data && v.data && nkv > 0 && D > 0 && rot >= 0 && (rot == 0 || inv_freq) && !q == !q_out);
    B2_REQUIRE(!q || (q->data && q_out->data && nq > 0));
    if (rot > D || (rot & 7) || S > (1 << 30) || batch > 65535 || !rows_fit(k) || !rows_fit(v) ||
        (q && (!rows_fit(*q) || !rows_fit(*q_out))))
        return B2_ERR_UNSUPPORTED;
    if (q) a.q = *q, a.q_out = *q_out;
    a.k = k;
    a.v = v;
    a.counts = counts;
    a.positions = positions;
    a.S = (int)S;
    a.nq = q ? nq : 0;
    a.nkv = nkv;
    a.D = D;
    a.rot = rot;
    for (int i = 0; i < rot / 2; ++i) a.turns[i] = inv_freq[i] / 6.283185307179586476925286766559;
    // whole tokens while they fill the GPU, shares of the heads else
    a.tokens = S < kApTokens ? (int)S : kApTokens;
    while (a.tokens > 1 && (S + a.tokens - 1) / a.tokens * batch < 2 * sm_count()) a.tokens /= 2;
    const int64_t ctas = (S + a.tokens - 1) / a.tokens * batch;
    a.shares = 1;
    while (a.shares < nkv && a.shares < 8 && ctas * a.shares * 2 <= sm_count()) a.shares *= 2;
    if (a.shares > nkv) a.shares = nkv;
    return B2_OK;
}

template <bool KV4>
static int append_launch(AppendArgs& a, int batch, cudaStream_t s) {
    const int vec = (a.rot / 2) % 8 == 0 ? 8 : 4;
    a.per = a.rot / (2 * vec) + (a.D - a.rot + 2 * vec - 1) / (2 * vec);
    a.by_item = block_div(a.per);
    const dim3 grid((unsigned)((a.S + a.tokens - 1) / a.tokens), (unsigned)a.shares, (unsigned)batch);
    if (vec == 8)
        B2_TRY(launch(append_kernel<KV4, 8>, grid, dim3(kApThreads), 0, s, true, a));
    else
        B2_TRY(launch(append_kernel<KV4, 4>, grid, dim3(kApThreads), 0, s, true, a));
    return B2_OK;
}

}  // namespace b2

extern "C" int b2_paged_kv_append(const b2_paged_kv* kv, b2_kv_view k, b2_kv_view v, const b2_kv_view* q,
                                  const b2_kv_view* q_out, const double* inv_freq, int rotary_dim, const int* counts,
                                  const int* positions, int batch, int64_t S, int nq, int nkv, int D, void* stream) {
    using namespace b2;
    if (batch <= 0 || S <= 0) return B2_OK;
    const int rc = check_paged(kv, nkv, D);
    if (rc != B2_OK) return rc;
    AppendArgs a = {};
    const int rc2 = append_args(a, q, q_out, k, v, inv_freq, rotary_dim, counts, positions, batch, S, nq, nkv, D);
    if (rc2 != B2_OK) return rc2;
    a.kv = *kv;
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.bf16 = kv->bf16;
    return append_launch<false>(a, batch, as_stream(stream));
}

extern "C" int b2_paged_kv4_append(const b2_paged_kv4* kv, b2_kv_view k, b2_kv_view v, const b2_kv_view* q,
                                   const b2_kv_view* q_out, const double* inv_freq, int rotary_dim, const int* counts,
                                   const int* positions, int batch, int64_t S, int nq, int nkv, int D, void* stream) {
    using namespace b2;
    if (batch <= 0 || S <= 0) return B2_OK;
    const int rc = check_paged4(kv, nkv, D);
    if (rc != B2_OK) return rc;
    AppendArgs a = {};
    const int rc2 = append_args(a, q, q_out, k, v, inv_freq, rotary_dim, counts, positions, batch, S, nq, nkv, D);
    if (rc2 != B2_OK) return rc2;
    a.pool = static_cast<uint8_t*>(kv->pool);
    a.pool_block = kv->stride_block;
    a.head_bytes = (int64_t)(kv->block_size / 16) * kv4_tile(kv4_dp(D));
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.bf16 = kv->bf16;
    return append_launch<true>(a, batch, as_stream(stream));
}

extern "C" int b2_paged_kv4_read(const b2_paged_kv4* kv, b2_kv_view k_out, b2_kv_view v_out, const int* counts,
                                 int batch, int64_t T, int nkv, int D, void* stream) {
    using namespace b2;
    if (batch <= 0 || T <= 0) return B2_OK;
    B2_REQUIRE(k_out.data && v_out.data);
    const int rc = check_paged4(kv, nkv, D);
    if (rc != B2_OK) return rc;
    if (!rows_fit(k_out) || !rows_fit(v_out) || batch > 65535 || nkv > 65535 || T > (1 << 30)) return B2_ERR_UNSUPPORTED;
    ReadArgs a = {};
    a.k = k_out;
    a.v = v_out;
    a.pool = static_cast<const uint8_t*>(kv->pool);
    a.pool_block = kv->stride_block;
    a.head_bytes = (int64_t)(kv->block_size / 16) * kv4_tile(kv4_dp(D));
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.counts = counts;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.T = (int)T;
    a.nkv = nkv;
    a.D = D;
    a.bf16 = kv->bf16;
    const int64_t cap = (int64_t)kv->max_blocks * kv->block_size, most = T < cap ? T : cap;
    // up to most positions, whose first and last tile may be partial
    const dim3 grid((unsigned)((most + 30) / 16 / 4 + 1), (unsigned)nkv, (unsigned)batch);
    cudaStream_t s = as_stream(stream);
    switch (kv4_dp(D)) {
        case 64: B2_TRY(launch(kv4_read_kernel<64>, grid, dim3(128), 0, s, true, a)); break;
        case 96: B2_TRY(launch(kv4_read_kernel<96>, grid, dim3(128), 0, s, true, a)); break;
        case 128: B2_TRY(launch(kv4_read_kernel<128>, grid, dim3(128), 0, s, true, a)); break;
        case 192: B2_TRY(launch(kv4_read_kernel<192>, grid, dim3(128), 0, s, true, a)); break;
        default: B2_TRY(launch(kv4_read_kernel<256>, grid, dim3(128), 0, s, true, a)); break;
    }
    return B2_OK;
}
