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
// turns: position times f / 2 pi, of f / 2 pi as two 64-bit numbers, with what the
// product's rounding leaves, so that dropping the whole part leaves 2^-53 of a turn
// wherever the position is (of one 64-bit number: 2^-53 of all turns since
// position 0, 2^-22 of an angle near position 2^31).  Sine and cosine then in 32
// bits, for which rows of 16 bits are too coarse to notice.
//
// 4-bit codes are decided exactly: a key near the border between two codes would
// otherwise fall either way by the rounding of whoever rotates it.  Rows are
// quantised in 32 bits with a bound on what that is off by; where the minimum,
// the scale or a code could round otherwise within it (1 row in 100 or so) the
// warp does them again in 64 bits, from sines and cosines kept as two 32-bit
// numbers each.  (All of it in 64 bits: 540 instructions for 8 channels a lane,
// 101 us for 8192 tokens.)
//
// Measured: 8192 tokens, 32 query and 8 K/V heads of 128, into a 4-bit cache 58
// us (floor 27): keys and values alone 39, 365 instructions for 8 channels a lane,
// 0.59 of the issue slots with the 20 warps per SM that 80 registers leave (56 bytes
// spilled, 88 at 64 channels, 24 for rows of 16 bits); queries alone 21, bound by
// HBM.  Their CTAs stand between the others, which overlaps little (one kind after
// the other: 63 us).  16 channels a lane: fewer instructions by an eighth, but more
// spills (68 us).  One token of one sequence 4 us in a graph: the
// chain length, table entry, row.
#include <cmath>
#include <type_traits>

#include "kv4.cuh"
#include "mma.cuh"

namespace b2 {

using namespace packed;

constexpr int kApThreads = 256;
constexpr int kApTokens = 8;
constexpr int64_t kNoRow = INT64_MIN;  // a token whose rows have no place
constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnRest = -0x1.6b01ec5417056p-57;  // 1 / 2 pi to 107 bits

struct AppendArgs {
    b2_kv_view q, k, v, q_out;
    b2_paged_kv kv;       // 16-bit rows
    uint8_t* pool;        // 4-bit rows
    int64_t pool_block, head_bytes;
    const int *block_tables, *seq_lens, *counts, *positions;
    int num_blocks, block_size, max_blocks;
    int S, nq, nkv, D, rot, tokens, shares, q_shares, q_heads, k_heads, bf16;  // heads of a share
    int vec, per, fit, groups;  // threads that a row takes; rows side by side, and for each token where a CTA has all of its
    uint32_t per_inv, tokens_inv, half_inv;  // 2^20 / d + 1 of them
    double inv_freq[128];
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
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
    return BF16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) : h2_to_f2(x);
}

// Where quad x of angles stands: lanes 4 or 8 quads apart read different banks.
__device__ __forceinline__ int spread(int x) { return x + (x >> 3); }

// floor(i / d) by inv = 2^20 / d + 1, for i d < 2^20
__device__ __forceinline__ int over(int i, uint32_t inv) { return (int)(((uint32_t)i * inv) >> 20); }
__device__ __forceinline__ uint64_t pair(float2 x) { return pair(x.x, x.y); }

// WIDE: rows of 4 bits, 1 << WIDE lanes for each; 0: rows of 16 bits.  VEC: channels per load, 8, or 4 where half the rotated
// channels are no multiple of 8.
template <int WIDE, int VEC, bool BF16>
__global__ void __launch_bounds__(kApThreads, 3) append_kernel(const __grid_constant__ AppendArgs a) {
    using Vec = typename Chunk<VEC>::T;
    constexpr bool KV4 = WIDE > 0;
    // of two pairs of channels, at spread(pair / 2): cosines, sines; and what their rounding to 32 bits left
    __shared__ float4 s_cs[kApTokens][72], s_rest[KV4 ? kApTokens : 1][72];
    __shared__ int64_t s_row[kApTokens];  // where a token's rows go: element offset of its first head, or byte offset of its tile
    __shared__ int s_in[KV4 ? kApTokens : 1][3];  // in the tile: K row, V units, scales
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // rows of 4 bits have CTAs of their own, in turn with those of the queries
    const int kinds = KV4 ? a.q_shares + a.shares : a.shares, kind = blockIdx.x % kinds;
    const bool rows4 = KV4 && kind >= a.q_shares;
    const int b = blockIdx.y, share = kind - (rows4 ? a.q_shares : 0), t0 = blockIdx.x / kinds * a.tokens;
    griddep_wait();
    griddep_launch_dependents();
    const int news = a.counts ? max(0, min(a.S, a.counts[b])) : a.S;
    const int64_t place = (int64_t)a.seq_lens[b] - news + t0;  // of this CTA's first token
    const int nt = min(a.tokens, news - t0);
    if (nt <= 0) return;
    if (tid < nt) {
        const int64_t pos = place + tid;
        int64_t at = kNoRow;
        if (pos >= 0 && pos < (int64_t)a.max_blocks * a.block_size) {
            const int blk = (int)pos / a.block_size, slot = (int)pos - blk * a.block_size;
            const int id = a.block_tables[(int64_t)b * a.max_blocks + blk];
            if ((unsigned)id < (unsigned)a.num_blocks) {
                if (KV4) {
                    const int DP = kv4_dp(a.D), p = slot & 15;
                    at = (int64_t)id * a.pool_block + (int64_t)(slot >> 4) * kv4_tile(DP);
                    s_in[tid][0] = p * (DP / 2);
                    s_in[tid][1] = 8 * DP + ((p & 7) >> 1) * 8 + (p >> 3) * 4 + (p & 1) * 2;
                    s_in[tid][2] = 16 * DP + kv4_slot(p) * kv4_groups(DP) * 4;
                } else
                    at = (int64_t)id * a.kv.stride_block + (int64_t)slot * a.kv.stride_slot +
                         share * a.k_heads * a.kv.stride_head;
            }
        }
        s_row[tid] = at;
    }
    const int half = a.rot / 2;
    const int64_t first = a.positions ? (int64_t)a.positions[b] + t0 : place;
    for (int i = tid; i < nt * half; i += kApThreads) {
        const int t = over(i, a.half_inv), e = i - t * half;
        // f / 2 pi as two numbers; turns, and what is left of them without the whole ones (two numbers per channel among the
        // arguments, read by every lane at a place of its own: 74 us instead of 69 for 8192 tokens and their reading back)
        const double f = a.inv_freq[e], hi = f * kTurn, lo = fma(f, kTurnRest, fma(f, kTurn, -hi));
        const double at = (double)(first + t), all = at * hi, turn = all - rint(all) + fma(at, lo, fma(at, hi, -all));
        float sn, cn;
        if (rows4) {  // rounded from 64 bits: within 2^-25 (a quarter of the rows that have to be done again)
            double sd, cd;
            sincospi(2.0 * turn, &sd, &cd);
            sn = (float)sd, cn = (float)cd;
            float* rest = reinterpret_cast<float*>(&s_rest[KV4 ? t : 0][spread(e >> 1)]) + (e & 1);
            rest[0] = (float)(cd - cn);
            rest[2] = (float)(sd - sn);
        } else {
            sincospif((float)(2.0 * turn), &sn, &cn);
        }
        float* cs = reinterpret_cast<float*>(&s_cs[t][spread(e >> 1)]) + (e & 1);
        cs[0] = cn;
        cs[2] = sn;
    }
    __syncthreads();

    const int q0 = min(a.nq, share * a.q_heads), q1 = min(a.nq, q0 + a.q_heads);
    const int k0 = min(a.nkv, share * a.k_heads), k1 = min(a.nkv, k0 + a.k_heads);
    // ---- rows of 16 bits: a thread has two chunks of VEC channels that are rotated together, or two to be copied, of one
    // token (its angles stay in registers) and goes through heads
    if (!rows4) {
        const int pairs = a.rot / (2 * VEC), lead = over(tid, a.per_inv), e = tid - lead * a.per;
        const bool turns = e < pairs;
        const int c0 = turns ? e * VEC : a.rot + (e - pairs) * 2 * VEC, c1 = turns ? half + c0 : c0 + VEC;
        const bool both = c1 < a.D;
        // tokens side by side, and threads for each; this thread's
        const bool all = nt == a.tokens;
        const int tp = min(nt, a.fit), groups = all ? a.groups : a.fit / tp, group = all ? over(lead, a.tokens_inv) : lead / tp;
        const int mine = lead - group * tp;
        // rows of `heads` heads from h0 on; TURN: rotated.  Into the cache where `to` is null
        auto all_of = [&](auto turn, const b2_kv_view& view, int h0, int heads, uint16_t* to, int64_t to_s, int64_t to_h,
                          int group, int groups) {
            constexpr bool TURN = decltype(turn)::value;
            constexpr int ON = 4;  // rows of a thread on their way
            for (int tok = mine; tok < nt && group < groups; tok += tp) {
                uint16_t* dst = to ? to + tok * to_s : static_cast<uint16_t*>(TURN ? a.kv.k : a.kv.v) + s_row[tok];
                if (!to && s_row[tok] == kNoRow) continue;
                const uint16_t* src = static_cast<const uint16_t*>(view.data) + b * view.stride_b +
                                      (int64_t)(t0 + tok) * view.stride_s + (h0 + group) * view.stride_h + c0;
                dst += group * to_h + c0;
                const int64_t step = groups * view.stride_h, to_step = groups * to_h;
                const int next = c1 - c0;
                uint64_t cn[VEC / 2], sn[VEC / 2], ns[VEC / 2];
                if (TURN && turns) {
#pragma unroll
                    for (int j = 0; j < VEC / 2; ++j) {
                        const float4 t = s_cs[tok][spread((c0 >> 1) + j)];
                        cn[j] = pair(t.x, t.y), sn[j] = pair(t.z, t.w), ns[j] = pair(-t.z, -t.w);
                    }
                }
                for (int h = group; h < heads; h += ON * groups) {
                    Vec x[ON], y[ON];
#pragma unroll
                    for (int n = 0; n < ON; ++n) {
                        if (h + n * groups < heads) {
                            x[n] = *reinterpret_cast<const Vec*>(src);
                            if (both) y[n] = *reinterpret_cast<const Vec*>(src + next);
                        }
                        src += step;
                    }
#pragma unroll
                    for (int n = 0; n < ON; ++n) {
                        if (h + n * groups < heads) {
                            if (TURN && turns) {
                                uint32_t* xs = reinterpret_cast<uint32_t*>(&x[n]);
                                uint32_t* ys = reinterpret_cast<uint32_t*>(&y[n]);
#pragma unroll
                                for (int j = 0; j < VEC / 2; ++j) {
                                    const uint64_t u = pair(unpack2<BF16>(xs[j])), w = pair(unpack2<BF16>(ys[j]));
                                    const float2 p = two(fma2(w, ns[j], mul2(u, cn[j]))), q = two(fma2(u, sn[j], mul2(w, cn[j])));
                                    xs[j] = pack16<BF16>(p.x, p.y);
                                    ys[j] = pack16<BF16>(q.x, q.y);
                                }
                            }
                            *reinterpret_cast<Vec*>(dst) = x[n];
                            if (both) *reinterpret_cast<Vec*>(dst + next) = y[n];
                        }
                        dst += to_step;
                    }
                }
            }
        };
        uint16_t* const qo = static_cast<uint16_t*>(const_cast<void*>(a.q_out.data)) + b * a.q_out.stride_b +
                             t0 * a.q_out.stride_s + q0 * a.q_out.stride_h;
        const int nqh = q1 - q0, nkh = KV4 ? 0 : k1 - k0;  // (heads are counted from k0 in the cache too)
        if (groups < 3 || nqh == 0 || nkh == 0) {
            if (nqh) all_of(std::true_type{}, a.q, q0, nqh, qo, a.q_out.stride_s, a.q_out.stride_h, group, groups);
            if (nkh) {
                all_of(std::true_type{}, a.k, k0, nkh, nullptr, 0, a.kv.stride_head, group, groups);
                all_of(std::false_type{}, a.v, k0, nkh, nullptr, 0, a.kv.stride_head, group, groups);
            }
        } else {  // each thread has queries, keys or values, in the proportion of their heads
            const int gk = max(1, groups * nkh / (nqh + 2 * nkh)), gq = groups - 2 * gk;
            if (group < gq)
                all_of(std::true_type{}, a.q, q0, nqh, qo, a.q_out.stride_s, a.q_out.stride_h, group, gq);
            else if (group < gq + gk)
                all_of(std::true_type{}, a.k, k0, nkh, nullptr, 0, a.kv.stride_head, group - gq, gk);
            else
                all_of(std::false_type{}, a.v, k0, nkh, nullptr, 0, a.kv.stride_head, group - gq - gk, gk);
        }
    }
    if (!rows4) return;

    // ---- rows of 4 bits: a lane holds 8 channels, 8 lanes a group, 8, 16 or 32 lanes a row
    const int DP = kv4_dp(a.D), NG = kv4_groups(DP), kvh = k1 - k0;
    constexpr int at_once = 32 >> WIDE;
    const int sub = lane >> WIDE, c = (lane & ((1 << WIDE) - 1)) * 8;
    const bool in = c < a.D, turned = c < a.rot;
    const bool empty = c >= DP;  // (192 channels: 8 lanes have nothing)
    // K is rotated with the sign of the sine taken to the partner: whole chunks of 4 channels have one sign
    const bool low0 = c < half, low1 = c + 4 < half;
    const int e0 = low0 ? c : c - half, e1 = low1 ? c + 4 : c + 4 - half;  // pairs of channels c and c + 4
    const int g0 = low0 ? c + half : c - half, g1 = low1 ? c + 4 + half : c + 4 - half;  // and their partners
    constexpr int STEP = kApThreads / 32;
    // this lane's places in a K row, among a position's V units, among its scales
    const int in_k = (((c >> 3) & 3) * (DP / 32) + (c >> 5)) * 4, in_v = ((c >> 5) * 8 + ((c & 31) >> 2)) * 32;
    const int in_s = (c >> 6) * 4;
    // a warp has a token (several warps where there are fewer tokens than warps): its angles and places stay in registers
    // while the warp goes through heads, K's from the first warp on, V's from the last one
    const int team = max(1, STEP / nt), member = warp % team;
    auto rows_of = [&](auto is_key, int tok, int first_h) {
        constexpr bool key = decltype(is_key)::value;
        const b2_kv_view& view = key ? a.k : a.v;
        const int64_t at = s_row[tok];
        const int by = team * at_once;  // heads from a row to the lane's next one
        int h = first_h + sub;
        const uint16_t* src = static_cast<const uint16_t*>(view.data) + b * view.stride_b + (int64_t)(t0 + tok) * view.stride_s +
                              (k0 + h) * view.stride_h + c;
        uint8_t* tile = a.pool + at + (k0 + h) * a.head_bytes;
        const int64_t step = by * view.stride_h, tile_step = by * a.head_bytes;
        const int place = s_in[tok][key ? 0 : 1] + (key ? in_k : in_v), scales = s_in[tok][2] + (key ? 0 : 64 * NG) + in_s;
        float4 cs[4];
        if (key && turned) {
    #pragma unroll
            for (int i = 0; i < 8; i += 2) cs[i / 2] = s_cs[tok][spread((VEC == 8 || i < 4 ? e0 + i : e1 + i - 4) >> 1)];
        }
        // a row and the partners of its channels: the next row's are on their way while one is worked on
        struct Row {
            uint4 own;
            uint2 other[2];
        };
        auto fetch = [&](int hh, const uint16_t* p) {
            Row w;
            const bool there = in && hh < kvh;
            w.own = there ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
            w.other[0] = w.other[1] = make_uint2(0, 0);
            if (key && turned && there) {
                if (VEC == 8) {
                    const uint4 x = *reinterpret_cast<const uint4*>(p + (g0 - c));
                    w.other[0] = make_uint2(x.x, x.y), w.other[1] = make_uint2(x.z, x.w);
                } else {
                    w.other[0] = *reinterpret_cast<const uint2*>(p + (g0 - c));
                    w.other[1] = *reinterpret_cast<const uint2*>(p + (g1 - c));
                }
            }
            return w;
        };
        Row ahead = fetch(h, src);
        for (int hb = first_h; hb < kvh; hb += by) {
            const Row row = ahead;
            const bool mine = h < kvh && c < DP;
            uint8_t* const to = tile;
            src += step;
            h += by;
            tile += tile_step;
            ahead = fetch(h, src);
            const uint4 own = row.own;
            const uint2 other[2] = {row.other[0], row.other[1]};
            float f[8];
            auto unpack = [&](uint2 x, float* v) {
                const float2 p0 = unpack2<BF16>(x.x), p1 = unpack2<BF16>(x.y);
                v[0] = p0.x, v[1] = p0.y, v[2] = p1.x, v[3] = p1.y;
            };
            unpack(make_uint2(own.x, own.y), f);
            unpack(make_uint2(own.z, own.w), f + 4);
            if (key && turned) {
                const uint32_t n0 = low0 ? 0x80008000u : 0u, n1 = (VEC == 8 ? low0 : low1) ? 0x80008000u : 0u;
                float g[8];
                unpack(make_uint2(other[0].x ^ n0, other[0].y ^ n0), g);
                unpack(make_uint2(other[1].x ^ n1, other[1].y ^ n1), g + 4);
    #pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float4 t = cs[i / 2];
                    const float2 y = two(fma2(pair(make_float2(f[i], f[i + 1])), pair(make_float2(t.x, t.y)),
                                              mul2(pair(make_float2(g[i], g[i + 1])), pair(make_float2(t.z, t.w)))));
                    f[i] = y.x, f[i + 1] = y.y;
                }
            }
            float lo = f[0], hi = f[0], most = fabsf(f[0]);
    #pragma unroll
            for (int i = 1; i < 8; ++i) {
                lo = fminf(lo, f[i]);
                hi = fmaxf(hi, f[i]);
                most = max_nan(most, fabsf(f[i]));
            }
            if (!in) lo = INFINITY, hi = -INFINITY;
    #pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
                most = max_nan(most, __shfl_xor_sync(~0u, most, o));
            }
            const bool fine = most < INFINITY;
            // what f is off by, at most: sine and cosine 2^-25 each, a product 2^-24 |x2|, the sum 2^-24 of itself.  Turning
            // keeps x1^2 + x2^2, so with M the larger of what the two become |x1| + |x2| <= 2 M and |x2| <= 1.42 M: 2^-22 M
            float off = 0.f;
            if (key && a.rot) {
                off = most;
                for (int o = 8; o < (1 << WIDE); o <<= 1) off = max_nan(off, __shfl_xor_sync(~0u, off, o));
                off *= 0x1p-22f;
            }
            auto to_half = [](float x) { return __half2float(__float2half_rn(x)); };
            auto finite_half = [&](float x) { return to_half(fminf(fmaxf(x, -65504.f), 65504.f)); };
            float m = finite_half(lo);
            // the span is off by off + 2^-24 (hi - m), as a 15th of it by two roundings more
            const float span = fmaxf((hi - m) * (1.f / 15.f), 0.f), wrong = fmaf(off, 1.f / 15.f, span * 0x1p-22f);
            float s = to_half(fminf(span, 65504.f));
            bool sure = to_half(span - wrong) == to_half(span + wrong);
            if (key) sure = sure && to_half(lo - off) == to_half(lo + off);
            sure = sure && most < 65000.f;
            // u as the nearest whole number to t = (f - m) / s, cut to 0 .. 15: a 15th of it is cut to 0 .. 1 by its
            // multiply-add; adding 1.5 * 2^23 then leaves the whole number in the low bits
            constexpr float MAGIC = 12582912.f;
            const float rs = s > 0.f ? __frcp_rn(s) : 0.f, r15 = rs * (1.f / 15.f), m15 = -m * r15;
            uint32_t codes = 0;
            float worst = 0.f;
    #pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = __saturatef(fmaf(f[i], r15, m15)), v = fmaf(t, 15.f, MAGIC);
                worst = fmaxf(worst, fabsf(fmaf(t, 15.f, MAGIC - v)));
                codes += __float_as_uint(v) << (4 * i);
            }
            codes -= 0x4b400000u * 0x11111111u;
            // t is off by (off + 2^-21 most) / s and 2^-18: nearer to a half than that, it may round otherwise
            if (!in) worst = 0.f;
            bool near = !(worst < 0.5f - (fmaf(most, 0x1p-21f, off) * rs + 0x1p-18f));
            if (__any_sync(~0u, near && fine && off == 0.f)) {
                // numbers of 8 or 11 bits often lie half way exactly (1 group in 30 of bf16): what is left of f - m is exact in
                // 32 bits then, where f - m is
                bool exact = true;
                uint32_t fixed = 0;
    #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = f[i] - m, back = d - f[i];
                    exact = exact && (f[i] - (d - back)) == (m + back);
                    float u = fminf(fmaxf(rintf(d * rs), 0.f), 15.f);
                    const float left = fmaf(-u, s, d);
                    const bool odd = (int)u & 1;
                    if (left > 0.5f * s || (left == 0.5f * s && odd)) u += 1.f;
                    if (left < -0.5f * s || (left == -0.5f * s && odd)) u -= 1.f;
                    fixed |= (uint32_t)fminf(fmaxf(u, 0.f), 15.f) << (4 * i);
                }
                if (off == 0.f) {
                    codes = s > 0.f ? fixed : 0u;
                    near = near && !exact;
                }
            }
            sure = sure && !near;
            if (__any_sync(~0u, !(sure || !fine || empty))) {
                // in 64 bits
                double x[8];
                auto four = [&](uint2 own4, uint2 oth, bool low, int e, double* y) {
                    float u[4], g[4];
                    unpack(own4, u);
                    unpack(oth, g);
                    const float *cs = reinterpret_cast<const float*>(s_cs[tok]), *rest = reinterpret_cast<const float*>(s_rest[tok]);
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        y[i] = u[i];
                        if (key && turned) {
                            const int n = spread((e + i) >> 1) * 4 + (i & 1);  // (e is a multiple of 4)
                            const double cn = (double)cs[n] + rest[n], sn = (double)cs[n + 2] + rest[n + 2];
                            y[i] = fma((double)u[i], cn, (low ? -(double)g[i] : (double)g[i]) * sn);
                        }
                    }
                };
                four(make_uint2(own.x, own.y), other[0], low0, e0, x);
                four(make_uint2(own.z, own.w), other[1], VEC == 8 ? low0 : low1, VEC == 8 ? e0 + 4 : e1, x + 4);
                double l = in ? x[0] : INFINITY, u = in ? x[0] : -INFINITY;
                for (int i = 1; i < 8; ++i)
                    if (in) l = x[i] < l ? x[i] : l, u = x[i] > u ? x[i] : u;
                for (int o = 1; o < 8; o <<= 1) {
                    const double y = __shfl_xor_sync(~0u, l, o), z = __shfl_xor_sync(~0u, u, o);
                    l = y < l ? y : l;
                    u = z > u ? z : u;
                }
                m = finite_half((float)l);
                s = finite_half(fmaxf((float)((u - (double)m) / 15.0), 0.f));
                const double rs64 = s > 0.f ? __frcp_rn(s) : 0.f;  // (off by 2^-24: one step at most, put right by what is left)
                codes = 0;
#pragma unroll 1
                for (int i = 0; i < 8; ++i) {  // the nearest whole number to d / s, of two equally near ones the even
                    const double d = x[i] - (double)m;
                    int n = (int)rint(fmin(fmax(d * rs64, 0.0), 15.0));
                    const double left = fma((double)-n, (double)s, d);
                    const bool odd = n & 1;
                    if (left > 0.5 * s || (left == 0.5 * s && odd)) ++n;
                    if (left < -0.5 * s || (left == -0.5 * s && odd)) --n;
                    if (s > 0.f) codes |= (uint32_t)max(0, min(n, 15)) << (4 * i);
                }
            }
            if (!mine) continue;
            if (!in || !fine) codes = 0;
            if (key) {
                *reinterpret_cast<uint32_t*>(to + place) = codes;
            } else {
                *reinterpret_cast<uint16_t*>(to + place) = (uint16_t)codes;
                *reinterpret_cast<uint16_t*>(to + place + 32) = (uint16_t)(codes >> 16);
            }
            if ((c & 63) == 0) {
                __half2 sm = __floats2half2_rn(s, m);
                if (!fine) sm = __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff));
                *reinterpret_cast<__half2*>(to + scales) = sm;
            }
        }
    };
    for (int tok = warp / team; tok < nt && warp < nt * team; tok += STEP / team) {
        if (s_row[tok] == kNoRow) continue;
        rows_of(std::true_type{}, tok, member * at_once);
        rows_of(std::false_type{}, tok, (team - 1 - member) * at_once);
    }
}

struct ReadArgs {
    b2_kv_view k, v;
    const uint8_t* pool;
    int64_t pool_block, head_bytes;
    const int *block_tables, *seq_lens, *counts;
    int num_blocks, block_size, max_blocks, T, nkv, D, bf16;
};

// Bound by HBM: 1/4 of it read, the rest written (8192 tokens of 8 heads of 128: 8.5 us, 5.0 TB/s).
// A warp per tile of 16 positions and kv head; its lanes read what they read in
// the attention's products (kv4.cuh) and write 16 bytes of K, 8 of V at a time.
template <int DP, bool BF16>
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
                make_uint4(pack16<BF16>(f[0], f[1]), pack16<BF16>(f[2], f[3]), pack16<BF16>(f[4], f[5]),
                           pack16<BF16>(f[6], f[7]));
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
                make_uint2(pack16<BF16>(f[0], f[1]), pack16<BF16>(f[2], f[3]));
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// The stride of a dimension of one may be anything and is not used.
static void drop_unused(b2_kv_view& v, int batch, int64_t S, int heads) {
    if (batch == 1) v.stride_b = 0;
    if (S == 1) v.stride_s = 0;
    if (heads == 1) v.stride_h = 0;
}

static bool rows_fit(const b2_kv_view& v) {
    return aligned16(v.data) && v.stride_d == 1 && !((v.stride_b | v.stride_h | v.stride_s) & 7);
}

// Rows that are written have places of their own: no stride of 0.
static bool rows_apart(const b2_kv_view& v, int batch, int64_t S, int heads) {
    return (batch == 1 || v.stride_b) && (S == 1 || v.stride_s) && (heads == 1 || v.stride_h);
}

// What both kinds of cache share: arguments checked and filled in but for the cache.
static int append_args(AppendArgs& a, const b2_append& r) {
    const int batch = r.batch, nkv = r.num_kv_heads, nq = r.q.data ? r.num_q_heads : 0, D = r.head_dim, rot = r.rotary_dim;
    const int64_t S = r.S;
    B2_REQUIRE(r.k.data && r.v.data && nkv > 0 && D > 0 && rot >= 0 && (rot == 0 || r.inv_freq) && !r.q.data == !r.q_out.data &&
               (!r.q.data || nq > 0));
    a.k = r.k, a.v = r.v, a.q = r.q, a.q_out = r.q_out;
    drop_unused(a.k, batch, S, nkv);
    drop_unused(a.v, batch, S, nkv);
    drop_unused(a.q, batch, S, nq);
    drop_unused(a.q_out, batch, S, nq);
    if (rot > D || (rot & 7) || S > (1 << 30) || batch > 65535 || !rows_fit(a.k) || !rows_fit(a.v) ||
        (nq && (!rows_fit(a.q) || !rows_fit(a.q_out))))
        return B2_ERR_UNSUPPORTED;
    B2_REQUIRE(!nq || rows_apart(a.q_out, batch, S, nq));
    a.counts = r.counts;
    a.positions = r.positions;
    a.S = (int)S;
    a.nq = nq;
    a.nkv = nkv;
    a.D = D;
    a.rot = rot;
    for (int i = 0; i < rot / 2; ++i) a.inv_freq[i] = r.inv_freq[i];
    // whole tokens while they fill the GPU, shares of the heads else
    a.tokens = S < kApTokens ? (int)S : kApTokens;
    while (a.tokens > 1 && (S + a.tokens - 1) / a.tokens * batch < 3 * sm_count()) a.tokens /= 2;
    const int64_t ctas = (S + a.tokens - 1) / a.tokens * batch;
    a.shares = 1;
    while (a.shares < nkv && a.shares < 8 && ctas * a.shares * 2 <= sm_count()) a.shares *= 2;
    a.k_heads = (nkv + a.shares - 1) / a.shares;
    a.q_heads = (nq + a.shares - 1) / a.shares;
    a.q_shares = nq ? a.shares : 0;
    auto inverse = [](int d) { return (uint32_t)((1 << 20) / d + 1); };
    a.vec = (rot / 2) % 8 == 0 ? 8 : 4;
    a.per = rot / (2 * a.vec) + (D - rot + 2 * a.vec - 1) / (2 * a.vec);
    a.fit = kApThreads / a.per;
    const int side = a.tokens < a.fit ? a.tokens : a.fit;
    a.groups = a.fit / side;
    a.per_inv = inverse(a.per);
    a.tokens_inv = inverse(side);
    a.half_inv = rot ? inverse(rot / 2) : 0;
    return B2_OK;
}

template <int WIDE>
static int append_launch(AppendArgs& a, int batch, cudaStream_t s) {
    // (with several shares there are few CTAs)
    const dim3 grid((unsigned)((a.S + a.tokens - 1) / a.tokens * (WIDE ? a.q_shares + a.shares : a.shares)), (unsigned)batch);
    if (a.bf16)
        B2_TRY(a.vec == 8 ? launch(append_kernel<WIDE, 8, true>, grid, dim3(kApThreads), 0, s, true, a)
                        : launch(append_kernel<WIDE, 4, true>, grid, dim3(kApThreads), 0, s, true, a));
    else
        B2_TRY(a.vec == 8 ? launch(append_kernel<WIDE, 8, false>, grid, dim3(kApThreads), 0, s, true, a)
                        : launch(append_kernel<WIDE, 4, false>, grid, dim3(kApThreads), 0, s, true, a));
    return B2_OK;
}

template <int DP>
static cudaError_t read_launch(const ReadArgs& a, dim3 grid, cudaStream_t s) {
    return a.bf16 ? launch(kv4_read_kernel<DP, true>, grid, dim3(128), 0, s, true, a)
                  : launch(kv4_read_kernel<DP, false>, grid, dim3(128), 0, s, true, a);
}

}  // namespace b2

extern "C" int b2_paged_kv_append(const b2_paged_kv* kv, const b2_append* rows, void* stream) {
    using namespace b2;
    B2_REQUIRE(rows);
    if (rows->batch <= 0 || rows->S <= 0) return B2_OK;
    int rc = check_paged(kv, rows->num_kv_heads, rows->head_dim);
    if (rc != B2_OK) return rc;
    AppendArgs a = {};
    rc = append_args(a, *rows);
    if (rc != B2_OK) return rc;
    B2_REQUIRE((kv->num_blocks == 1 || kv->stride_block) && (kv->block_size == 1 || kv->stride_slot) &&
               (rows->num_kv_heads == 1 || kv->stride_head));
    a.kv = *kv;
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.bf16 = kv->bf16;
    return append_launch<0>(a, rows->batch, as_stream(stream));
}

extern "C" int b2_paged_kv4_append(const b2_paged_kv4* kv, const b2_append* rows, void* stream) {
    using namespace b2;
    B2_REQUIRE(rows);
    if (rows->batch <= 0 || rows->S <= 0) return B2_OK;
    const int D = rows->head_dim;
    int rc = check_paged4(kv, rows->num_kv_heads, D);
    if (rc != B2_OK) return rc;
    AppendArgs a = {};
    rc = append_args(a, *rows);
    if (rc != B2_OK) return rc;
    a.pool = static_cast<uint8_t*>(kv->pool);
    a.pool_block = kv->stride_block;
    a.head_bytes = (int64_t)(kv->block_size / 16) * kv4_tile(kv4_dp(D));
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.bf16 = kv->bf16;
    cudaStream_t s = as_stream(stream);
    return D <= 64 ? append_launch<3>(a, rows->batch, s) : D <= 128 ? append_launch<4>(a, rows->batch, s)
                                                                    : append_launch<5>(a, rows->batch, s);
}

extern "C" int b2_paged_kv4_read(const b2_paged_kv4* kv, const b2_kv_view* k_out, const b2_kv_view* v_out, const int* counts,
                                 int batch, int64_t T, int nkv, int D, void* stream) {
    using namespace b2;
    if (batch <= 0 || T <= 0) return B2_OK;
    B2_REQUIRE(k_out && v_out && k_out->data && v_out->data);
    const int rc = check_paged4(kv, nkv, D);
    if (rc != B2_OK) return rc;
    ReadArgs a = {};
    a.k = *k_out;
    a.v = *v_out;
    drop_unused(a.k, batch, T, nkv);
    drop_unused(a.v, batch, T, nkv);
    if (!rows_fit(a.k) || !rows_fit(a.v) || batch > 65535 || nkv > 65535 || T > (1 << 30)) return B2_ERR_UNSUPPORTED;
    B2_REQUIRE(rows_apart(a.k, batch, T, nkv) && rows_apart(a.v, batch, T, nkv));
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
        case 64: B2_TRY(read_launch<64>(a, grid, s)); break;
        case 96: B2_TRY(read_launch<96>(a, grid, s)); break;
        case 128: B2_TRY(read_launch<128>(a, grid, s)); break;
        case 192: B2_TRY(read_launch<192>(a, grid, s)); break;
        default: B2_TRY(read_launch<256>(a, grid, s)); break;
    }
    return B2_OK;
}
