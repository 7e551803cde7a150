// kv4_attn.cu -- GQA attention of the newest token of each sequence over a
// paged K/V cache held in 4 bits (operator API paged_decode_gqa on a 4-bit
// cache), whole, with window and sinks, or over listed blocks.
//
//   out = sum_i p_i v_i,  p = softmax over the visible positions of
//   q . k_i / sqrt(D),  k_i and v_i = m + u s per group of 64 channels
//
// The work is one read of the visible rows, 72 bytes for 128 channels (4-bit
// codes, 16-bit scales): a quarter of the bytes of 16-bit rows for the same
// arithmetic, so unpacking has to stay near one instruction per code.
//
// Codes as operands.  A 4-bit code in the low bits of a half is a subnormal,
// u 2^-24, and shifted up by 4 bits u 2^-20: both exact, and the matrix
// instructions take subnormals.  So (w & 0x000f000f), (w & 0x00f000f0) and the
// same of w >> 8 are four operand registers out of a word of 8 codes with 5
// instructions and no conversion.  The factor 16 between them is put into the
// queries for K (channels whose codes come out smaller are multiplied by 16)
// and into the end for V, where it depends on the output's channel alone.
//   scores   s_i = sum_g s_ig (sum_d q_d u_id) + m_ig (sum_d q_d): one product
//            per group into its own sums, then one multiply-add each; the second
//            terms are a product too, of the scale words as they are stored with
//            the sums of q as half and remainder.
//   outputs  o_d = sum_i (p_i s_ig) (u_id - 4) + sum_i p_i (m_ig + 4 s_ig): the
//            weights times the scale are the operand, as a half and what its
//            rounding left as a half beside it: 22 bits of each, or 2^-39 of the
//            largest.  (A bare half is off by up to 2^-11 of p s |u - 4|, while
//            the m + u s that the two sums come to may vanish.)  The second sum is
//            kept in 32 bits per group.  Less 4, because the matrix instruction
//            truncates what it adds to the size of its sum: a product with a
//            constant -4 is where each unit's sums start, and with codes of 7.5
//            on average they go through zero on their way (131001 tokens, 8 heads,
//            in half: the arithmetic is off by a quarter of what the output's
//            rounding is; less 8 by up to 0.4 of it; less 5, whose own products
//            are truncated, by more than it).
// Queries are scaled by a power of two into the middle of the halves' range
// (bf16 ones are then exact in half), the weights by one that follows the
// largest scale seen so far, like the running max of the softmax.
//
// Layout of the products: positions, then channels, are the 16 rows and the
// heads the 8 columns.  Up to 4 heads (H = 4) stand twice in the columns: for the
// outputs the second copy holds the remainders, in the same product.  (Heads as the rows
// of S take twice the products and, since half of each operand's registers are
// then zeros that have to be put there, 456 instructions a tile instead of 340.)
//
// Split: paged_split.cuh.  Each of 4 warps streams tiles of 16 positions (kv4.cuh)
// through its own ring of shared-memory stages (cp.async).
//
// Measured: 32 sequences of up to 32768 tokens, 32/8 heads of 128, bf16: 227 us in a
// long run (4.5 TB/s, 69 % of a copy; floor 158; without remainders 218), 210 for one
// launch: 252 instructions a tile, 0.54 of the issue slots with 8 warps per SM, whose
// stalls are mostly the fixed wait for the instruction before.  131001 tokens,
// 64/8 heads, half: 49 us (floor 23): eight columns of heads, the remainders in
// products of their own, 295 instructions a tile, 37 pieces joined per segment.  8
// sequences of up to 4096: 17 us, 301 tokens of 14/2 heads of 64: 7 us: the chain
// length, table, rows, merge, join.
#include <cmath>
#include <type_traits>

#include "kv4.cuh"
#include "paged_split.cuh"

namespace b2 {

using namespace packed;

struct Kv4Args : SplitArgs {
    const void* q;
    int64_t ldq;
    const uint8_t* pool;
    int64_t stride_block;
    int64_t head_bytes;  // of one kv head in a block
    float scale_log2;
    int bf16;
};

// DP: padded head dim.  H: most heads of a segment, 4, 8 or 16.
template <int DP, int H>
struct Kv4Cfg {
    static constexpr int NG = kv4_groups(DP);
    static constexpr int W = DP / 32;                  // K words of a lane and row, V pieces of a lane
    static constexpr int TILE = kv4_tile(DP);
    // tiles per warp and unit: as many as there are registers for (128 channels, 4 heads, without remainders, one launch:
    // 187 us for 32 x 32768 with 4, 210 with 2 and three CTAs per SM, 250 with 1 and four)
    static constexpr int T = DP <= 128 && H <= 8 ? 4 : 2;
    static constexpr int U = kPgWarps * T * 16;        // positions per unit
    static constexpr int STAGES = DP <= 96 || T == 2 && DP == 128 ? 3 : 2;
    static constexpr int STAGE = T * TILE;
    static constexpr int LDO = DP + 4;
    static constexpr int OFF_O = kPgWarps * STAGES * STAGE;
    static constexpr int BYTES = OFF_O + 2 * H * LDO * 4;
    static constexpr int CTAS = 2;                     // per SM
};

// N consecutive 32-bit words of shared memory at an address aligned to the largest of 16, 8 and 4 bytes that divides 4 N
template <int N>
__device__ __forceinline__ void lds(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(p + 4 * i);
            w[i] = x.x, w[i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
    }
}
// d = a b + c of halves
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, const float* c) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_f16_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0, const float* c) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%8,%9,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t hmax2(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// BF16: type of q and out.
template <int DP, int H, bool BF16, bool LIST>
__global__ void __launch_bounds__(kPgThreads, Kv4Cfg<DP, H>::CTAS) kv4_attn_kernel(const Kv4Args a) {
    using C = Kv4Cfg<DP, H>;
    constexpr int U = C::U, T = C::T, W = C::W, NG = C::NG;
    constexpr bool TWO = H > 4;  // remainders of the weights in products of their own
    // and in sums of their own: added to the weights' they are truncated to the size of those (131001 tokens, 8 heads,
    // standard normal rows, in half: 8 % above the error that the output's rounding leaves, 2.5 % so, for 2 % of the time; in
    // bf16 neither shows)
    constexpr bool APART = TWO && !BF16;
    constexpr int NT = H == 16 ? 2 : 1;  // products side by side, 8 heads each
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ SplitShared s_split;
    // what is looked at once a segment or once a batch of units lies here and not in registers: the CTA's place and share,
    // each warp's place of its next batch
    __shared__ Place<U, LIST> s_at, s_next[kPgWarps];
    __shared__ Share s_share;
    __shared__ __align__(8) uint16_t s_vis[kPgWarps][C::STAGES][T];  // visible rows of a tile, first | end << 8; 0: none
    __shared__ float s_m[kPgWarps][16], s_l[kPgWarps][16];
    __shared__ float2 s_ml[16];
    float* s_o = reinterpret_cast<float*>(smem + C::OFF_O);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int lr = lane >> 2, lc = lane & 3;

    griddep_wait();
    griddep_launch_dependents();

    int r0, r1, seg0, seg_n;  // this CTA's units; the current segment's first one and how many it has
    {
        Share w;
        Place<U, LIST> at;
        if (!split_units(a, s_split, w, at)) return;
        r0 = w.r0, r1 = w.r1;
        seg0 = r0 - at.u, seg_n = at.s.n;
        if (lane == 0) s_next[warp] = at;
        if (tid == 0) s_at = at, s_share = w;
        __syncthreads();
    }

    // ---- producer: tiles of the next unit into a stage.  Where they are is looked up for up to 32 tiles of the warp at a
    // time, one per lane, a batch before it is needed (looked up unit by unit, that alone was 100 of 380 instructions a
    // tile)
    constexpr int BATCH = 32 / T;            // units of a batch, all of one segment
    int pr = r0, pf = r0;                    // units requested, units looked up
    int used = 0, count = 0, next = 0;       // units of the current batch: requested, all; units of the next batch
    int pid = -1, vis2 = 0, vis = 0;         // table entry and visible rows (first | end << 8) of the next batch; current
    int64_t off = 0, from = -1;              // in the block, next batch; in the pool (-1: nothing), current one
    auto lookup = [&]() {
        pid = -1;
        vis2 = 0;
        next = 0;
        if (pf >= r1) return;
        Place<U, LIST> pp = s_next[warp];
        next = min(BATCH, min(pp.s.n - pp.u, r1 - pf));
        const int u = pp.u + lane / T;
        if (lane < next * T) {
            const int pos = pp.s.base(u) + (warp * T + lane % T) * 16;
            int blk = a.div.block(pos), v0 = 0, v1 = 0;
            const int slot = a.div.slot(pos, blk);
            if constexpr (LIST) {  // blk counts entries of the list
                if (blk < pp.s.s0) {
                    blk = a.blocks[((int64_t)pp.b * a.nkv + pp.kvh) * a.listed + blk];
                    if ((unsigned)blk < (unsigned)a.max_blocks) v1 = min(16, pp.s.L - blk * a.block_size - slot);
                }
            } else if (u < pp.s.ns) {
                v1 = min(16, pp.s.s0 - pos);
            } else {
                v0 = max(0, pp.s.lo - pos);
                v1 = min(16, pp.s.L - pos);
            }
            if (v0 < v1) {
                pid = a.block_tables[(int64_t)pp.b * a.max_blocks + blk];
                vis2 = v0 | v1 << 8;
                off = pp.kvh * a.head_bytes + (int64_t)(slot >> 4) * C::TILE;
            }
        }
        pf += next;
        pp.u += next - 1;
        pp.next(a);
        __syncwarp();
        if (lane == 0) s_next[warp] = pp;
        __syncwarp();
    };
    const uint64_t policy = read_once();
    uint8_t* const ring = smem + warp * C::STAGES * C::STAGE;
    const uint32_t ring_at = smem_addr(ring) + lane * 16;
    const uint8_t* const pool = a.pool + lane * 16;
    auto issue = [&](int stage) {
        if (pr < r1) {
            if (used == count) {
                const bool there = (unsigned)pid < (unsigned)a.num_blocks;
                from = there ? pid * a.stride_block + off : -1;
                vis = there ? vis2 : 0;
                count = next;
                used = 0;
                lookup();
            }
            const int v = __shfl_sync(~0u, vis, used * T + lane % T);
            if (lane < T) s_vis[warp][stage][lane] = (uint16_t)v;
            int64_t f[T];
            bool all = true;
#pragma unroll
            for (int t = 0; t < T; ++t) f[t] = __shfl_sync(~0u, from, used * T + t), all = all && f[t] >= 0;
            auto copy = [&](int t) {
                const uint32_t dst = ring_at + stage * C::STAGE + t * C::TILE;
#pragma unroll
                for (int i = 0; i < (C::TILE + 511) / 512; ++i)
                    if (i < C::TILE / 512 || lane * 16 < C::TILE % 512) cp16(dst + i * 512, pool + f[t] + i * 512, true, policy);
            };
            if (all) {
#pragma unroll
                for (int t = 0; t < T; ++t) copy(t);
            } else {
#pragma unroll
                for (int t = 0; t < T; ++t)
                    if (f[t] >= 0) copy(t);
            }
            ++used;
            ++pr;
        }
        cp_commit();
    };
    lookup();
#pragma unroll
    for (int s = 0; s < C::STAGES; ++s) issue(s);

    // ---- consumer.  Lane (lr, lc) holds positions lr and lr + 8, then channels 32 x + 4 lr .. + 3, of heads 2 lc and
    // 2 lc + 1 (of each 8; H = 4: modulo 4)
    uint32_t qb[W][2][NT][2], mb[NT][2];         // fragments of Q and of its sums over the groups
    float fq[NT][2];                             // from scores as they come out of the products to base-2 logits
    float o[W][2][NT][4], m[NT][2], l[NT][2], am[NT][2][NG];
    int E;                                       // scales of V below 2^E so far: weights are 2^(14 - E) times theirs
    auto start = [&]() {  // a new segment (or the rest of one): its queries, nothing summed yet
        const Place<U, LIST>& at = s_at;
        const int h0 = at.head0(a), nh = at.heads(a);
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + at.b * a.ldq + (int64_t)h0 * a.D;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = (H == 4 ? lr & 3 : lr) + 8 * n;
            uint4 raw[W];
            float top = 0.f;
            auto eight = [&](const uint4& x, float (&f)[8]) {
                const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 y = BF16 ? make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u))
                                            : h2_to_f2(u[i]);
                    f[2 * i] = y.x, f[2 * i + 1] = y.y;
                }
            };
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int c0 = 32 * j + 8 * lc;
                raw[j] = row < nh && c0 < a.D ? *reinterpret_cast<const uint4*>(q + (int64_t)row * a.D + c0)
                                              : make_uint4(0, 0, 0, 0);
                float f[8];
                eight(raw[j], f);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]));
            }
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
            // the largest |q| to 2^5 .. 2^6: times 16, and summed over a group, still inside half.  Elements 2^-30 below
            // it are lost
            const int e = top > 0.f && top < INFINITY ? min(120, 5 - ((int)(__float_as_uint(top) >> 23) - 127)) : 0;
            const float sc = pow2(e);
            float sums[NG] = {};
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float f[8];
                eight(raw[j], f);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] *= sc, sums[j / 2] += f[i];
                qb[j][0][n][0] = f2_to_h2(f[0] * 16.f, f[4] * 16.f);
                qb[j][0][n][1] = f2_to_h2(f[1], f[5]);
                qb[j][1][n][0] = f2_to_h2(f[2] * 16.f, f[6] * 16.f);
                qb[j][1][n][1] = f2_to_h2(f[3], f[7]);
            }
            // rows 2 g + 1 of this operand meet m of group g, rows 2 g its s
            mb[n][0] = mb[n][1] = 0u;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float x = sums[g];
                x += __shfl_xor_sync(~0u, x, 1);
                x += __shfl_xor_sync(~0u, x, 2);
                const uint32_t hi = f2_to_h2(0.f, x), lo = f2_to_h2(0.f, x - h2_to_f2(hi).y);
                if (lc == g) mb[n][0] = hi, mb[n][1] = lo;
            }
            const float f = a.scale_log2 * pow2(-e);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                fq[n][h] = __shfl_sync(~0u, f, (lc * 2 + h) * 4);
                m[n][h] = -INFINITY;
                l[n][h] = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) am[n][h][g] = 0.f;
            }
        }
        E = -15;  // the first tile raises it
#pragma unroll
        for (int x = 0; x < W; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[x][h][n][e] = 0.f;
    };

    start();
    int piece0 = r0;  // where the current piece of a segment began
    int stage = 0;
    for (int r = r0; r < r1; ++r) {
        cp_wait<C::STAGES - 1>();
        __syncwarp();
        using Seen16 = std::conditional_t<T == 4, uint64_t, std::conditional_t<T == 2, uint32_t, uint16_t>>;
        const Seen16 seen = *reinterpret_cast<const Seen16*>(s_vis[warp][stage]);  // 16 bits a tile
        constexpr Seen16 kFull = (Seen16)0x1000100010001000ull;
        const uint8_t* const unit = ring + stage * C::STAGE;
        if (__any_sync(~0u, seen != 0)) {
            constexpr float zero[4] = {0.f, 0.f, 0.f, 0.f};
            float x[T][NT][4];        // scores of (lr, 2 lc), (lr, 2 lc + 1), (lr + 8, ..)
            uint32_t vm[T][2][NG];    // scale words of V at positions lr and lr + 8
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const uint8_t* tile = unit + t * C::TILE;
                const uint8_t* meta = tile + 16 * DP + kv4_slot(lr) * (4 * NG);  // (position lr + 8: two slots on)
                uint32_t kw[2][W], km[2][NG];
#pragma unroll
                for (int pp = 0; pp < 2; ++pp) {
                    lds(kw[pp], tile + (lr + 8 * pp) * (DP / 2) + lc * (4 * W));
                    lds(km[pp], meta + pp * (8 * NG));
                    lds(vm[t][pp], meta + 64 * NG + pp * (8 * NG));
                }
                const uint8_t* own = meta + (lc < NG ? lc : 0) * 4;
                const uint32_t w0 = *reinterpret_cast<const uint32_t*>(own),
                               w1 = *reinterpret_cast<const uint32_t*>(own + 8 * NG);
                float acc[NT][NG][4], y[NT][4];
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const uint32_t u0 = kw[0][j], u1 = kw[1][j], v0 = u0 >> 8, v1 = u1 >> 8;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float(&c)[4] = acc[n][j / 2];
                        mma_f16(c, u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, qb[j][0][n][0],
                                qb[j][0][n][1], j & 1 ? c : zero);
                        mma_f16(c, v0 & 0x000f000fu, v1 & 0x000f000fu, v0 & 0x00f000f0u, v1 & 0x00f000f0u, qb[j][1][n][0],
                                qb[j][1][n][1], c);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_f16_k8(y[n], w0, w1, mb[n][0], zero);
                    mma_f16_k8(y[n], w0, w1, mb[n][1], y[n]);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int pp = 0; pp < 2; ++pp) {
                        const float sc = h2_to_f2(km[pp][g]).x;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int i = 2 * pp + h;
                                x[t][n][i] = g ? fmaf(sc, acc[n][g][i], x[t][n][i]) : sc * acc[n][g][i];
                            }
                    }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][n][i] = fmaf(x[t][n][i], 1048576.f, y[n][i]);
            }
            if (seen != kFull) {  // rows that are not visible hold anything
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const int v0 = (int)(seen >> (16 * t)) & 255, v1 = (int)(seen >> (16 * t + 8)) & 255;
#pragma unroll
                    for (int pp = 0; pp < 2; ++pp) {
                        const bool there = lr + 8 * pp >= v0 && lr + 8 * pp < v1;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int h = 0; h < 2; ++h) x[t][n][2 * pp + h] = there ? x[t][n][2 * pp + h] : -INFINITY;
#pragma unroll
                        for (int g = 0; g < NG; ++g) vm[t][pp][g] = there ? vm[t][pp][g] : 0u;
                    }
                }
            }
            // does a score pass its head's running max, or a scale of V 2^E?  (NaN and infinities do not count)
            float top[NT][2];
            uint32_t big = vm[0][0][0];
            bool moved = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float y = fmaxf(x[0][n][h], x[0][n][2 + h]);
#pragma unroll
                    for (int t = 1; t < T; ++t) y = fmaxf(y, fmaxf(x[t][n][h], x[t][n][2 + h]));
                    top[n][h] = y;
                    moved |= y > m[n][h];
                }
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i) big = hmax2(big, vm[t][i / NG][i % NG]);
            big &= 0xffffu;
            if (big > 0x7bffu) big = 0u;
            moved |= (int)big >= (E + 15) * 1024;
            if (__any_sync(~0u, moved)) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) big = max(big, __shfl_xor_sync(~0u, big, d));
                const int En = (int)big >= (E + 15) * 1024 ? max(1, (int)(big >> 10)) - 13 : E;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float y = fmaxf(m[n][h], top[n][h]);
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) y = fmaxf(y, __shfl_xor_sync(~0u, y, d));
                        const float f = ex2(fmaf(m[n][h] - y, fq[n][h], (float)(E - En)));
                        m[n][h] = y;
                        l[n][h] *= f;
#pragma unroll
                        for (int g = 0; g < NG; ++g) am[n][h][g] *= f;
#pragma unroll
                        for (int v = 0; v < W; ++v)
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                o[v][k][n][h] *= f;
                                o[v][k][n][2 + h] *= f;
                            }
                    }
                E = En;
            }
            // the weights, 2^(14 - E) times theirs
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float less = fmaf(-m[n][h], fq[n][h], (float)(14 - E));
#pragma unroll
                    for (int t = 0; t < T; ++t)
#pragma unroll
                        for (int pp = 0; pp < 2; ++pp) {
                            float& p = x[t][n][2 * pp + h];
                            p = ex2(fmaf(p, fq[n][h], less));
                            l[n][h] += p;
                        }
                }
            // O += V^T (P s), group by group, with codes less 4; the weights as half and remainder, turned from
            // (position, head) to (head, position) pairs
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t hi[T][NT][2], lo[T][NT][2];
                float less[APART ? 2 * NT : NT][4];  // (the remainders' behind)
#pragma unroll
                for (int t = 0; t < T; ++t) {
#pragma unroll
                    for (int pp = 0; pp < 2; ++pp) {
                        const float2 sm = h2_to_f2(vm[t][pp][g]);
                        const float mid = fmaf(4.f, sm.x, sm.y);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const float p0 = x[t][n][2 * pp], p1 = x[t][n][2 * pp + 1];
                            am[n][0][g] = fmaf(p0, mid, am[n][0][g]);
                            am[n][1][g] = fmaf(p1, mid, am[n][1][g]);
                            const float w0 = p0 * sm.x, w1 = p1 * sm.x;
                            const uint32_t u = f2_to_h2(w0, w1);
                            // (in one multiply-add of halves and a 32-bit number each)
                            const uint32_t r = f2_to_h2(fma_f16_f32<0>(u, 0xbc00bc00u, w0), fma_f16_f32<1>(u, 0xbc00bc00u, w1));
                            hi[t][n][pp] = transpose8x8(TWO || lc < 2 ? u : r);
                            if constexpr (TWO) lo[t][n][pp] = transpose8x8(r);
                        }
                    }
                    // -4 units in the rows of either nibble: what the products of the codes start from
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_f16(less[n], 0x80048004u, 0x80408040u, 0x80048004u, 0x80408040u, hi[t][n][0], hi[t][n][1],
                                t ? less[n] : zero);
                        if constexpr (TWO) {
                            float(&d)[4] = less[APART ? NT + n : n];
                            mma_f16(d, 0x80048004u, 0x80408040u, 0x80048004u, 0x80408040u, lo[t][n][0], lo[t][n][1],
                                    APART && t == 0 ? zero : d);
                        }
                    }
                }
#pragma unroll
                for (int v = 2 * g; v < 2 * g + 2 && v < W; ++v) {
                    uint32_t vw[T][2];
#pragma unroll
                    for (int t = 0; t < T; ++t) lds(vw[t], unit + t * C::TILE + 8 * DP + (v * 32 + lane) * 8);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float c[APART ? 2 * NT : NT][4];
#pragma unroll
                        for (int t = 0; t < T; ++t) {
                            const uint32_t u0 = vw[t][0] >> (8 * k), u1 = vw[t][1] >> (8 * k);
                            const uint32_t b0 = u0 & 0x000f000fu, b1 = u0 & 0x00f000f0u, b2 = u1 & 0x000f000fu,
                                           b3 = u1 & 0x00f000f0u;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                mma_f16(c[n], b0, b1, b2, b3, hi[t][n][0], hi[t][n][1], t ? c[n] : less[n]);
                                if constexpr (TWO) {
                                    constexpr int r = APART ? NT : 0;
                                    mma_f16(c[r + n], b0, b1, b2, b3, lo[t][n][0], lo[t][n][1],
                                            APART && t == 0 ? less[r + n] : c[r + n]);
                                }
                            }
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float(&d)[4] = o[v][k][n];
                            if constexpr (APART) {
                                const float2 z0 = two(add2(pair(c[n][0], c[n][1]), pair(c[NT + n][0], c[NT + n][1])));
                                const float2 z1 = two(add2(pair(c[n][2], c[n][3]), pair(c[NT + n][2], c[NT + n][3])));
                                c[n][0] = z0.x, c[n][1] = z0.y, c[n][2] = z1.x, c[n][3] = z1.y;
                            }
                            const float2 y0 = two(add2(pair(d[0], d[1]), pair(c[n][0], c[n][1])));
                            const float2 y1 = two(add2(pair(d[2], d[3]), pair(c[n][2], c[n][3])));
                            d[0] = y0.x, d[1] = y0.y, d[2] = y1.x, d[3] = y1.y;
                        }
                    }
                }
            }
        }
        __syncwarp();
        issue(stage);
        stage = stage + 1 == C::STAGES ? 0 : stage + 1;

        if (r - seg0 == seg_n - 1 || r == r1 - 1) {
            // ---- the warps meet: max and sum of each head, then the outputs, in warp order
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    auto all = [&](float v) -> float {
                        v += __shfl_xor_sync(~0u, v, 4);
                        v += __shfl_xor_sync(~0u, v, 8);
                        return v + __shfl_xor_sync(~0u, v, 16);
                    };
                    l[n][h] = all(l[n][h]);
#pragma unroll
                    for (int g = 0; g < NG; ++g) am[n][h][g] = all(am[n][h][g]);
                    if (lr == 0 && lc * 2 + h + 8 * n < H) {
                        s_m[warp][lc * 2 + h + 8 * n] = fmaf(m[n][h], fq[n][h], (float)(E - 14));
                        s_l[warp][lc * 2 + h + 8 * n] = l[n][h];
                    }
                }
            __syncthreads();
            if (tid < H) {
                float M = -1e30f, Ls = 0.f;
#pragma unroll
                for (int v = 0; v < kPgWarps; ++v) M = fmaxf(M, s_m[v][tid]);
#pragma unroll
                for (int v = 0; v < kPgWarps; ++v) Ls = fmaf(s_l[v][tid], ex2(s_m[v][tid] - M), Ls);
                s_ml[tid] = make_float2(M, Ls);
            }
            float wt[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = (H == 4 ? (lc * 2 + h) & 3 : lc * 2 + h) + 8 * n;
                    float M = -1e30f;
#pragma unroll
                    for (int v = 0; v < kPgWarps; ++v) M = fmaxf(M, s_m[v][row]);
                    wt[n][h] = ex2(s_m[warp][row] - M);
                }
            // rows of codes in the low nibble of a byte hold sums 16 times smaller
            constexpr float k0 = 16777216.f, k1 = 1048576.f;
            if (H == 4) {
#pragma unroll
                for (int x = 0; x < W; ++x)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[x][k][0][e] += __shfl_xor_sync(~0u, o[x][k][0][e], 2);
            }
#pragma unroll 1
            for (int turn = 0; turn < kPgWarps / 2; ++turn) {
                if (warp / 2 == turn && (H > 4 || lc < 2)) {
                    float* buf = s_o + (warp % 2) * H * C::LDO;
#pragma unroll
                    for (int x = 0; x < W; ++x)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float4* d = reinterpret_cast<float4*>(buf + (n * 8 + lc * 2 + h) * C::LDO + x * 32 + lr * 4);
                                const float4 old = turn ? *d : make_float4(0.f, 0.f, 0.f, 0.f);
                                const float mid = am[n][h][x / 2], f = wt[n][h];
                                *d = make_float4(fmaf(fmaf(o[x][0][n][h], k0, mid), f, old.x),
                                                 fmaf(fmaf(o[x][0][n][2 + h], k1, mid), f, old.y),
                                                 fmaf(fmaf(o[x][1][n][h], k0, mid), f, old.z),
                                                 fmaf(fmaf(o[x][1][n][2 + h], k1, mid), f, old.w));
                            }
                }
                __syncthreads();
            }
            auto sum = [&](int row, int d) -> float4 {
                const float4 v = *reinterpret_cast<const float4*>(s_o + row * C::LDO + d);
                const float4 y = *reinterpret_cast<const float4*>(s_o + (H + row) * C::LDO + d);
                return make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
            };
            Place<U, LIST> at = s_at;
            Share w = s_share;
            at.u = r - seg0;
            finish_piece(a, s_split, w, at, r, piece0, s_ml, sum, [&](int64_t i, float4 v, float scale) {
                store4<BF16>(a.out, i, v, scale);
            });
            __syncthreads();
            if (r + 1 < r1) {
                at.next(a);
                seg0 = piece0 = r + 1;
                seg_n = at.s.n;
                if (tid == 0) s_at = at;
                __syncthreads();
                start();
            }
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

struct Kv4Sizes {
    int gs, hg, h, grid;
    size_t parts, pml;  // bytes
};

// Segments take up to 16 heads, 8 above 128 channels (the outputs of 16 would not fit the registers); a larger group is
// cut evenly.
static Kv4Sizes kv4_sizes(int nq, int nkv, int D) {
    Kv4Sizes z = {};
    const int group = nq / nkv, most = D <= 128 ? 16 : 8;
    z.hg = (group + most - 1) / most;
    z.gs = (group + z.hg - 1) / z.hg;
    z.h = z.gs <= 4 ? 4 : z.gs <= 8 ? 8 : 16;
    z.grid = sm_count() * Kv4Cfg<128, 4>::CTAS;
    z.parts = (size_t)2 * z.grid * z.gs * D * sizeof(float);
    z.pml = (size_t)2 * z.grid * z.gs * sizeof(float2);
    return z;
}

template <int DP, int H, bool BF16, bool LIST>
static int kv4_launch(const Kv4Args& a, const Kv4Sizes& z, cudaStream_t s) {
    auto kern = kv4_attn_kernel<DP, H, BF16, LIST>;
    static bool done[64];
    B2_TRY(allow_smem(kern, Kv4Cfg<DP, H>::BYTES, done));
    B2_TRY(launch(kern, dim3(z.grid), dim3(kPgThreads), Kv4Cfg<DP, H>::BYTES, s, true, a));
    return B2_OK;
}
template <int DP, int H, bool LIST>
static int kv4_dispatch(const Kv4Args& a, const Kv4Sizes& z, cudaStream_t s) {
    return a.bf16 ? kv4_launch<DP, H, true, LIST>(a, z, s) : kv4_launch<DP, H, false, LIST>(a, z, s);
}
template <int DP, bool LIST>
static int kv4_dispatch(const Kv4Args& a, const Kv4Sizes& z, cudaStream_t s) {
    if constexpr (DP <= 128)
        if (z.h == 16) return kv4_dispatch<DP, 16, LIST>(a, z, s);
    return z.h == 8 ? kv4_dispatch<DP, 8, LIST>(a, z, s) : kv4_dispatch<DP, 4, LIST>(a, z, s);
}
template <bool LIST>
static int kv4_dispatch(const Kv4Args& a, const Kv4Sizes& z, cudaStream_t s) {
    switch (kv4_dp(a.D)) {
        case 64: return kv4_dispatch<64, LIST>(a, z, s);
        case 96: return kv4_dispatch<96, LIST>(a, z, s);
        case 128: return kv4_dispatch<128, LIST>(a, z, s);
        case 192: return kv4_dispatch<192, LIST>(a, z, s);
        default: return kv4_dispatch<256, LIST>(a, z, s);
    }
}

}  // namespace b2

extern "C" size_t b2_kv4_tile_bytes(int D) {
    return D <= 0 || D > 256 || (D & 7) ? 0 : b2::kv4_tile(b2::kv4_dp(D));
}

extern "C" size_t b2_paged_kv4_decode_workspace_bytes(int nq, int nkv, int D) {
    if (nq <= 0 || nkv <= 0 || nq % nkv || D <= 0 || D > 256) return 0;
    const b2::Kv4Sizes z = b2::kv4_sizes(nq, nkv, D);
    return z.parts + z.pml;
}

extern "C" int b2_paged_kv4_decode_gqa(const void* q, int64_t ldq, const b2_paged_kv4* kv, const int* blocks,
                                       int listed, void* out, int batch, int nq, int nkv, int D, int window, int sinks,
                                       b2_workspace* ws, void* stream) {
    using namespace b2;
    if (batch <= 0) return B2_OK;
    B2_REQUIRE(q && out && nq > 0 && nkv > 0 && nq % nkv == 0 && window >= 0 && sinks >= 0);
    B2_REQUIRE(!blocks || (listed > 0 && window == 0));
    const int rc = check_paged4(kv, nkv, D);
    if (rc != B2_OK) return rc;
    if (!aligned16(q) || !aligned16(out) || (ldq & 7)) return B2_ERR_UNSUPPORTED;
    const Kv4Sizes z = kv4_sizes(nq, nkv, D);
    const int64_t span = (int64_t)(blocks ? listed : kv->max_blocks) * kv->block_size;
    // positions and units are counted in 32 bits
    if (span > (1 << 30) || (int64_t)batch * nkv * z.hg * (span / Kv4Cfg<256, 4>::U + 4) > (1ll << 31) - 1)
        return B2_ERR_UNSUPPORTED;
    Kv4Args a = {};
    a.q = q;
    a.ldq = ldq;
    a.pool = static_cast<const uint8_t*>(kv->pool);
    a.stride_block = kv->stride_block;
    a.head_bytes = (int64_t)(kv->block_size / 16) * kv4_tile(kv4_dp(D));
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.div = block_div(kv->block_size);
    a.blocks = blocks;
    a.listed = listed;
    a.out = out;
    a.batch = batch;
    a.nq = nq;
    a.nkv = nkv;
    a.D = D;
    a.group = nq / nkv;
    a.hg = z.hg;
    a.gs = z.gs;
    a.window = window;
    a.sinks = sinks;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)D);
    a.bf16 = kv->bf16;
    if (ws) {
        if (ws->bytes < z.parts + z.pml || z.grid > kWsCounters) return B2_ERR_WORKSPACE;
        a.parts = static_cast<float*>(ws->ptr);
        a.pml = reinterpret_cast<float2*>(static_cast<uint8_t*>(ws->ptr) + z.parts);
        a.counters = ws->counters;
    }
    cudaStream_t s = as_stream(stream);
    return blocks ? kv4_dispatch<true>(a, z, s) : kv4_dispatch<false>(a, z, s);
}
