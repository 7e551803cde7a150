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
//            per group into its own sums, then one multiply-add each.
//   outputs  o_d = sum_i (p_i s_ig) u_id + sum_i p_i m_ig: the weights times the
//            scale are the operand, split into a half and the half of what the
//            rounding left, so that it costs no accuracy beside the output's
//            own rounding; the second sum is kept in 32 bits per group.
// Queries are scaled by a power of two into the middle of the halves' range
// (bf16 ones are then exact in half), the weights times the scale by one that
// follows the largest scale seen so far, like the running max of the softmax.
//
// Layout of the products: heads are the rows of S = Q K^T and the columns of O
// = V^T P, so a lane's S values are its fragment of P as they are.  Up to 4
// heads (H = 4) stand twice in the rows: the second copy becomes the
// remainders, the other 4 columns of the same product.
//
// Split: paged_split.cuh.  Each of 4 warps streams tiles of 16 positions (kv4.cuh)
// through its own ring of shared-memory stages (cp.async).
#include <cmath>

#include "kv4.cuh"
#include "paged_split.cuh"

namespace b2 {

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
    static constexpr int T = DP <= 128 ? 2 : 1;        // tiles per warp and unit
    static constexpr int U = kPgWarps * T * 16;        // positions per unit
    static constexpr int STAGES = 2;
    static constexpr int STAGE = T * TILE;
    static constexpr int LDO = DP + 4;
    static constexpr int OFF_O = kPgWarps * STAGES * STAGE;
    static constexpr int BYTES = OFF_O + 2 * H * LDO * 4;
    static constexpr int CTAS = DP <= 128 ? (H <= 8 ? 3 : 2) : (H <= 8 ? 3 : 2);  // per SM
};

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

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
// two 32-bit numbers in a register pair: one instruction for both
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 two(uint64_t p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint32_t hmax2(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <int DP, int H, bool LIST>
__global__ void __launch_bounds__(kPgThreads, Kv4Cfg<DP, H>::CTAS) kv4_attn_kernel(const Kv4Args a) {
    using C = Kv4Cfg<DP, H>;
    constexpr int U = C::U, T = C::T, W = C::W, NG = C::NG;
    constexpr int R = H == 16 ? 2 : 1;  // rows of S per lane: head lr (H = 4: lr % 4), and head lr + 8
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ SplitShared s_split;
    __shared__ int s_vis[kPgWarps][C::STAGES][T];  // visible rows of a tile, first | end << 8; 0: none
    __shared__ float s_m[kPgWarps][16], s_l[kPgWarps][16];
    __shared__ float2 s_ml[16];
    float* s_o = reinterpret_cast<float*>(smem + C::OFF_O);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int lr = lane >> 2, lc = lane & 3;

    griddep_wait();
    griddep_launch_dependents();

    Share w;
    Place<U, LIST> at;
    if (!split_units(a, s_split, w, at)) return;
    const int r0 = w.r0, r1 = w.r1;

    // ---- producer: tiles of the next unit into a stage.  The table entries of the two next units are on their way,
    // lane t's that of tile t
    Place<U, LIST> pp = at;
    int pr = r0, pf = r0, pid[2], vis[2];  // units requested, units looked up
    int64_t off[2];
    auto lookup = [&](int k) {
        pid[k] = -1;
        vis[k] = 0;
        off[k] = 0;
        if (pf < r1) {
            const int pos = pp.s.base(pp.u) + (warp * T + lane) * 16;
            int blk = a.div.block(pos), v0 = 0, v1 = 0;
            const int slot = a.div.slot(pos, blk);
            if (lane < T) {
                if constexpr (LIST) {  // blk counts entries of the list
                    if (blk < a.listed) {
                        blk = a.blocks[((int64_t)pp.b * a.nkv + pp.kvh) * a.listed + blk];
                        if ((unsigned)blk < (unsigned)a.max_blocks) v1 = min(16, pp.s.L - blk * a.block_size - slot);
                    }
                } else if (pp.u < pp.s.ns) {
                    v1 = min(16, pp.s.s0 - pos);
                } else {
                    v0 = max(0, pp.s.lo - pos);
                    v1 = min(16, pp.s.L - pos);
                }
                if (v0 < v1) {
                    pid[k] = a.block_tables[(int64_t)pp.b * a.max_blocks + blk];
                    vis[k] = v0 | v1 << 8;
                    off[k] = pp.kvh * a.head_bytes + (int64_t)(slot >> 4) * C::TILE;
                }
            }
            ++pf;
            pp.next(a);
        }
    };
    const uint64_t policy = read_once();
    uint8_t* const ring = smem + warp * C::STAGES * C::STAGE;
    auto issue = [&](int stage) {
        if (pr < r1) {
            const bool mine = (unsigned)pid[0] < (unsigned)a.num_blocks;
            const int64_t from = (int64_t)pid[0] * a.stride_block + off[0];
            if (lane < T) s_vis[warp][stage][lane] = mine ? vis[0] : 0;
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int64_t f = __shfl_sync(~0u, from, t);
                if (__shfl_sync(~0u, (int)mine, t)) {
                    const uint8_t* src = a.pool + f + lane * 16;
                    const uint32_t dst = smem_addr(ring + stage * C::STAGE + t * C::TILE + lane * 16);
#pragma unroll
                    for (int i = 0; i < (C::TILE + 511) / 512; ++i)
                        if (i < C::TILE / 512 || lane * 16 < C::TILE % 512) cp16(dst + i * 512, src + i * 512, true, policy);
                }
            }
            ++pr;
            pid[0] = pid[1];
            vis[0] = vis[1];
            off[0] = off[1];
            lookup(1);
        }
        cp_commit();
    };
    lookup(0);
    lookup(1);
#pragma unroll
    for (int s = 0; s < C::STAGES; ++s) issue(s);

    // ---- consumer
    uint32_t qa[W][2][R][2];         // fragments of Q: word, step, row, half
    float mq[NG][R], fq[R];          // sums of q over a group, and the factor of the products, both with the log2 scale
    float o[W][2][R][4], m[R];
    uint64_t l[R], am[R][NG];        // even and odd positions apart
    int E;                           // scales of V below 2^E so far: weights are 2^(14 - E) times theirs
    auto start = [&]() {  // a new segment (or the rest of one): its queries, nothing summed yet
        const int h0 = at.head0(a), nh = at.heads(a);
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + at.b * a.ldq + (int64_t)h0 * a.D;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = (H == 4 ? lr & 3 : lr) + 8 * r;
            uint4 raw[W];
            float top = 0.f;
            auto eight = [&](const uint4& x, float (&f)[8]) {
                const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 y = a.bf16 ? make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u))
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
            // the largest |q| to 2^9 .. 2^10, times 16 still inside half; elements 2^-34 below it are lost
            const int e = top > 0.f && top < INFINITY ? min(120, 9 - ((int)(__float_as_uint(top) >> 23) - 127)) : 0;
            const float sc = pow2(e);
            fq[r] = a.scale_log2 * pow2(20) * pow2(-e);
#pragma unroll
            for (int g = 0; g < NG; ++g) mq[g][r] = 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float f[8];
                eight(raw[j], f);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += f[i], f[i] *= sc;
                mq[j / 2][r] += sum;
                qa[j][0][r][0] = f2_to_h2(f[0] * 16.f, f[4] * 16.f);
                qa[j][0][r][1] = f2_to_h2(f[1], f[5]);
                qa[j][1][r][0] = f2_to_h2(f[2] * 16.f, f[6] * 16.f);
                qa[j][1][r][1] = f2_to_h2(f[3], f[7]);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float x = mq[g][r];
                x += __shfl_xor_sync(~0u, x, 1);
                x += __shfl_xor_sync(~0u, x, 2);
                mq[g][r] = x * a.scale_log2;
                am[r][g] = 0;
            }
            m[r] = -INFINITY;
            l[r] = 0;
        }
        E = -15;  // the first tile raises it
#pragma unroll
        for (int x = 0; x < W; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[x][h][r][e] = 0.f;
    };

    start();
    int piece0 = r0;  // where the current piece of a segment began
    for (int r = r0; r < r1; ++r) {
        const int stage = (r - r0) % C::STAGES;
        cp_wait<C::STAGES - 1>();
        __syncwarp();
        int seen[T], any = 0;
#pragma unroll
        for (int t = 0; t < T; ++t) any |= seen[t] = s_vis[warp][stage][t];
        const uint8_t* const unit = ring + stage * C::STAGE;
        if (__any_sync(~0u, any)) {
            constexpr float zero[4] = {0.f, 0.f, 0.f, 0.f};
            // S of positions 2 lc, 2 lc + 1 (pp = 0) and those + 8 (pp = 1) of each tile, and the scales of V there
            uint64_t x[T][R][2];
            uint32_t vm[T][4 * NG];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const uint8_t* tile = unit + t * C::TILE;
                uint32_t meta[4 * NG];
                lds(meta, tile + 16 * DP + lc * 16 * NG);
                lds(vm[t], tile + 16 * DP + 64 * NG + lc * 16 * NG);
#pragma unroll
                for (int pp = 0; pp < 2; ++pp) {
                    float acc[NG][4];
                    uint32_t kw[W];
                    lds(kw, tile + (lr + 8 * pp) * (DP / 2) + lc * (4 * W));
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        const uint32_t u = kw[j], v = u >> 8;
                        float(&c)[4] = acc[j / 2];
                        mma_f16(c, qa[j][0][0][0], R == 2 ? qa[j][0][R - 1][0] : 0u, qa[j][0][0][1],
                                R == 2 ? qa[j][0][R - 1][1] : 0u, u & 0x000f000fu, u & 0x00f000f0u, j & 1 ? c : zero);
                        mma_f16(c, qa[j][1][0][0], R == 2 ? qa[j][1][R - 1][0] : 0u, qa[j][1][0][1],
                                R == 2 ? qa[j][1][R - 1][1] : 0u, v & 0x000f000fu, v & 0x00f000f0u, c);
                    }
                    uint64_t y[R];
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const float2 a0 = h2_to_f2(meta[2 * pp * NG + g]), a1 = h2_to_f2(meta[(2 * pp + 1) * NG + g]);
                        const uint64_t sc = pair(a0.x, a1.x), mn = pair(a0.y, a1.y);
#pragma unroll
                        for (int k = 0; k < R; ++k) {
                            const uint64_t c = pair(acc[g][2 * k], acc[g][2 * k + 1]), q2 = pair(mq[g][k], mq[g][k]);
                            x[t][k][pp] = g ? fma2(sc, c, x[t][k][pp]) : mul2(sc, c);
                            y[k] = g ? fma2(mn, q2, y[k]) : mul2(mn, q2);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < R; ++k) x[t][k][pp] = fma2(x[t][k][pp], pair(fq[k], fq[k]), y[k]);
                }
                if (seen[t] != 16 << 8) {  // rows that are not visible hold anything
                    const int v0 = seen[t] & 255, v1 = seen[t] >> 8;
#pragma unroll
                    for (int pp = 0; pp < 2; ++pp) {
                        const int p = pp * 8 + 2 * lc;
                        const bool there[2] = {p >= v0 && p < v1, p + 1 >= v0 && p + 1 < v1};
#pragma unroll
                        for (int k = 0; k < R; ++k) {
                            const float2 y = two(x[t][k][pp]);
                            x[t][k][pp] = pair(there[0] ? y.x : -INFINITY, there[1] ? y.y : -INFINITY);
                        }
#pragma unroll
                        for (int g = 0; g < 2 * NG; ++g) vm[t][2 * pp * NG + g] = there[g / NG] ? vm[t][2 * pp * NG + g] : 0u;
                    }
                }
            }
            // running max of the heads, finite, so that exp2(-inf - m) is 0, and the largest scale of V (NaN and
            // infinities do not count)
            float top[R];
            uint32_t big = vm[0][0];
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int i = 0; i < 4 * NG; ++i) big = hmax2(big, vm[t][i]);
            big = hmax2(big, __shfl_xor_sync(~0u, big, 1));
            big = hmax2(big, __shfl_xor_sync(~0u, big, 2)) & 0xffffu;
            if (big > 0x7bffu) big = 0u;
            bool moved = (int)big >= (E + 15) * 1024;
#pragma unroll
            for (int k = 0; k < R; ++k) {
                float y = -1e30f;
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const float2 a0 = two(x[t][k][0]), a1 = two(x[t][k][1]);
                    y = fmaxf(y, fmaxf(fmaxf(a0.x, a0.y), fmaxf(a1.x, a1.y)));
                }
                y = fmaxf(y, __shfl_xor_sync(~0u, y, 1));
                y = fmaxf(y, __shfl_xor_sync(~0u, y, 2));
                top[k] = fmaxf(m[k], y);
                moved |= top[k] > m[k];
            }
            if (__any_sync(~0u, moved)) {
                const int En = (int)big >= (E + 15) * 1024 ? max(1, (int)(big >> 10)) - 13 : E;
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    const float f = ex2(m[k] - top[k] + (float)(E - En));
                    m[k] = top[k];
                    l[k] = mul2(l[k], pair(f, f));
#pragma unroll
                    for (int g = 0; g < NG; ++g) am[k][g] = mul2(am[k][g], pair(f, f));
                    const float f0 = __shfl_sync(~0u, f, lc * 8), f1 = __shfl_sync(~0u, f, lc * 8 + 4);
#pragma unroll
                    for (int v = 0; v < W; ++v)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            o[v][h][k][0] *= f0, o[v][h][k][1] *= f1;
                            o[v][h][k][2] *= f0, o[v][h][k][3] *= f1;
                        }
                }
                E = En;
            }
            // the weights, 2^(14 - E) times theirs
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const float less = (float)(14 - E) - m[k];
                const uint64_t by = pair(less, less);
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int pp = 0; pp < 2; ++pp) {
                        const float2 y = two(add2(x[t][k][pp], by));
                        x[t][k][pp] = pair(ex2(y.x), ex2(y.y));
                        l[k] = add2(l[k], x[t][k][pp]);
                    }
            }
            // O += V^T (P s), group by group, with codes less 8
            const uint64_t eight = pair(8.f, 8.f);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t hi[T][R][2], lo[T][R][2];
                float less[R][4];
#pragma unroll
                for (int t = 0; t < T; ++t) {
#pragma unroll
                    for (int pp = 0; pp < 2; ++pp) {
                        const float2 a0 = h2_to_f2(vm[t][2 * pp * NG + g]), a1 = h2_to_f2(vm[t][(2 * pp + 1) * NG + g]);
                        const uint64_t sc = pair(a0.x, a1.x), mid = fma2(eight, sc, pair(a0.y, a1.y));
#pragma unroll
                        for (int k = 0; k < R; ++k) {
                            am[k][g] = fma2(x[t][k][pp], mid, am[k][g]);
                            const uint64_t ws = mul2(x[t][k][pp], sc);
                            const float2 a = two(ws);
                            hi[t][k][pp] = f2_to_h2(a.x, a.y);
                            const float2 b = h2_to_f2(hi[t][k][pp]), rest = two(add2(ws, pair(-b.x, -b.y)));
                            lo[t][k][pp] = f2_to_h2(rest.x, rest.y);
                            if (H == 4) hi[t][k][pp] = lr >= 4 ? lo[t][k][pp] : hi[t][k][pp];
                        }
                    }
                    // -8 units in the rows of either nibble: what the products of the codes start from
#pragma unroll
                    for (int k = 0; k < R; ++k) {
                        mma_f16(less[k], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, hi[t][k][0], hi[t][k][1],
                                t ? less[k] : zero);
                        if (H > 4)
                            mma_f16(less[k], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, lo[t][k][0], lo[t][k][1],
                                    less[k]);
                    }
                }
#pragma unroll
                for (int v = 2 * g; v < 2 * g + 2 && v < W; ++v) {
                    uint32_t vw[T][2];
#pragma unroll
                    for (int t = 0; t < T; ++t) lds(vw[t], unit + t * C::TILE + 8 * DP + (v * 32 + lane) * 8);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float c[R][4];
#pragma unroll
                        for (int t = 0; t < T; ++t) {
                            const uint32_t u0 = vw[t][0] >> (8 * h), u1 = vw[t][1] >> (8 * h);
                            const uint32_t b0 = u0 & 0x000f000fu, b1 = u0 & 0x00f000f0u, b2 = u1 & 0x000f000fu,
                                           b3 = u1 & 0x00f000f0u;
#pragma unroll
                            for (int k = 0; k < R; ++k) {
                                mma_f16(c[k], b0, b1, b2, b3, hi[t][k][0], hi[t][k][1], t ? c[k] : less[k]);
                                if (H > 4) mma_f16(c[k], b0, b1, b2, b3, lo[t][k][0], lo[t][k][1], c[k]);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < R; ++k) {
                            float(&d)[4] = o[v][h][k];
                            const float2 y0 = two(add2(pair(d[0], d[1]), pair(c[k][0], c[k][1])));
                            const float2 y1 = two(add2(pair(d[2], d[3]), pair(c[k][2], c[k][3])));
                            d[0] = y0.x, d[1] = y0.y, d[2] = y1.x, d[3] = y1.y;
                        }
                    }
                }
            }
        }
        __syncwarp();
        issue(stage);

        const bool done = at.u == at.s.n - 1;
        if (done || r == r1 - 1) {
            // ---- the warps meet: max and sum of each head, then the outputs, in warp order
            float mids[R][NG];
#pragma unroll
            for (int k = 0; k < R; ++k) {
                auto all = [&](uint64_t p) -> float {
                    float v = two(p).x + two(p).y;
                    v += __shfl_xor_sync(~0u, v, 1);
                    v += __shfl_xor_sync(~0u, v, 2);
                    return v;
                };
                const float total = all(l[k]);
#pragma unroll
                for (int g = 0; g < NG; ++g) mids[k][g] = all(am[k][g]);
                if (lc == 0 && lr + 8 * k < H) {
                    s_m[warp][lr + 8 * k] = m[k] + (float)(E - 14);
                    s_l[warp][lr + 8 * k] = total;
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
            float wt[R][2], mn[R][NG][2];
#pragma unroll
            for (int k = 0; k < R; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = (H == 4 ? (lc * 2 + e) & 3 : lc * 2 + e) + 8 * k;
                    float M = -1e30f;
#pragma unroll
                    for (int v = 0; v < kPgWarps; ++v) M = fmaxf(M, s_m[v][row]);
                    wt[k][e] = ex2(s_m[warp][row] - M);
#pragma unroll
                    for (int g = 0; g < NG; ++g) mn[k][g][e] = __shfl_sync(~0u, mids[k][g], (lc * 2 + e) * 4);
                }
            // rows of codes in the low nibble of a byte hold sums 16 times smaller
            const float k0 = pow2(24), k1 = pow2(20);
            if (H == 4) {
#pragma unroll
                for (int x = 0; x < W; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[x][h][0][e] += __shfl_xor_sync(~0u, o[x][h][0][e], 2);
            }
#pragma unroll 1
            for (int turn = 0; turn < kPgWarps / 2; ++turn) {
                if (warp / 2 == turn && (H > 4 || lc < 2)) {
                    float* buf = s_o + (warp % 2) * H * C::LDO;
#pragma unroll
                    for (int x = 0; x < W; ++x)
#pragma unroll
                        for (int k = 0; k < R; ++k)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float4* d = reinterpret_cast<float4*>(buf + (k * 8 + lc * 2 + e) * C::LDO + x * 32 + lr * 4);
                                const float4 old = turn ? *d : make_float4(0.f, 0.f, 0.f, 0.f);
                                const float n = mn[k][x / 2][e], f = wt[k][e];
                                *d = make_float4(fmaf(fmaf(o[x][0][k][e], k0, n), f, old.x),
                                                 fmaf(fmaf(o[x][0][k][2 + e], k1, n), f, old.y),
                                                 fmaf(fmaf(o[x][1][k][e], k0, n), f, old.z),
                                                 fmaf(fmaf(o[x][1][k][2 + e], k1, n), f, old.w));
                            }
                }
                __syncthreads();
            }
            auto sum = [&](int row, int d) -> float4 {
                const float4 v = *reinterpret_cast<const float4*>(s_o + row * C::LDO + d);
                const float4 y = *reinterpret_cast<const float4*>(s_o + (H + row) * C::LDO + d);
                return make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
            };
            finish_piece(a, s_split, w, at, r, piece0, s_ml, sum, [&](int64_t i, float4 v, float scale) {
                if (a.bf16)
                    store4<true>(a.out, i, v, scale);
                else
                    store4<false>(a.out, i, v, scale);
            });
            __syncthreads();
            at.next(a);
            piece0 = r + 1;
            if (r + 1 < r1) start();
        } else {
            at.next(a);
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

struct Kv4Sizes {
    int gs, hg, h, ctas, grid, unit;
    size_t parts, pml;  // bytes
};

template <int DP>
static void kv4_shape(Kv4Sizes& z) {
    z.ctas = z.h == 16 ? Kv4Cfg<DP, 16>::CTAS : z.h == 8 ? Kv4Cfg<DP, 8>::CTAS : Kv4Cfg<DP, 4>::CTAS;
    z.unit = Kv4Cfg<DP, 4>::U;
}
// Segments take up to 16 heads; a larger group is cut evenly.
static Kv4Sizes kv4_sizes(int nq, int nkv, int D) {
    Kv4Sizes z = {};
    const int group = nq / nkv;
    z.hg = (group + 15) / 16;
    z.gs = (group + z.hg - 1) / z.hg;
    z.h = z.gs <= 4 ? 4 : z.gs <= 8 ? 8 : 16;
    switch (kv4_dp(D)) {
        case 64: kv4_shape<64>(z); break;
        case 96: kv4_shape<96>(z); break;
        case 128: kv4_shape<128>(z); break;
        case 192: kv4_shape<192>(z); break;
        default: kv4_shape<256>(z); break;
    }
    z.grid = sm_count() * z.ctas;
    z.parts = (size_t)2 * z.grid * z.gs * D * sizeof(float);
    z.pml = (size_t)2 * z.grid * z.gs * sizeof(float2);
    return z;
}

template <int DP, int H, bool LIST>
static int kv4_launch(const Kv4Args& a, const Kv4Sizes& z, cudaStream_t s) {
    auto kern = kv4_attn_kernel<DP, H, LIST>;
    static bool done[64];
    B2_TRY(allow_smem(kern, Kv4Cfg<DP, H>::BYTES, done));
    B2_TRY(launch(kern, dim3(z.grid), dim3(kPgThreads), Kv4Cfg<DP, H>::BYTES, s, true, a));
    return B2_OK;
}
template <int DP, bool LIST>
static int kv4_dispatch(const Kv4Args& a, const Kv4Sizes& z, cudaStream_t s) {
    return z.h == 16 ? kv4_launch<DP, 16, LIST>(a, z, s)
                     : z.h == 8 ? kv4_launch<DP, 8, LIST>(a, z, s) : kv4_launch<DP, 4, LIST>(a, z, s);
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
    if (span > (1 << 30) || (int64_t)batch * nkv * z.hg * (span / z.unit + 4) > (1ll << 31) - 1)
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
