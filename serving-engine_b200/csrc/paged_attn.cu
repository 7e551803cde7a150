// paged_attn.cu -- GQA attention of the newest token of each sequence over a
// paged K/V cache, with window, sinks and accumulated attention weights
// (operator API paged_decode_gqa).
//
//   out = sum_i p_i v_i,  p = softmax over the visible positions of
//   q . k_i / sqrt(D);  score_i += sum over the group's heads of p_i
//
// The work is one read of the visible K and V rows: 4 D bytes per (position,
// kv head) for up to 4 D G flops (G heads of the group), so HBM bounds it.
//
// Split: paged_split.cuh, segments of up to 16 heads.
//
// Inside a CTA each of 4 warps streams its own quarter of every unit through
// its own ring of shared-memory stages (cp.async, no barrier between warps),
// with its own running max and sum; the warps meet once per segment.  Rows
// come through the block table 16 bytes per lane, rows that are not visible
// are filled with zeros and never read.  Products on mma.sync m16n8k16, fp32
// accumulation: far below its rate at this memory speed, and it takes any row
// addresses, where tensor-map copies would need one map per layout and whole
// swizzle atoms per block.  Positions, then head-dim elements, are the 16 rows
// of a product and the heads its 8 columns (S = K Q^T, O = V^T P): heads as
// rows would leave half of every product empty, at twice the products (and the
// chip is at its power limit here: 566 us for 32 x 32768 in a long run of graph
// replays, 528 this way).  P is split into a 16-bit value and a 16-bit remainder, so that
// rounding the weights costs no accuracy next to the output's own rounding.
//
// Weights (scores): the logits go to the workspace as they are computed (G
// floats beside the 4 D bytes of a position's rows, written and read once), and
// a second kernel turns them into weights with the joined max and sum, instead
// of reading K again.  (An L2 policy that keeps the logits until then gains 4 us
// of 117 for 131001 tokens, but they stay there after the call: a tensor of 96
// MB that is read over and over next takes 31 us a time instead of 25.)
//
// Measured (4 D bytes per visible position and kv head, and the scores' 8),
// called in a row: 32 sequences of up to 32768, 8 kv heads of 128: 550 us, 6.7
// TB/s (the measured copy is 6.47; 521 us in the shortest graph replay, 537 in
// most); window 1024 of 16384: 27 us, 5.0 TB/s; 8 of up to 4096 with weights: 28
// us, 3.9 TB/s; one of 131001 with weights: 119 us, 4.6 TB/s; 301 tokens of a
// small model: 6.5 us.  The short ones are bound by the chain length -> tables
// -> rows -> merge -> join (8.5 k cycles before the first product, 3 to 6 k
// after the last).  A head_dim below 64, 128 or 256 costs what that costs (8 of
// up to 4096: 26 us at 80 and 96, 25 at 128, 46 at 192, 45 at 256).
#include <cmath>

#include "paged_split.cuh"

namespace b2 {

constexpr int kPgStages = 3;
constexpr int kPgScoreThreads = 128;

struct PagedArgs : SplitArgs {
    const void* q;
    int64_t ldq;
    b2_paged_kv kv;
    float* scores;
    float scale_log2;
    int whole;      // blocks are whole groups of 16 positions
    float* logits;  // [batch][nq][cap]; scores only
    int cap;
};

// DP: head dim rounded up to 64, 128 or 256.  GH: more than 8 heads a segment.
template <int DP, bool GH>
struct PagedCfg {
    static constexpr int TP = DP == 64 ? 32 : 16;     // positions per warp and unit
    static constexpr int U = kPgWarps * TP;           // positions per unit
    static constexpr int ROW = DP * 2;                // bytes of a row
    static constexpr int CH = DP / 8;                 // 16-byte chunks of a row
    static constexpr int STAGE = 2 * TP * ROW;        // K and V rows of a warp's tile
    static constexpr int G = GH ? 16 : 8;             // heads of a segment, a row each in the warps' meeting
    static constexpr int NB = GH ? 1 : 2;             // buffers of the warps' meeting
    static constexpr int LDO = DP + 4;
    static constexpr int OFF_O = kPgWarps * kPgStages * STAGE;
    static constexpr int BYTES = OFF_O + NB * G * LDO * 4;
    static constexpr int CTAS = DP == 256 ? 1 : 2;    // per SM
};

// (a, b) as 16-bit values and what the rounding left, again in 16 bits
template <bool BF16>
__device__ __forceinline__ void split16(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack16<BF16>(a, b);
    float2 f;
    if constexpr (BF16) {
        f.x = __uint_as_float(hi << 16);
        f.y = __uint_as_float(hi & 0xffff0000u);
    } else {
        f = h2_to_f2(hi);
    }
    lo = pack16<BF16>(a - f.x, b - f.y);
}

template <int DP, bool GH, bool BF16, bool LIST>
__global__ void __launch_bounds__(kPgThreads, PagedCfg<DP, GH>::CTAS) paged_attn_kernel(const PagedArgs a) {
    using C = PagedCfg<DP, GH>;
    constexpr int U = C::U, TP = C::TP, G = C::G;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ SplitShared s_split;
    __shared__ uint32_t s_there[kPgWarps][kPgStages];
    __shared__ float s_m[kPgWarps][16], s_l[kPgWarps][16];
    __shared__ float2 s_ml[16];
    float* s_o = reinterpret_cast<float*>(smem + C::OFF_O);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // Chunks of a row past D are never copied, but the products read them: zeros, whatever an earlier kernel left
    // there.  A warp clears those of its own ring, which no other warp touches and its copies never write.
    if (a.D < DP) {
        const int pads = C::CH - a.D / 8;
        uint8_t* rows = smem + warp * kPgStages * C::STAGE;
        for (int i = lane; i < kPgStages * 2 * TP * pads; i += 32) {
            const int r = i / pads, ch = a.D / 8 + i - r * pads;
            *reinterpret_cast<uint4*>(rows + r * C::ROW + ((ch ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
    }
    griddep_wait();
    griddep_launch_dependents();

    // ---- this CTA's range of units, and the place where it starts
    Share w;
    Place<U, LIST> at;
    if (!split_units(a, s_split, w, at)) return;
    const int r0 = w.r0, r1 = w.r1;

    // ---- producer: rows of the next unit into a stage.  The table entries of the two next units are on their way:
    // lane l's is that of row l % TP of the unit (-1: not visible), with the rest of the row's offset
    Place<U, LIST> pp = at;
    int pr = r0, pf = r0, pid[2];  // units requested, units looked up
    int64_t add[2];
    auto lookup = [&](int k) {
        pid[k] = -1;
        if (pf < r1) {
            const int pos = pp.s.base(pp.u) + warp * TP + (lane & (TP - 1));
            int blk = a.div.block(pos);
            const int slot = a.div.slot(pos, blk);
            bool sees = pp.s.sees(pp.u, pos);
            if constexpr (LIST) {  // blk counts entries of the list
                sees = false;
                if (blk < pp.s.s0) {
                    blk = a.blocks[((int64_t)pp.b * a.nkv + pp.kvh) * a.listed + blk];
                    sees = (unsigned)blk < (unsigned)a.max_blocks && slot < pp.s.L - blk * a.block_size;
                }
            }
            if (sees) pid[k] = a.block_tables[(int64_t)pp.b * a.max_blocks + blk];
            add[k] = (int64_t)slot * a.kv.stride_slot + (int64_t)pp.kvh * a.kv.stride_head;
            ++pf;
            pp.next(a);
        }
    };
    const uint64_t policy = read_once();
    const uint32_t ring = smem_addr(smem) + warp * kPgStages * C::STAGE;
    const int chunk = lane % C::CH;
    auto issue = [&](int stage) {
        if (pr < r1) {
            const bool there = (unsigned)pid[0] < (unsigned)a.num_blocks;
            const int64_t off = (int64_t)pid[0] * a.kv.stride_block + add[0];
            const uint32_t mask = __ballot_sync(~0u, there);
            if (lane == 0) s_there[warp][stage] = mask;
            const uint32_t st = ring + stage * C::STAGE;
            const uint16_t *K = static_cast<const uint16_t*>(a.kv.k), *V = static_cast<const uint16_t*>(a.kv.v);
            if (mask == ~0u && a.whole && a.D == DP) {
                // every 16 rows are consecutive slots of one block: one address and a stride
                constexpr int STEP = 32 / C::CH;  // rows per instruction
#pragma unroll
                for (int t = 0; t < TP / 16; ++t) {
                    const int64_t o0 = __shfl_sync(~0u, off, 16 * t) + (lane / C::CH) * a.kv.stride_slot + chunk * 8;
                    const uint16_t *kp = K + o0, *vp = V + o0;
                    uint32_t d = st + (16 * t + lane / C::CH) * C::ROW;
#pragma unroll
                    for (int i = 0; i < 16 / STEP; ++i) {
                        const uint32_t x = d + i * STEP * C::ROW + ((chunk ^ ((lane / C::CH + i * STEP) & 7)) << 4);
                        cp16(x, kp, true, policy);
                        cp16(x + TP * C::ROW, vp, true, policy);
                        kp += STEP * a.kv.stride_slot;
                        vp += STEP * a.kv.stride_slot;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < TP * C::CH / 32; ++i) {
                    const int r = lane / C::CH + i * (32 / C::CH);
                    const int64_t ro = __shfl_sync(~0u, off, r);
                    const bool ok = (mask >> r) & 1;
                    if (chunk * 8 < a.D) {
                        const uint32_t d = st + r * C::ROW + ((chunk ^ (r & 7)) << 4);
                        const int64_t so = ok ? ro + chunk * 8 : 0;
                        cp16(d, K + so, ok, policy);
                        cp16(d + TP * C::ROW, V + so, ok, policy);
                    }
                }
            }
            ++pr;
            pid[0] = pid[1];
            add[0] = add[1];
            lookup(1);
        }
        cp_commit();
    };
    add[0] = add[1] = 0;
    lookup(0);
    lookup(1);
#pragma unroll
    for (int s = 0; s < kPgStages - 1; ++s) issue(s);

    // ---- consumer.  Positions are the rows of S, head-dim elements those of O: lane (lr, lc) holds positions lr and
    // lr + 8, then outputs lr and lr + 8, of heads 2 lc and 2 lc + 1 (and those + 8)
    constexpr int NT = GH ? 2 : 1;  // 8 heads each
    const int lr = lane >> 2, lc = lane & 3;
    uint32_t qb[DP / 16][NT][2];
    float o[DP / 16][NT][4], m[NT][2], l[NT][2];
    float* logits = nullptr;  // where this lane's of the segment go
    auto start = [&]() {  // a new segment (or the rest of one): its queries, nothing summed yet
        const int h0 = at.head0(a), nh = at.heads(a);
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + at.b * a.ldq + (int64_t)h0 * a.D;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = n * 8 + lr, col = kk * 16 + e * 8 + lc * 2;
                    qb[kk][n][e] =
                        row < nh && col < a.D ? *reinterpret_cast<const uint32_t*>(q + (int64_t)row * a.D + col) : 0u;
                }
#pragma unroll
        for (int x = 0; x < DP / 16; ++x)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[x][n][e] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[n][e] = -INFINITY;
                l[n][e] = 0.f;
            }
        if (a.logits) logits = a.logits + ((int64_t)at.b * a.nq + h0 + lc * 2) * a.cap + warp * TP + lr;
    };

    start();
    int piece0 = r0;  // where the current piece of a segment began
    for (int r = r0; r < r1; ++r) {
        const int stage = (r - r0) % kPgStages;
        cp_wait<kPgStages - 2>();
        __syncwarp();
        const uint32_t there = s_there[warp][stage];
        const uint32_t st = ring + stage * C::STAGE;
        if (there) {
#pragma unroll
            for (int t = 0; t < TP / 16; ++t) {
                // S = K Q^T: 16 positions x 8 (or 16) heads, even and odd steps of the head dim in sums of their own
                float s[NT][4] = {}, s2[NT][4] = {};
                const uint32_t kb = st + t * 16 * C::ROW, vb = kb + TP * C::ROW;
                const int mi = lane >> 3, mr = lane & 7;
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    uint32_t kf[4];
                    ldsm4(kf, kb + ((mi & 1) * 8 + mr) * C::ROW + (((kk * 2 + (mi >> 1)) ^ mr) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float* c = kk & 1 ? s2[n] : s[n];
                        mma16816<BF16>(c[0], c[1], c[2], c[3], kf[0], kf[1], kf[2], kf[3], qb[kk][n][0], qb[kk][n][1]);
                    }
                }
                const uint32_t tm = there >> (t * 16);
                const bool see[2] = {((tm >> lr) & 1) != 0, ((tm >> (lr + 8)) & 1) != 0};
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = see[e >> 1] ? (s[n][e] + s2[n][e]) * a.scale_log2 : -INFINITY;
                if (a.logits) {
                    const int nh = at.heads(a);
                    float* lg = logits + at.u * U + t * 16;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (n * 8 + lc * 2 + (e & 1) < nh) lg[(int64_t)(n * 8 + (e & 1)) * a.cap + (e >> 1) * 8] = s[n][e];
                }
                // running max of the heads; finite, so that exp2(-inf - m) is 0
                float top[NT][2];
                bool moved = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(s[n][e], s[n][2 + e]);
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
                        top[n][e] = fmaxf(fmaxf(m[n][e], x), -1e30f);
                        moved |= top[n][e] > m[n][e];
                    }
                if (__any_sync(~0u, moved)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float f = ex2(m[n][e] - top[n][e]);
                            m[n][e] = top[n][e];
                            l[n][e] *= f;
#pragma unroll
                            for (int x = 0; x < DP / 16; ++x) {
                                o[x][n][e] *= f;
                                o[x][n][2 + e] *= f;
                            }
                        }
                }
                // the weights as value + remainder, turned from (position, head) to (head, position) pairs
                uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float p0 = ex2(s[n][2 * k] - m[n][0]), p1 = ex2(s[n][2 * k + 1] - m[n][1]);
                        l[n][0] += p0;
                        l[n][1] += p1;
                        split16<BF16>(p0, p1, ph[n][k], pl[n][k]);
                        ph[n][k] = transpose8x8(ph[n][k]);
                        pl[n][k] = transpose8x8(pl[n][k]);
                    }
                // O += V^T P
#pragma unroll
                for (int x = 0; x < DP / 16; ++x) {
                    uint32_t vf[4];
                    ldsm4t(vf, vb + ((mi >> 1) * 8 + mr) * C::ROW + (((x * 2 + (mi & 1)) ^ mr) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float* c = o[x][n];
                        mma16816<BF16>(c[0], c[1], c[2], c[3], vf[0], vf[1], vf[2], vf[3], ph[n][0], ph[n][1]);
                        mma16816<BF16>(c[0], c[1], c[2], c[3], vf[0], vf[1], vf[2], vf[3], pl[n][0], pl[n][1]);
                    }
                }
            }
        }
        __syncwarp();
        issue((r - r0 + kPgStages - 1) % kPgStages);

        const bool done = at.u == at.s.n - 1;
        if (done || r == r1 - 1) {
            // ---- the warps meet: max and sum of each head, then the outputs, in warp order
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    l[n][e] += __shfl_xor_sync(~0u, l[n][e], 4);
                    l[n][e] += __shfl_xor_sync(~0u, l[n][e], 8);
                    l[n][e] += __shfl_xor_sync(~0u, l[n][e], 16);
                    if (lr == 0) {
                        s_m[warp][n * 8 + lc * 2 + e] = m[n][e];
                        s_l[warp][n * 8 + lc * 2 + e] = l[n][e];
                    }
                }
            __syncthreads();
            float wt[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = n * 8 + lc * 2 + e;
                    float M = -1e30f;
#pragma unroll
                    for (int v = 0; v < kPgWarps; ++v) M = fmaxf(M, s_m[v][row]);
                    wt[n][e] = ex2(s_m[warp][row] - M);
                    if (warp == 0 && lr == 0) {
                        float Ls = 0.f;
#pragma unroll
                        for (int v = 0; v < kPgWarps; ++v) Ls = fmaf(s_l[v][row], ex2(s_m[v][row] - M), Ls);
                        s_ml[row] = make_float2(M, Ls);
                    }
                }
#pragma unroll 1
            for (int turn = 0; turn < kPgWarps / C::NB; ++turn) {
                if (warp / C::NB == turn) {
                    float* buf = s_o + (warp % C::NB) * G * C::LDO;
#pragma unroll
                    for (int x = 0; x < DP / 16; ++x)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float* d = buf + (n * 8 + lc * 2 + (e & 1)) * C::LDO + x * 16 + lr + (e >> 1) * 8;
                                *d = fmaf(o[x][n][e], wt[n][e & 1], turn ? *d : 0.f);
                            }
                }
                __syncthreads();
            }
            auto sum = [&](int row, int d) -> float4 {
                float4 v = *reinterpret_cast<const float4*>(s_o + row * C::LDO + d);
                if (C::NB == 2) {
                    const float4 x = *reinterpret_cast<const float4*>(s_o + (G + row) * C::LDO + d);
                    v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
                }
                return v;
            };
            finish_piece(a, s_split, w, at, r, piece0, s_ml, sum,
                         [&](int64_t i, float4 v, float scale) { store4<BF16>(a.out, i, v, scale); });
            __syncthreads();
            at.next(a);
            piece0 = r + 1;
            if (r + 1 < r1) start();
        } else {
            at.next(a);
        }
    }
}

// One thread per 4 stored logit columns: the weights their positions get from
// the group's heads, in head order, onto their scores.  Slots and scores are
// read while the kernel before still runs (8 x 4096: 27.0 us with, 28.2
// without; one sequence of 4000: 13.0 and 14.2), 4 heads at a time keep 8 CTAs
// on an SM (131001 tokens: 116.4 us; 8 heads at a time and 5 CTAs: 117.3).
template <int U>
__global__ void __launch_bounds__(kPgScoreThreads, 8) paged_scores_kernel(const PagedArgs a) {
    // Until the logits are there: what the kernel before only reads.  (It starts this one behind its own wait, so
    // what came before it is complete.)
    const int kvh = blockIdx.y, b = blockIdx.z;
    Seen<U> s;
    s.of(a, b);
    const int i = (blockIdx.x * blockDim.x + threadIdx.x) * 4, u = i / U;
    const int pos0 = s.base(u) + i - u * U, bs = a.block_size;
    float* sc[4];
    float w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        sc[e] = nullptr;
        if (u >= s.n || !s.sees(u, pos0 + e)) continue;
        const int at = a.div.block(pos0 + e), blk = a.block_tables[(int64_t)b * a.max_blocks + at];
        if ((unsigned)blk < (unsigned)a.num_blocks)
            sc[e] = a.scores + ((int64_t)blk * a.nkv + kvh) * bs + a.div.slot(pos0 + e, at);
    }
    float old[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (sc[e] && pos0 + e != s.L - 1) old[e] = *sc[e];
    griddep_wait();
    griddep_launch_dependents();
    if (u >= s.n) return;
    const int h0 = b * a.nq + kvh * a.group;
    const float* lg = a.logits + (int64_t)h0 * a.cap + i;
    float4 x[4];
    float2 st[4];
#pragma unroll
    for (int h = 0; h < 4; ++h)
        if (h < a.group) {
            x[h] = __ldcg(reinterpret_cast<const float4*>(lg + (int64_t)h * a.cap));
            st[h] = a.stats[h0 + h];
        }
    auto add = [&](float4 l, float2 ml) {
        const float inv = ml.y > 0.f ? 1.f / ml.y : 0.f;
        w[0] = fmaf(ex2(l.x - ml.x), inv, w[0]);
        w[1] = fmaf(ex2(l.y - ml.x), inv, w[1]);
        w[2] = fmaf(ex2(l.z - ml.x), inv, w[2]);
        w[3] = fmaf(ex2(l.w - ml.x), inv, w[3]);
    };
#pragma unroll
    for (int h = 0; h < 4; ++h)
        if (h < a.group) add(x[h], st[h]);
#pragma unroll 4
    for (int h = 4; h < a.group; ++h)
        add(__ldcg(reinterpret_cast<const float4*>(lg + (int64_t)h * a.cap)), a.stats[h0 + h]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (sc[e]) *sc[e] = old[e] + w[e];
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

struct PagedSizes {
    int gs, hg, grid;
    int64_t cap;
    size_t parts, pml, stats, logits;  // bytes
};

// Segments take up to 16 heads; a larger group is cut evenly.
static PagedSizes paged_sizes(int batch, int nq, int nkv, int D, int64_t max_positions, bool scored) {
    PagedSizes z = {};
    const int group = nq / nkv;
    z.hg = (group + 15) / 16;
    z.gs = (group + z.hg - 1) / z.hg;
    z.grid = sm_count() * (D > 128 ? 1 : 2);
    // whole units of up to 128 positions over the sinks and over the window, whose first may begin 15 early; rows of
    // whole 128-byte lines
    z.cap = (max_positions + 2 * 127 + 15 + 31) & ~int64_t(31);
    z.parts = (size_t)2 * z.grid * z.gs * D * sizeof(float);
    z.pml = (size_t)2 * z.grid * z.gs * sizeof(float2);
    z.stats = scored ? ((size_t)batch * nq * sizeof(float2) + 15) & ~size_t(15) : 0;
    z.logits = scored ? (size_t)batch * nq * z.cap * sizeof(float) : 0;
    return z;
}

template <int DP, bool GH, bool BF16, bool LIST>
static int paged_launch(const PagedArgs& a, const PagedSizes& z, cudaStream_t s) {
    using C = PagedCfg<DP, GH>;
    auto kern = paged_attn_kernel<DP, GH, BF16, LIST>;
    static bool done[64];
    B2_TRY(allow_smem(kern, C::BYTES, done));
    B2_TRY(launch(kern, dim3(z.grid), dim3(kPgThreads), C::BYTES, s, true, a));
    if (a.scores)
        B2_TRY(launch(paged_scores_kernel<C::U>, dim3((unsigned)((a.cap + 4 * kPgScoreThreads - 1) / (4 * kPgScoreThreads)), a.nkv, a.batch),
                      dim3(kPgScoreThreads), 0, s,
                      true, a));
    return B2_OK;
}

template <int DP, bool LIST>
static int paged_dispatch(const PagedArgs& a, const PagedSizes& z, cudaStream_t s) {
    if (a.kv.bf16)
        return a.gs > 8 ? paged_launch<DP, true, true, LIST>(a, z, s) : paged_launch<DP, false, true, LIST>(a, z, s);
    return a.gs > 8 ? paged_launch<DP, true, false, LIST>(a, z, s) : paged_launch<DP, false, false, LIST>(a, z, s);
}
template <bool LIST>
static int paged_dispatch(const PagedArgs& a, const PagedSizes& z, cudaStream_t s) {
    if (a.D <= 64) return paged_dispatch<64, LIST>(a, z, s);
    if (a.D <= 128) return paged_dispatch<128, LIST>(a, z, s);
    return paged_dispatch<256, LIST>(a, z, s);
}

// Checks and arguments of both entry points: blocks null, or the listed blocks of each (sequence, kv head).
static int paged_call(const void* q, int64_t ldq, const b2_paged_kv* kv, void* out, float* scores, const int* blocks,
                      int listed, int batch, int nq, int nkv, int D, int window, int sinks, b2_workspace* ws,
                      void* stream) {
    if (batch <= 0) return B2_OK;
    B2_REQUIRE(q && out && nq > 0 && nkv > 0 && nq % nkv == 0 && window >= 0 && sinks >= 0);
    const int rc = check_paged(kv, nkv, D);
    if (rc != B2_OK) return rc;
    if (!aligned16(q) || !aligned16(out) || (ldq & 7)) return B2_ERR_UNSUPPORTED;
    if (scores && !ws) return B2_ERR_WORKSPACE;
    const int64_t span = (int64_t)(blocks ? listed : kv->max_blocks) * kv->block_size;
    if (span > (1 << 30)) return B2_ERR_UNSUPPORTED;
    const int64_t most = window > 0 && (int64_t)window + sinks < span ? (int64_t)window + sinks : span;
    const PagedSizes z = paged_sizes(batch, nq, nkv, D, most, scores != nullptr);
    // units are counted in 32 bits; the scores' grid has (nkv, batch) as (y, z)
    if ((int64_t)batch * nkv * z.hg * ((most >> 6) + 4) > (1ll << 31) - 1 ||
        (scores && (batch > 65535 || nkv > 65535)))
        return B2_ERR_UNSUPPORTED;
    PagedArgs a = {};
    a.q = q;
    a.ldq = ldq;
    a.kv = *kv;
    a.block_tables = kv->block_tables;
    a.seq_lens = kv->seq_lens;
    a.num_blocks = kv->num_blocks;
    a.block_size = kv->block_size;
    a.max_blocks = kv->max_blocks;
    a.div = block_div(kv->block_size);
    a.blocks = blocks;
    a.listed = listed;
    a.out = out;
    a.scores = scores;
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
    a.whole = kv->block_size % 16 == 0;
    a.cap = (int)z.cap;
    if (ws) {
        if (ws->bytes < z.parts + z.pml + z.stats + z.logits || z.grid > kWsCounters) return B2_ERR_WORKSPACE;
        uint8_t* w = static_cast<uint8_t*>(ws->ptr);
        a.logits = scores ? reinterpret_cast<float*>(w) : nullptr;
        a.stats = scores ? reinterpret_cast<float2*>(w + z.logits) : nullptr;
        a.parts = reinterpret_cast<float*>(w + z.logits + z.stats);
        a.pml = reinterpret_cast<float2*>(w + z.logits + z.stats + z.parts);
        a.counters = ws->counters;
    }
    cudaStream_t s = as_stream(stream);
    return blocks ? paged_dispatch<true>(a, z, s) : paged_dispatch<false>(a, z, s);
}

}  // namespace b2

extern "C" size_t b2_paged_decode_workspace_bytes(int batch, int nq, int nkv, int D, int64_t max_positions,
                                                  int scored) {
    if (batch <= 0 || nq <= 0 || nkv <= 0 || nq % nkv || D <= 0 || max_positions < 0) return 0;
    const b2::PagedSizes z = b2::paged_sizes(batch, nq, nkv, D, max_positions, scored != 0);
    return z.parts + z.pml + z.stats + z.logits;
}

extern "C" int b2_paged_decode_gqa(const void* q, int64_t ldq, const b2_paged_kv* kv, void* out, float* scores,
                                   int batch, int nq, int nkv, int D, int window, int sinks, b2_workspace* ws,
                                   void* stream) {
    return b2::paged_call(q, ldq, kv, out, scores, nullptr, 0, batch, nq, nkv, D, window, sinks, ws, stream);
}

extern "C" int b2_paged_decode_gqa_blocks(const void* q, int64_t ldq, const b2_paged_kv* kv, const int* blocks,
                                          int listed, void* out, int batch, int nq, int nkv, int D, b2_workspace* ws,
                                          void* stream) {
    if (batch <= 0) return B2_OK;
    B2_REQUIRE(blocks && listed > 0);
    return b2::paged_call(q, ldq, kv, out, nullptr, blocks, listed, batch, nq, nkv, D, 0, 0, ws, stream);
}
