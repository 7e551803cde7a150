// window.cu -- causal GQA attention of a chunk of query tokens with a sliding
// window and sinks (operator API window_prefill_gqa).
//
//   out_i = sum_j p_ij v_j,  p_i = softmax over {j <= i : i - j < W or j < K}
//   of q_i . k_j / sqrt(D)
//
// Tensor-core form (window_tc_kernel, head_dim <= 128).  4 D flops per
// visible (query, key) pair against 2 D bytes per key of each 256-query pair
// of tiles: bound by the tensor cores and, beside them, by the exponentials.
// One persistent CTA per SM takes pairs of 128-query tiles (A, B) of one head;
// a pair visits only the 128-key tiles that one of its rows sees:
//   the window's tiles of A, the sinks' tiles (as wide as the sinks, in steps
//   of 16 keys), then the tiles only B reaches --
// an order in which the tiles of A, and those of B, are each consecutive.
//   S_t = Q_t K^T   M = 128 queries, N = keys of the tile, in TMEM
//   O_t += P_t V    P_t, 16-bit, over S_t's columns in TMEM (A operand)
// with the order PV_A, S_A', PV_B, S_B' per key tile, so that one tile's
// products run while the other's softmax does.  Across pairs nothing drains:
// the next pair's Q, K and V are requested as soon as their buffers are read,
// and its first S is issued behind the last PV, while the softmax warps still
// write the outputs.
// Online softmax in the log2 domain, one query row per thread; the reference
// max moves only when a row's max exceeds it by more than 8, so O is rescaled
// rarely and P stays below 2^8.  Masks only in tiles that a row of the warp
// does not see whole; 32-key stretches that no row of the warp sees cost a
// zero store.  P is rounded to 16 bits for the product (its row sum is not):
// one more rounding the size of the output's own.
#include <cmath>

#include "tc.cuh"

namespace b2 {

struct WinArgs {
    b2_kv_view q, k, v;
    void* out;
    const int* seq_lens;
    int S, q_start, nq, nkv, D, batch;
    int window, sinks;
    float scale_log2;
};

template <bool BF16>
__device__ __forceinline__ float ld16f(const void* p, int64_t i) {
    if constexpr (BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

template <bool BF16>
__device__ __forceinline__ void st16f(void* p, int64_t i, float v) {
    if constexpr (BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// One warp per (query, head); lane l holds elements l, l + 32, .. of the
// rows.  Any element alignment, D <= 256.
template <bool BF16>
__global__ void __launch_bounds__(256) window_rows_kernel(const WinArgs a) {
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t n = (int64_t)a.batch * a.S * a.nq;
    for (int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; w < n;
         w += ((int64_t)gridDim.x * blockDim.x) >> 5) {
        const int h = (int)(w % a.nq);
        const int i = (int)((w / a.nq) % a.S);
        const int b = (int)(w / ((int64_t)a.nq * a.S));
        const int pos = a.q_start + i;
        const int len = a.seq_lens ? min(a.seq_lens[b], a.q_start + a.S) : a.q_start + a.S;
        const int kvh = h / (a.nq / a.nkv);
        float q[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = lane + 32 * e;
            q[e] = d < a.D ? ld16f<BF16>(a.q.data, b * a.q.stride_b + h * a.q.stride_h + i * a.q.stride_s + d) : 0.f;
            o[e] = 0.f;
        }
        if (pos < len) {
            const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
            const int64_t kb = b * a.k.stride_b + kvh * a.k.stride_h, vb = b * a.v.stride_b + kvh * a.v.stride_h;
            for (int j = 0; j <= pos; ++j) {
                if (j < lo && j >= a.sinks) j = lo;
                float s = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (lane + 32 * e < a.D) s = fmaf(q[e], ld16f<BF16>(a.k.data, kb + j * a.k.stride_s + lane + 32 * e), s);
                s = warp_sum(s) * a.scale_log2;
                const float m_new = fmaxf(m, s);
                const float al = exp2f(m - m_new), p = exp2f(s - m_new);
                m = m_new;
                l = fmaf(l, al, p);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (lane + 32 * e < a.D)
                        o[e] = fmaf(o[e], al, p * ld16f<BF16>(a.v.data, vb + j * a.v.stride_s + lane + 32 * e));
            }
        }
        const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < a.D) st16f<BF16>(a.out, w * a.D + lane + 32 * e, o[e] * inv);
    }
}

// ---------------------------------------------------------------------------
// tensor-core form
// ---------------------------------------------------------------------------

template <int D>
struct WinCfg {
    static constexpr int ATOMS = D / 64;              // 128-byte swizzle atoms per row
    static constexpr uint32_t ATOM = 128 * 128;       // bytes of one 128-row atom
    static constexpr uint32_t TILE = 128 * D * 2;     // a Q, K or V tile
    static constexpr int ST = D == 64 ? 4 : 2;        // K and V stages
    static constexpr uint32_t OFF_K = 2 * TILE;
    static constexpr uint32_t OFF_V = OFF_K + ST * TILE;
    static constexpr uint32_t OFF_BAR = OFF_V + ST * TILE;
    // above half an SM's shared memory: one CTA, with all 512 TMEM columns, per SM
    static constexpr size_t NEED = OFF_BAR + 256 + 1024;
    static constexpr size_t SMEM = NEED > 122880 ? NEED : 122880;
    // warps 0-7 softmax, 8 TMA, 9 MMA, 10 and 11 idle (a warpgroup gives up its registers as a whole)
    static constexpr int THREADS = 384;
};

// The launch gives each of the three warpgroups 168 registers a thread; the
// last one hands most of its share to the two that hold a row of S.
constexpr int kWinRegsFew = 104, kWinRegsMany = 200;
static_assert(kWinRegsFew + 2 * kWinRegsMany <= 3 * 168, "more registers than the block is launched with");

template <bool BF16>
__device__ __forceinline__ uint32_t win_pack(float a, float b) {
    if constexpr (BF16) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    } else {
        return f2_to_h2(a, b);
    }
}

// 2^x on the SFU: 2^-22 relative, far below the 16-bit rounding P gets next
__device__ __forceinline__ float win_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One pair of query tiles of one head, and the key tiles it visits.
struct WinItem {
    int b, h, row0;        // first query row of tile A
    int len;               // tokens of the sequence
    int p0;                // position of row0
    bool hasB;
    int loA, nw, ns, hiA;  // window tiles loA .. loA + nw - 1 = hiA of A, sinks' tiles 0 .. ns - 1
    int nA, n, dB;         // A visits steps 0 .. nA - 1, B steps dB .. n - 1

    // Number of valid pairs of sequence b.
    static __device__ __forceinline__ int length(const WinArgs& a, int b) {
        const int T = a.q_start + a.S;
        return a.seq_lens ? max(0, min(a.seq_lens[b], T)) : T;
    }
    static __device__ __forceinline__ int pairs(const WinArgs& a, int len) {
        return (max(0, len - a.q_start) + 255) >> 8;
    }

    __device__ __forceinline__ void of(const WinArgs& a, int b_, int len_, int pair, int h_) {
        b = b_;
        h = h_;
        len = len_;
        row0 = pair * 256;
        p0 = a.q_start + row0;
        hasB = row0 + 128 < a.S && p0 + 128 < len;
        loA = a.window > 0 ? max(0, p0 - a.window + 1) >> 7 : 0;
        hiA = min(p0 + 127, len - 1) >> 7;
        nw = hiA - loA + 1;
        const int st = a.window > 0 ? (a.sinks + 127) >> 7 : 0;
        ns = min(st, loA);
        nA = nw + ns;
        n = nA;
        dB = 0;
        if (hasB) {
            n += (min(p0 + 255, len - 1) >> 7) - hiA;
            // B skips A's first tiles, unless they hold sinks
            if (a.window > 0 && loA >= st) dB = (max(0, p0 + 128 - a.window + 1) >> 7) - loA;
        }
    }
    // Key tile of step j.
    __device__ __forceinline__ int tile(int j) const {
        return j < nw ? loA + j : j < nA ? j - nw : j - ns + loA;
    }
    // Keys of step j's tile that query tile t may see, in steps of 16.
    __device__ __forceinline__ int width(const WinArgs& a, int t, int j) const {
        const int kb = tile(j) << 7;
        int end = min(p0 + 128 * t + 127, len - 1) + 1;
        if (j >= nw && j < nA) end = min(end, a.sinks);
        return min(128, (end - kb + 15) & ~15);
    }
};

// The valid pairs of all sequences, each with all its heads, dealt round robin
// to the CTAs; a sequence's later (longer) pairs first.
struct WinList {
    int b = 0, len = 0, np = 0;
    int64_t before = 0;  // items of sequences before b
    __device__ __forceinline__ bool get(const WinArgs& a, int64_t i, WinItem& it) {
        if (b == 0 && before == 0 && np == 0) enter(a);
        while (b < a.batch && i - before >= (int64_t)np * a.nq) {
            before += (int64_t)np * a.nq;
            ++b;
            enter(a);
        }
        if (b >= a.batch) return false;
        const int k = (int)(i - before);
        it.of(a, b, len, np - 1 - k / a.nq, k % a.nq);
        return true;
    }
    __device__ __forceinline__ void enter(const WinArgs& a) {
        if (b >= a.batch) return;
        len = WinItem::length(a, b);
        np = WinItem::pairs(a, len);
    }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(WinCfg<D>::THREADS, 1)
    window_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const WinArgs a, int* err) {
    using C = WinCfg<D>;
    constexpr uint32_t TILE = C::TILE, ATOM = C::ATOM;
    constexpr int ST = C::ST;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = sm;
    uint8_t* sK = sm + C::OFF_K;
    uint8_t* sV = sm + C::OFF_V;
    uint64_t* bar = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t* q_full = bar;
    uint64_t* q_empty = bar + 1;        // every S of the pair is done
    uint64_t* k_full = bar + 2;         // [ST]
    uint64_t* k_empty = k_full + ST;    // [ST]
    uint64_t* v_full = k_empty + ST;    // [ST]
    uint64_t* v_empty = v_full + ST;    // [ST]
    uint64_t* s_full = v_empty + ST;    // [tile]
    uint64_t* p_full = s_full + 2;      // [tile]
    uint64_t* o_done = p_full + 2;      // [tile]: the pair's last P V of the tile is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        tc::mbar_init(q_full, 1);
        tc::mbar_init(q_empty, 1);
        for (int s = 0; s < ST; ++s) {
            tc::mbar_init(&k_full[s], 1);
            tc::mbar_init(&k_empty[s], 1);
            tc::mbar_init(&v_full[s], 1);
            tc::mbar_init(&v_empty[s], 1);
        }
        for (int t = 0; t < 2; ++t) {
            tc::mbar_init(&s_full[t], 1);
            tc::mbar_init(&p_full[t], 128);
            tc::mbar_init(&o_done[t], 1);
        }
        tc::fence_barrier_init();
    }
    if (warp == 0) tc::tmem_alloc(tmem_slot, 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    griddep_wait();
    griddep_launch_dependents();

    WinList list;
    WinItem it;
    uint32_t g = 0;  // key tiles of the pairs before this one

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWinRegsFew));
        if (warp == 8) {
            // ---------------- TMA producer ----------------
            if (lane == 0) {
                bool ok = true;
                uint32_t k = 0;
                for (int64_t i = blockIdx.x; ok && list.get(a, i, it); i += gridDim.x, ++k) {
                    const int kvh = it.h / (a.nq / a.nkv);
                    if (k > 0 && !tc::mbar_wait(q_empty, (k - 1) & 1u, err, 91)) break;
                    tc::mbar_arrive_expect_tx(q_full, 2 * TILE);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
                            tc::tma_load_4d(sQ + t * TILE + c * ATOM, &tmQ, q_full, c * 64, it.h, it.row0 + t * 128, it.b);
                    for (int j = 0; j < it.n; ++j, ++g) {
                        const uint32_t s = g % ST, u = g / ST;
                        const int row = it.tile(j) * 128;
                        if (g >= ST && !(ok = tc::mbar_wait(&k_empty[s], (u - 1) & 1u, err, 92))) break;
                        tc::mbar_arrive_expect_tx(&k_full[s], TILE);
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
                            tc::tma_load_4d(sK + s * TILE + c * ATOM, &tmK, &k_full[s], c * 64, kvh, row, it.b);
                        if (g >= ST && !(ok = tc::mbar_wait(&v_empty[s], (u - 1) & 1u, err, 93))) break;
                        tc::mbar_arrive_expect_tx(&v_full[s], TILE);
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
                            tc::tma_load_4d(sV + s * TILE + c * ATOM, &tmV, &v_full[s], c * 64, kvh, row, it.b);
                    }
                }
            }
        } else if (warp == 9) {
            // ---------------- MMA issuer ----------------
            if (lane == 0) {
                constexpr uint32_t idO = tc::idesc_f16(128, D, BF16, true);
                const uint32_t aQ = tc::smem_u32(sQ), aK = tc::smem_u32(sK), aV = tc::smem_u32(sV);
                bool ok = true;
                uint32_t k = 0, np = 0;  // pairs; bit t: parity of the P tiles consumed of query tile t
                // a descriptor's address field counts 16 bytes: steps are added to it
                auto issue_s = [&](int t, int j) {
                    const uint32_t idS = tc::idesc_f16(128, 0, BF16, false) | ((uint32_t)(it.width(a, t, j) >> 3) << 17);
                    const uint64_t dq = tc::desc_k_sw128(aQ + (uint32_t)t * TILE),
                                   dk = tc::desc_k_sw128(aK + ((g + j) % ST) * TILE);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = ((uint32_t)(kk >> 2) * ATOM + (uint32_t)(kk & 3) * 32) >> 4;
                        tc::mma_f16(tmem + (uint32_t)t * 256, dq + off, dk + off, idS, kk > 0 ? 1u : 0u);
                    }
                    tc::mma_commit(&s_full[t]);
                };
                auto issue_pv = [&](int t, int j, bool first, bool last) {
                    const uint64_t dv = tc::desc_mn_sw128(aV + ((g + j) % ST) * TILE, ATOM);
                    const int steps = it.width(a, t, j) >> 4;
                    const uint32_t tP = tmem + (uint32_t)t * 256;
                    tc::mma_f16_ts(tP + 128, tP, dv, idO, first ? 0u : 1u);
#pragma unroll
                    for (int kk = 1; kk < 8; ++kk)
                        if (kk < steps) tc::mma_f16_ts(tP + 128, tP + (uint32_t)kk * 8, dv + (uint32_t)kk * 128u, idO, 1u);
                    if (last) tc::mma_commit(&o_done[t]);
                };
                auto wait_k = [&](int j) { return tc::mbar_wait(&k_full[(g + j) % ST], ((g + j) / ST) & 1u, err, 94); };
                auto wait_v = [&](int j) { return tc::mbar_wait(&v_full[(g + j) % ST], ((g + j) / ST) & 1u, err, 95); };
                for (int64_t i = blockIdx.x; ok && list.get(a, i, it); i += gridDim.x, ++k) {
                    ok = tc::mbar_wait(q_full, k & 1u, err, 96) && wait_k(0);
                    if (!ok) break;
                    tc::fence_after_sync();
                    issue_s(0, 0);
                    if (it.hasB && it.dB == 0) issue_s(1, 0);
                    tc::mma_commit(&k_empty[g % ST]);
                    if (it.n == 1) tc::mma_commit(q_empty);
                    for (int j = 0; j < it.n; ++j) {
                        const bool more = j + 1 < it.n;
                        bool v_ok = false, k_ok = false;
#pragma unroll 1
                        for (int t = 0; t < 2; ++t) {
                            const int from = t == 0 ? 0 : it.dB, to = t == 0 ? it.nA : it.hasB ? it.n : 0;
                            if (j >= from && j < to) {
                                ok = ok && tc::mbar_wait(&p_full[t], (np >> t) & 1u, err, 97) && (v_ok || wait_v(j));
                                if (!ok) break;
                                v_ok = true;
                                np ^= 1u << t;
                                tc::fence_after_sync();
                                issue_pv(t, j, j == from, j + 1 == to);
                            }
                            if (j + 1 >= from && j + 1 < to) {
                                ok = ok && (k_ok || wait_k(j + 1));
                                if (!ok) break;
                                k_ok = true;
                                tc::fence_after_sync();
                                issue_s(t, j + 1);
                            }
                        }
                        if (!ok) break;
                        tc::mma_commit(&v_empty[(g + j) % ST]);
                        if (more) tc::mma_commit(&k_empty[(g + j + 1) % ST]);
                        if (j + 2 == it.n) tc::mma_commit(q_empty);
                    }
                    g += it.n;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWinRegsMany));
        // ---------------- softmax and output: tile t, one query row per thread ----------------
        const int t = warp >> 2, rq = warp & 3;
        const int r = rq * 32 + lane;
        const uint32_t lane_base = (uint32_t)(rq * 32) << 16;
        const uint32_t tS = tmem + (uint32_t)t * 256 + lane_base, tO = tS + 128;
        const int T = a.q_start + a.S;
        bool ok = true;
        uint32_t cs = 0, co = 0;  // S tiles and outputs of this tile so far
        for (int64_t i = blockIdx.x; ok && list.get(a, i, it); i += gridDim.x) {
            const int from = t == 0 ? 0 : it.dB, to = t == 0 ? it.nA : it.hasB ? it.n : 0;
            const int wp = it.p0 + t * 128 + rq * 32;        // position of the warp's first row
            const int pos = it.p0 + t * 128 + r < it.len ? it.p0 + t * 128 + r : -1;
            float m = -1e30f, l = 0.f;  // finite: a row that has seen nothing keeps P = 0 and l = 0
            for (int j = from; j < to; ++j, ++cs) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait(&s_full[t], cs & 1u, err, 98));
                if (!ok) break;
                tc::fence_after_sync();
                const int kb = it.tile(j) << 7, w = it.width(a, t, j);
                uint32_t v[128];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (32 * c < w) tc::tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&v[32 * c]));
                tc::tmem_wait_ld();
                // the tile whole, for every row of the warp?
                const bool whole = w == 128 && kb + 127 <= wp && wp + 31 < it.len &&
                                   (a.window == 0 || kb > wp + 31 - a.window || kb + 128 <= a.sinks);
                uint32_t some = 0xf;  // 32-key stretches that some row of the warp sees
                if (!whole) {
                    const int hi = pos - kb, lo = a.window > 0 ? pos - a.window + 1 - kb : 0, sk = a.window > 0 ? a.sinks - kb : 0;
                    const int whi = wp + 31 - kb, wlo = a.window > 0 ? wp - a.window + 1 - kb : 0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (32 * c >= w || 32 * c > whi || (32 * c + 31 < wlo && 32 * c >= sk)) some &= ~(1u << c);
                        if (some >> c & 1) {
#pragma unroll
                            for (int e = 32 * c; e < 32 * c + 32; ++e)
                                if (e > hi || (e < lo && e >= sk)) v[e] = 0xff800000u;  // -inf
                        }
                    }
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (some >> c & 1) {
#pragma unroll
                        for (int e = 32 * c; e < 32 * c + 32; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(v[e]));
                    }
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;
                const float m_new = fmaxf(m, mx);
                const bool resc = m_new > m + 8.f;
                const float m_use = resc ? m_new : m;
                const float alpha = win_ex2(m - m_use);
                if (j > from && __any_sync(0xffffffffu, resc)) {
                    // the P V before has completed (S, issued behind it, has)
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tc::tmem_ld32(tO + c, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tc::tmem_st32(tO + c, o);
                    }
                }
                m = m_use;
                float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (32 * c >= w) break;
                    uint32_t pk[16];
                    if (some >> c & 1) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float p0 = win_ex2(fmaf(__uint_as_float(v[32 * c + e]), a.scale_log2, -m));
                            const float p1 = win_ex2(fmaf(__uint_as_float(v[32 * c + e + 1]), a.scale_log2, -m));
                            l4[(e >> 1) & 3] += p0 + p1;
                            pk[e >> 1] = win_pack<BF16>(p0, p1);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) pk[e] = 0u;
                    }
                    tc::tmem_st16(tS + (uint32_t)(16 * c), pk);
                }
                l = l * alpha + ((l4[0] + l4[1]) + (l4[2] + l4[3]));
                tc::tmem_wait_st();
                if (kb + w > it.len && it.len < T) {
                    // rows past the sequence may hold anything: P is 0 there, and V has to be finite
                    const uint32_t gj = g + j, s = gj % ST;
                    ok = __all_sync(0xffffffffu, tc::mbar_wait(&v_full[s], (gj / ST) & 1u, err, 99));
                    if (!ok) break;
                    if (kb + r >= it.len) {
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                reinterpret_cast<uint4*>(sV + s * TILE + c * ATOM + r * 128)[q] = make_uint4(0, 0, 0, 0);
                    }
                    tc::fence_proxy_async_smem();
                }
                tc::fence_before_sync();
                tc::mbar_arrive(&p_full[t]);
            }
            if (ok && to > from) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait(&o_done[t], co & 1u, err, 100));
                ++co;
                tc::fence_after_sync();
                const float inv_l = l > 0.f ? 1.f / l : 0.f;
                const int row = it.row0 + t * 128 + r;
                uint16_t* orow = static_cast<uint16_t*>(a.out) + (((int64_t)it.b * a.S + row) * a.nq + it.h) * a.D;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tc::tmem_ld32(tO + c, o);
                    tc::tmem_wait_ld();
                    if (!ok || row >= a.S) continue;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (c + 8 * q >= a.D) break;
                        uint4 x;
                        x.x = win_pack<BF16>(__uint_as_float(o[8 * q + 0]) * inv_l, __uint_as_float(o[8 * q + 1]) * inv_l);
                        x.y = win_pack<BF16>(__uint_as_float(o[8 * q + 2]) * inv_l, __uint_as_float(o[8 * q + 3]) * inv_l);
                        x.z = win_pack<BF16>(__uint_as_float(o[8 * q + 4]) * inv_l, __uint_as_float(o[8 * q + 5]) * inv_l);
                        x.w = win_pack<BF16>(__uint_as_float(o[8 * q + 6]) * inv_l, __uint_as_float(o[8 * q + 7]) * inv_l);
                        *reinterpret_cast<uint4*>(orow + c + 8 * q) = x;
                    }
                }
            }
            g += it.n;
        }
        // rows of tiles past a sequence's end: zeros
        if (a.seq_lens) {
            const int64_t row16 = (int64_t)a.nq * a.D / 8;
            for (int b = 0; b < a.batch; ++b) {
                const int len = WinItem::length(a, b);
                int done = WinItem::pairs(a, len) * 256;
                if (done > 0 && a.q_start + done - 128 >= len) done -= 128;  // the last pair had no tile B
                if (done >= a.S) continue;
                uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + ((int64_t)b * a.S + done) * a.nq * a.D);
                for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (a.S - done) * row16;
                     i += (int64_t)gridDim.x * 256)
                    o[i] = make_uint4(0, 0, 0, 0);
            }
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 0) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, 512);
    }
}

static int window_map(CUtensorMap* m, const b2_kv_view& v, int heads, int64_t rows, const WinArgs& a, bool bf16) {
    const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)heads, (uint64_t)rows, (uint64_t)a.batch};
    const uint64_t st[3] = {(uint64_t)v.stride_h * 2, (uint64_t)v.stride_s * 2, (uint64_t)v.stride_b * 2};
    const uint32_t box[4] = {64, 1, 128, 1};
    return make_tensor_map(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, v.data,
                           dims, st, box);
}

// Rows that 16-byte copies can fetch.
static bool window_tma_view(const b2_kv_view& v, int heads, int64_t rows, int batch) {
    auto stride_ok = [](int64_t s, int64_t n) { return n <= 1 || (s > 0 && s % 8 == 0 && s < ((int64_t)1 << 38)); };
    return aligned16(v.data) && stride_ok(v.stride_h, heads) && stride_ok(v.stride_s, rows) && stride_ok(v.stride_b, batch);
}

template <int D, bool BF16>
static int launch_window_tc(const WinArgs& a_in, cudaStream_t s) {
    using C = WinCfg<D>;
    int* err = wait_error_word();
    if (!err) return B2_ERR_STATE;
    WinArgs a = a_in;
    const int64_t T = (int64_t)a.q_start + a.S;
    // the stride of a dimension of one is never used, but has to be encodable
    auto tidy = [&](b2_kv_view& v, int heads, int64_t rows) {
        if (heads == 1) v.stride_h = 8;
        if (rows == 1) v.stride_s = 8;
        if (a.batch == 1) v.stride_b = 8;
    };
    tidy(a.q, a.nq, a.S);
    tidy(a.k, a.nkv, T);
    tidy(a.v, a.nkv, T);
    CUtensorMap tq, tk, tv;
    int rc = window_map(&tq, a.q, a.nq, a.S, a, BF16);
    if (rc == B2_OK) rc = window_map(&tk, a.k, a.nkv, T, a, BF16);
    if (rc == B2_OK) rc = window_map(&tv, a.v, a.nkv, T, a, BF16);
    if (rc != B2_OK) return rc;
    auto kern = window_tc_kernel<D, BF16>;
    B2_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
    const int64_t items = (int64_t)a.batch * a.nq * ((a.S + 255) / 256);
    const unsigned grid = (unsigned)(items < sm_count() ? items : sm_count());
    B2_TRY(launch(kern, dim3(grid), dim3(C::THREADS), C::SMEM, s, true, tq, tk, tv, a, err));
    return B2_OK;
}

}  // namespace b2

extern "C" int b2_window_prefill_gqa(b2_kv_view q, b2_kv_view k, b2_kv_view v, void* out, const int* seq_lens,
                                     int64_t q_len, int64_t q_start, int nq, int nkv, int D, int batch,
                                     int64_t window, int64_t sinks, int bf16, void* stream) {
    using namespace b2;
    if (q_len <= 0 || batch <= 0) return B2_OK;
    B2_REQUIRE(q.data && k.data && v.data && out && q_start >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0 && D > 0 &&
               window >= 0 && sinks >= 0);
    if (D > 256 || q_len + q_start > (1 << 30) || q.stride_d != 1 || k.stride_d != 1 || v.stride_d != 1)
        return B2_ERR_UNSUPPORTED;
    WinArgs a = {};
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.seq_lens = seq_lens;
    a.S = (int)q_len;
    a.q_start = (int)q_start;
    a.nq = nq;
    a.nkv = nkv;
    a.D = D;
    a.batch = batch;
    // a window past the last position sees everything, and so do that many sinks
    a.window = window > q_len + q_start ? 0 : (int)window;
    a.sinks = (int)(sinks > q_len + q_start ? q_len + q_start : sinks);
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)D);
    const int64_t T = q_len + q_start;
    if (D <= 128 && D % 8 == 0 && aligned16(out) && window_tma_view(q, nq, q_len, batch) &&
        window_tma_view(k, nkv, T, batch) && window_tma_view(v, nkv, T, batch)) {
        cudaStream_t s = as_stream(stream);
        if (D <= 64) return bf16 ? launch_window_tc<64, true>(a, s) : launch_window_tc<64, false>(a, s);
        return bf16 ? launch_window_tc<128, true>(a, s) : launch_window_tc<128, false>(a, s);
    }
    const int64_t warps = q_len * nq * batch;
    int64_t blocks = (warps + 7) / 8;
    if (blocks > (int64_t)sm_count() * 64) blocks = (int64_t)sm_count() * 64;
    B2_TRY(launch(bf16 ? window_rows_kernel<true> : window_rows_kernel<false>, dim3((unsigned)blocks), dim3(256), 0,
                  as_stream(stream), true, a));
    return B2_OK;
}
