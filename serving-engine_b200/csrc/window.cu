// window.cu -- causal GQA attention of a chunk of query tokens with a sliding
// window and sinks (operator API window_prefill_gqa).
//
//   out_i = sum_j p_ij v_j,  p_i = softmax over {j <= i : i - j < W or j < K}
//   of q_i . k_j / sqrt(D)
//
// Tensor-core form (window_tc_kernel, head_dim <= 128).  4 D flops per
// visible (query, key) pair against 2 D bytes per key of each 256-query pair
// of tiles: bound by the tensor cores and, beside them, by the exponentials.
// One persistent CTA per SM takes pairs of 128-query tiles (A, B), two heads of
// a kv head's group at the same rows where it can, so that they visit the same
// key tiles: K and V come once for both.  A pair visits only the 128-key tiles
// that one of its rows sees:
//   the window's tiles of A, the sinks' tiles (as wide as the sinks, in steps
//   of 16 keys), then the tiles only B reaches --
// an order in which the tiles of A, and those of B, are each consecutive.
//   S_t = Q_t K^T   M = 128 queries, N = keys of the tile, in TMEM
//   O_t += P_t V    P_t, 16-bit, over S_t's columns in TMEM (A operand)
// with one MMA issuer warp per tile, taking turns: PV_A, S_A', PV_B, S_B' per
// key tile.  The turns keep the two softmaxes half a step apart (without them
// both run, then both wait: 83 us for a chunk of 512 after 5500 at 64 heads when
// it took 74 with them), and an issuer does its waiting and addressing while the other's
// products are queued.  Across pairs nothing drains: the next pair's Q, K and V
// are requested as soon as their buffers are read.
// Online softmax in the log2 domain, one query row per thread; the reference
// max moves only when a row's max exceeds it by more than 8, so O is rescaled
// rarely and P stays below 2^8.  P is handed over in two halves of 64 keys, so
// that P V starts while the second half's exponentials run.  Masks only in
// tiles that a row of the warp does not see whole.  P is rounded to 16 bits
// for the product (its row sum is not): one more rounding the size of the
// output's own.  Outputs leave by TMA from shared memory.
//
// A step of two tiles and 128 keys takes 3.1 k cycles at head dim 128: 2.0 k of
// products, and the chain S, softmax (2.0 k), P V, S around them, which is what
// a step lasts: P lies over S, so that the next S waits for P V.  Measured, 8192
// tokens, window 2048, 32 heads of 128, bf16: 260 us called in a row for long
// (927 TFLOP/s of visible pairs; the chip at 990 W and 1.7 GHz), 235 to 243 in
// graph replays, 224 in a short run at 1.97 GHz (1077 TFLOP/s, 66 % of the
// measured burst rate).  Without a window: 502 us in graph replays, 1095
// TFLOP/s.  Head dims between 64 and 128 cost what 128 costs (80 and 96: 218
// us in a short run).
#include <cmath>
#include <type_traits>

#include "mma.cuh"
#include "tc.cuh"

namespace b2 {

struct WinArgs {
    b2_kv_view q, k, v;
    void* out;
    const int* seq_lens;
    int S, q_start, nq, nkv, D, batch;
    int window, sinks;
    float scale_log2;
    int single;  // tiles are not paired
};

// ---------------------------------------------------------------------------
// mma.sync form: head_dim above 128, and rows that 16-byte copies cannot take
// ---------------------------------------------------------------------------
// A CTA takes 64 query rows of one head, 16 a warp, queries and outputs in
// registers; the keys any of its rows sees come 32 at a time through shared
// memory, first the sinks, then from the first row's window on.  Bound by
// mma.sync and by the loads it does not overlap: 8192 tokens, window 2048, 32
// heads of 128 take 2.35 ms this way (the tcgen05 form 0.24), of 256 3.6 ms, of
// 160, padded to 256, 5.0 ms.
constexpr int kWmRows = 64, kWmKeys = 32, kWmThreads = 128;

// 8 elements from p, of which n exist; vec: p is 16-byte aligned
__device__ __forceinline__ uint4 ld8(const uint16_t* p, int n, bool vec) {
    uint4 r = make_uint4(0, 0, 0, 0);
    if (vec && n >= 8) return *reinterpret_cast<const uint4*>(p);
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) w[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
    return r;
}

// DP: head dim rounded up to 64, 128 or 256
template <int DP, bool BF16>
__global__ void __launch_bounds__(kWmThreads) window_mma_kernel(const WinArgs a, int vec) {
    constexpr int ROW = DP * 2, CH = DP / 8;
    extern __shared__ __align__(16) uint8_t smem[];  // K rows, V rows; 16-byte pieces swizzled by the row
    griddep_wait();
    griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lr = lane >> 2, lc = lane & 3;
    const uint32_t sk = smem_addr(smem), sv = sk + kWmKeys * ROW;
    const int tiles = (a.S + kWmRows - 1) / kWmRows, T = a.q_start + a.S;
    const int64_t items = (int64_t)a.batch * tiles * a.nq;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int h = (int)(item % a.nq), tile = tiles - 1 - (int)((item / a.nq) % tiles);
        const int b = (int)(item / ((int64_t)a.nq * tiles)), kvh = h / (a.nq / a.nkv);
        const int len = a.seq_lens ? max(0, min(a.seq_lens[b], T)) : T;
        const int row0 = tile * kWmRows + warp * 16, p0 = a.q_start + tile * kWmRows;  // p0: position of the CTA's first row
        const int pos[2] = {a.q_start + row0 + lr, a.q_start + row0 + lr + 8};
        const uint16_t* K = static_cast<const uint16_t*>(a.k.data) + b * a.k.stride_b + kvh * a.k.stride_h;
        const uint16_t* V = static_cast<const uint16_t*>(a.v.data) + b * a.v.stride_b + kvh * a.v.stride_h;
        uint32_t qa[DP / 16][4];
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = row0 + lr + (e & 1) * 8, col = kk * 16 + lc * 2 + (e >> 1) * 8;
                const uint16_t* q = static_cast<const uint16_t*>(a.q.data) + b * a.q.stride_b + h * a.q.stride_h +
                                    (int64_t)row * a.q.stride_s + col;
                qa[kk][e] = 0u;
                if (row < a.S && col < a.D) qa[kk][e] = q[0];
                if (row < a.S && col + 1 < a.D) qa[kk][e] |= (uint32_t)q[1] << 16;
            }
        float o[DP / 8][4] = {}, m[2] = {-1e30f, -1e30f}, l[2] = {0.f, 0.f};
        const int lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0, hi = min(p0 + kWmRows, len);  // keys lo .. hi - 1
        const int s0 = min(a.sinks, lo);
        if (p0 < len) {
            for (int j0 = s0 > 0 ? 0 : lo; j0 < hi; j0 = j0 < s0 && j0 + kWmKeys >= s0 ? lo : j0 + kWmKeys) {
                const int n = min(kWmKeys, (j0 < s0 ? s0 : hi) - j0);
                __syncthreads();
                for (int i = threadIdx.x; i < kWmKeys * CH; i += kWmThreads) {
                    const int r = i / CH, c = i - r * CH, off = r * ROW + ((c ^ (r & 7)) << 4);
                    const int have = r < n ? a.D - c * 8 : 0;
                    *reinterpret_cast<uint4*>(smem + off) = ld8(K + (int64_t)(j0 + r) * a.k.stride_s + c * 8, have, vec);
                    *reinterpret_cast<uint4*>(smem + kWmKeys * ROW + off) =
                        ld8(V + (int64_t)(j0 + r) * a.v.stride_s + c * 8, have, vec);
                }
                __syncthreads();
                const int mi = lane >> 3, mr = lane & 7;
                float s[4][4] = {};
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {  // 16 keys
                        uint32_t kf[4];
                        ldsm4(kf, sk + (g * 16 + (mi >> 1) * 8 + mr) * ROW + (((kk * 2 + (mi & 1)) ^ mr) << 4));
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float* c = s[2 * g + x];
                            mma16816<BF16>(c[0], c[1], c[2], c[3], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], kf[2 * x],
                                           kf[2 * x + 1]);
                        }
                    }
                float t[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = j0 + x * 8 + lc * 2 + (e & 1), p = pos[e >> 1];
                        const bool sees = x * 8 + lc * 2 + (e & 1) < n && j <= p && p < len &&
                                          (a.window == 0 || j > p - a.window || j < a.sinks);
                        s[x][e] = sees ? s[x][e] * a.scale_log2 : -INFINITY;
                        t[e >> 1] = fmaxf(t[e >> 1], s[x][e]);
                    }
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    t[e] = fmaxf(t[e], __shfl_xor_sync(~0u, t[e], 1));
                    t[e] = fmaxf(fmaxf(t[e], __shfl_xor_sync(~0u, t[e], 2)), m[e]);
                    f[e] = ex2(m[e] - t[e]);
                    m[e] = t[e];
                    l[e] *= f[e];
                }
#pragma unroll
                for (int x = 0; x < DP / 8; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[x][e] *= f[e >> 1];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    uint32_t pa[4];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float* c = s[2 * g + x];
                        const float w0 = ex2(c[0] - m[0]), w1 = ex2(c[1] - m[0]), w2 = ex2(c[2] - m[1]), w3 = ex2(c[3] - m[1]);
                        l[0] += w0 + w1;
                        l[1] += w2 + w3;
                        pa[2 * x] = pack16<BF16>(w0, w1);
                        pa[2 * x + 1] = pack16<BF16>(w2, w3);
                    }
#pragma unroll
                    for (int x = 0; x < DP / 16; ++x) {
                        uint32_t vf[4];
                        ldsm4t(vf, sv + (g * 16 + (mi & 1) * 8 + mr) * ROW + (((x * 2 + (mi >> 1)) ^ mr) << 4));
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            float* c = o[2 * x + y];
                            mma16816<BF16>(c[0], c[1], c[2], c[3], pa[0], pa[1], pa[2], pa[3], vf[2 * y], vf[2 * y + 1]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(~0u, l[e], 1);
            l[e] += __shfl_xor_sync(~0u, l[e], 2);
            const float inv = l[e] > 0.f ? 1.f / l[e] : 0.f;
            const int row = row0 + lr + 8 * e;
            if (row >= a.S) continue;
            uint16_t* out = static_cast<uint16_t*>(a.out) + (((int64_t)b * a.S + row) * a.nq + h) * a.D;
#pragma unroll
            for (int x = 0; x < DP / 8; ++x) {
                const int col = x * 8 + lc * 2;
                const uint32_t w = pack16<BF16>(o[x][2 * e] * inv, o[x][2 * e + 1] * inv);
                if (col < a.D) out[col] = (uint16_t)w;
                if (col + 1 < a.D) out[col + 1] = (uint16_t)(w >> 16);
            }
        }
    }
}

template <int DP, bool BF16>
static int launch_window_mma(const WinArgs& a, int vec, cudaStream_t s) {
    const int64_t items = (int64_t)a.batch * a.nq * (((int64_t)a.S + kWmRows - 1) / kWmRows);
    const unsigned grid = (unsigned)(items < (1 << 30) ? items : 1 << 30);
    B2_TRY(launch(window_mma_kernel<DP, BF16>, dim3(grid), dim3(kWmThreads), 2 * kWmKeys * DP * 2, s, true, a, vec));
    return B2_OK;
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
    static constexpr uint32_t OFF_OUT = OFF_V + ST * TILE;  // 32 rows x 64 outputs per softmax warp
    static constexpr uint32_t OFF_BAR = OFF_OUT + 8 * 4096;
    // above half an SM's shared memory: one CTA, with all 512 TMEM columns, per SM
    static constexpr size_t NEED = OFF_BAR + 512 + 1024;
    static constexpr size_t SMEM = NEED > 122880 ? NEED : 122880;
    // Every SHARE-th pair of exponentials of a tile without masks goes to the FMA pipe: at head dim 64 the SFU (16 a
    // cycle and SM) is what a tile takes longest over (8192 tokens, window 2048, 32 heads: 187 us, 198 without); at
    // 128 the products are, and the chip's power, and it gains nothing (240 us, 237 without)
    static constexpr int SHARE = D == 64 ? 4 : 0;
    // warps 0-7 softmax, 8 TMA, 9 and 10 MMA of tile A and of tile B, 11 idle (a warpgroup gives up registers as a whole)
    static constexpr int THREADS = 384;
};

// The launch gives each of the three warpgroups 168 registers a thread; the
// last one hands part of its share to the two whose threads hold a row of S.
constexpr int kWinRegsFew = 104, kWinRegsMany = 200;
static_assert(kWinRegsFew + 2 * kWinRegsMany <= 3 * 168, "more registers than the block is launched with");

// Bits below position n (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t below(int n) {
    return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
}

// Two floats in a 64-bit register: one instruction for both.
__device__ __forceinline__ uint64_t two(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 one_each(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
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

// 2^x of two numbers on the FMA pipe: x = n + f with n the nearest integer
// (found by adding 1.5 * 2^23, which leaves it in the low mantissa bits), 2^f
// on [-1/2, 1/2] by a degree-4 polynomial (least squares of the relative error
// at Chebyshev nodes: 2.7e-6, far below the 16-bit rounding P gets next), n
// added to the exponent.  Below -126 x counts as -126.  NaN (which fmaxf would
// take for -126 too) gives the largest float: infinity as a 16-bit weight, so
// that it shows in the output.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 ex2_fma(float2 x) {
    const uint64_t y = two(max_nan(x.x, -126.f), max_nan(x.y, -126.f));
    const uint64_t t = add2(y, two(12582912.f, 12582912.f));
    const uint64_t f = fma2(add2(t, two(-12582912.f, -12582912.f)), two(-1.f, -1.f), y);
    uint64_t r = fma2(two(0.00956051f, 0.00956051f), f, two(0.05591704f, 0.05591704f));
    r = fma2(r, f, two(0.24024981f, 0.24024981f));
    r = fma2(r, f, two(0.69312197f, 0.69312197f));
    r = fma2(r, f, two(0.99999919f, 0.99999919f));
    const float2 p = one_each(r), n = one_each(t);
    return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(n.x) << 23)),
                       __int_as_float(__float_as_int(p.y) + (__float_as_int(n.y) << 23)));
}

// One pair of query tiles and the key tiles it visits.  The tiles of a kv head
// -- (128 rows, query head of the group), heads fastest -- are paired in order,
// so A and B are two heads at the same rows, or B is at the next 128 rows.
struct WinItem {
    int b, kvh, len;       // sequence, kv head, tokens of the sequence
    int h[2], row[2];      // head and first query row of A and B
    int p[2];              // the positions of those rows
    bool hasB;
    int loA, nw, ns;       // window tiles loA .. loA + nw - 1 of A, sinks' tiles 0 .. ns - 1
    int nA, n, dB;         // A visits steps 0 .. nA - 1, B steps dB .. n - 1

    static __device__ __forceinline__ int length(const WinArgs& a, int b) {
        const int T = a.q_start + a.S;
        return a.seq_lens ? max(0, min(a.seq_lens[b], T)) : T;
    }
    // Row tiles of a sequence of len tokens that hold a token.
    static __device__ __forceinline__ int tiles(const WinArgs& a, int len) {
        return (max(0, len - a.q_start) + 127) >> 7;
    }

    // Pair i of the kv head's list, of `count` tiles.
    __device__ __forceinline__ void of(const WinArgs& a, int b_, int len_, int kvh_, int i, int count) {
        const int group = a.nq / a.nkv;
        b = b_;
        len = len_;
        kvh = kvh_;
        hasB = !a.single && 2 * i + 1 < count;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int e = a.single ? i : 2 * i + (hasB ? t : 0), rt = e / group;
            h[t] = kvh * group + e - rt * group;
            row[t] = rt * 128;
            p[t] = a.q_start + row[t];
        }
        loA = a.window > 0 ? max(0, p[0] - a.window + 1) >> 7 : 0;
        const int hiA = min(p[0] + 127, len - 1) >> 7, st = a.window > 0 ? (a.sinks + 127) >> 7 : 0;
        nw = hiA - loA + 1;
        ns = min(st, loA);
        nA = nw + ns;
        n = nA;
        dB = 0;
        if (row[1] > row[0]) {
            n += (min(p[1] + 127, len - 1) >> 7) - hiA;
            // B skips A's first tiles, unless they hold sinks
            if (a.window > 0 && loA >= st) dB = (max(0, p[1] - a.window + 1) >> 7) - loA;
        }
    }
    // Key tile of step j.
    __device__ __forceinline__ int tile(int j) const {
        return j < nw ? loA + j : j < nA ? j - nw : j - ns + loA;
    }
    // Keys of step j's tile that query tile t may see, in steps of 16.
    __device__ __forceinline__ int width(const WinArgs& a, int t, int j) const {
        const int kb = tile(j) << 7;
        int end = min(p[t] + 127, len - 1) + 1;
        if (j >= nw && j < nA) end = min(end, a.sinks);
        return min(128, (end - kb + 15) & ~15);
    }
};

// The pairs of all sequences and kv heads, a sequence's later (longer) rows
// first, dealt to the CTAs back and forth: without a window the first CTA of a
// round would otherwise always get its longest pair (8192 tokens, 32 heads: 591
// us dealt one way, 551 back and forth, before the issuers were made quicker).
struct WinList {
    int b = 0, len = 0, count = 0, np = 0;  // of the sequence: tiles and pairs per kv head
    int64_t before = 0;                     // items of sequences before b
    __device__ __forceinline__ bool get(const WinArgs& a, int64_t i, WinItem& it) {
        if (b == 0 && before == 0 && np == 0) enter(a);
        while (b < a.batch && i - before >= (int64_t)np * a.nkv) {
            before += (int64_t)np * a.nkv;
            ++b;
            enter(a);
        }
        if (b >= a.batch) return false;
        const int k = (int)(i - before), pair = k / a.nkv;
        it.of(a, b, len, k - pair * a.nkv, np - 1 - pair, count);
        return true;
    }
    __device__ __forceinline__ void enter(const WinArgs& a) {
        if (b >= a.batch) return;
        len = WinItem::length(a, b);
        count = WinItem::tiles(a, len) * (a.nq / a.nkv);
        np = a.single ? count : (count + 1) >> 1;
    }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(WinCfg<D>::THREADS, 1)
    window_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const WinArgs a,
                     int* err) {
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
    uint64_t* p_lo = s_full + 2;        // [tile]: P of the tile's first 64 keys is in TMEM
    uint64_t* p_hi = p_lo + 2;          // [tile]: and of the others
    uint64_t* o_done = p_hi + 2;        // [tile]: the pair's last P V of the tile is done
    uint64_t* turn = o_done + 2;        // [tile]: its products of the next step may be issued
    uint64_t* i_full = turn + 2;        // [2]: the pair in s_item is the next one
    uint64_t* i_empty = i_full + 2;     // [2]: every warp has read it
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(i_empty + 2);
    __shared__ WinItem s_item[2];       // n 0: no more

    // a value that is the same in all lanes, told to the compiler
    auto same = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
    const int warp = same(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        tc::mbar_init(q_full, 1);
        tc::mbar_init(q_empty, 2);
        for (int s = 0; s < ST; ++s) {
            tc::mbar_init(&k_full[s], 1);
            tc::mbar_init(&k_empty[s], 2);
            tc::mbar_init(&v_full[s], 1);
            tc::mbar_init(&v_empty[s], 2);
        }
        for (int t = 0; t < 2; ++t) {
            tc::mbar_init(&s_full[t], 1);
            tc::mbar_init(&p_lo[t], 128);
            tc::mbar_init(&p_hi[t], 128);
            tc::mbar_init(&o_done[t], 1);
            tc::mbar_init(&turn[t], 1);
            tc::mbar_init(&i_full[t], 1);
            tc::mbar_init(&i_empty[t], 10);  // 2 issuers, 8 softmax warps
        }
        tc::fence_barrier_init();
    }
    if (warp == 0) tc::tmem_alloc(tmem_slot, 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = same(*tmem_slot);

    griddep_wait();
    griddep_launch_dependents();

    uint32_t g = 0;  // key tiles of the pairs before this one
    // Pair k as the producer found it: into `it`, false after the last one.  The whole warp calls it.
    auto next_item = [&](uint32_t k, WinItem& it, bool& ok) -> bool {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(&i_full[k & 1], (k >> 1) & 1u, err, 103));
        if (!ok) return false;
        it = s_item[k & 1];
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&i_empty[k & 1]);
        return it.n > 0;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWinRegsFew));
        if (warp == 8) {
            // ---------------- TMA producer ----------------
            if (lane == 0) {
                // Pair k + 1 is worked out and published while pair k is under way: divisions and a length's load that
                // no other warp has to wait for.
                WinList list;
                WinItem it, ahead;
                auto publish = [&](uint32_t k) -> bool {
                    if (k >= 2 && !tc::mbar_wait(&i_empty[k & 1], ((k >> 1) - 1) & 1u, err, 104)) return false;
                    const uint32_t c = k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
                    if (!list.get(a, (int64_t)k * gridDim.x + c, ahead)) ahead.n = 0;
                    s_item[k & 1] = ahead;
                    tc::mbar_arrive(&i_full[k & 1]);
                    return true;
                };
                bool ok = publish(0);
                for (uint32_t k = 0; ok && ahead.n > 0; ++k) {
                    it = ahead;
                    if (k > 0 && !tc::mbar_wait(q_empty, (k - 1) & 1u, err, 91)) break;
                    tc::mbar_arrive_expect_tx(q_full, 2 * TILE);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
                            tc::tma_load_4d(sQ + t * TILE + c * ATOM, &tmQ, q_full, c * 64, it.h[t], it.row[t], it.b);
                    for (int j = 0; ok && j < it.n; ++j, ++g) {
                        const uint32_t s = g % ST, u = g / ST;
                        const int row = it.tile(j) * 128;
                        if (g >= ST && !(ok = tc::mbar_wait(&k_empty[s], (u - 1) & 1u, err, 92))) break;
                        tc::mbar_arrive_expect_tx(&k_full[s], TILE);
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
                            tc::tma_load_4d(sK + s * TILE + c * ATOM, &tmK, &k_full[s], c * 64, it.kvh, row, it.b);
                        if (g >= ST && !(ok = tc::mbar_wait(&v_empty[s], (u - 1) & 1u, err, 93))) break;
                        tc::mbar_arrive_expect_tx(&v_full[s], TILE);
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
                            tc::tma_load_4d(sV + s * TILE + c * ATOM, &tmV, &v_full[s], c * 64, it.kvh, row, it.b);
                        if (j == 0) ok = publish(k + 1);
                    }
                }
            }
        } else if (warp <= 10) {
            // ---------------- MMA issuers: one warp per tile, so that the tensor core always has the other's
            // products queued while one waits or computes descriptors.  The whole warp runs the control flow.
            constexpr uint32_t idO = tc::idesc_f16(128, D, BF16, true);
            constexpr uint32_t idS = tc::idesc_f16(128, 0, BF16, false);
            const int t = warp - 9;
            const uint32_t tP = tmem + (uint32_t)t * 256, tO = tP + 128;
            // a descriptor's address field counts 16 bytes: steps are added to it
            const uint64_t dq = tc::desc_k_sw128(tc::smem_u32(sQ) + (uint32_t)t * TILE);
            const uint64_t dk0 = tc::desc_k_sw128(tc::smem_u32(sK)), dv0 = tc::desc_mn_sw128(tc::smem_u32(sV), ATOM);
            bool ok = true;
            uint32_t np = 0;  // P tiles consumed
            auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
                return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, err, where)) != 0;
            };
            // Turns: A's products of a step, then B's, and so on.  The other tile's products are in the
            // queue while this warp waits for its own operands, and the two softmaxes stay half a step apart.
            uint32_t turns = 0;
            auto my_turn = [&]() {
                const bool mine = (t == 0 && turns == 0) || wait(&turn[t], (turns - (t == 0)) & 1u, 102);
                ++turns;
                return mine;
            };
            WinItem it;
            for (uint32_t k = 0; ok && next_item(k, it, ok); ++k) {
                const int from = same(t == 0 ? 0 : it.dB), to = same(t == 0 ? it.nA : it.hasB ? it.n : 0), n = same(it.n);
                int w = 0;
                for (int j = -1; j < n; ++j) {
                    const uint32_t gj = g + (uint32_t)j, s = gj % ST, s1 = (gj + 1) % ST;
                    const bool pv = j >= from && j < to, qk = j + 1 >= from && j + 1 < to;
                    const int steps = w >> 4;
                    if (qk) w = same(it.width(a, t, j + 1));
                    if (j + 1 < n)
                        ok = (j >= 0 || wait(q_full, k & 1u, 96)) && wait(&k_full[s1], ((gj + 1) / ST) & 1u, 94);
                    if (j >= 0) ok = ok && wait(&v_full[s], (gj / ST) & 1u, 95);
                    if (pv) ok = ok && wait(&p_lo[t], np & 1u, 97);
                    ok = ok && my_turn();
                    if (!ok) break;
                    tc::fence_after_sync();
                    if (pv) {
                        const uint64_t dv = dv0 + s * (TILE >> 4);
                        if (tc::elect_one()) {
                            tc::mma_f16_ts(tO, tP, dv, idO, j > from ? 1u : 0u);
#pragma unroll
                            for (int kk = 1; kk < 4; ++kk)
                                if (kk < steps) tc::mma_f16_ts(tO, tP + (uint32_t)kk * 8, dv + (uint32_t)kk * 128u, idO, 1u);
                        }
                        if (!(ok = wait(&p_hi[t], np & 1u, 101))) break;
                        ++np;
                        tc::fence_after_sync();
                        if (tc::elect_one()) {
#pragma unroll
                            for (int kk = 4; kk < 8; ++kk)
                                if (kk < steps) tc::mma_f16_ts(tO, tP + (uint32_t)kk * 8, dv + (uint32_t)kk * 128u, idO, 1u);
                            if (j + 1 == to) tc::mma_commit(&o_done[t]);
                        }
                    }
                    if (qk) {
                        const uint64_t dk = dk0 + s1 * (TILE >> 4);
                        const uint32_t id = idS | ((uint32_t)(w >> 3) << 17);
                        if (tc::elect_one()) {
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk) {
                                const uint32_t off = ((uint32_t)(kk >> 2) * ATOM + (uint32_t)(kk & 3) * 32) >> 4;
                                tc::mma_f16(tP, dq + off, dk + off, id, kk > 0 ? 1u : 0u);
                            }
                            tc::mma_commit(&s_full[t]);
                        }
                    }
                    if (tc::elect_one()) {
                        tc::mbar_arrive(&turn[t ^ 1]);
                        // whatever this tile read of the step's K and V has been read once these arrive
                        if (j >= 0) tc::mma_commit(&v_empty[s]);
                        if (j + 1 < n) tc::mma_commit(&k_empty[s1]);
                        if (j + 2 == n) tc::mma_commit(q_empty);
                    }
                    __syncwarp();
                }
                g += (uint32_t)n;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWinRegsMany));
        // ---------------- softmax and output: tile t, one query row per thread ----------------
        const int t = warp >> 2, rq = warp & 3;
        const uint32_t lane_base = (uint32_t)(rq * 32) << 16;
        const uint32_t tS = tmem + (uint32_t)t * 256 + lane_base, tO = tS + 128;
        const uint64_t scale2 = two(a.scale_log2, a.scale_log2);
        bool ok = true;
        uint32_t cs = 0, co = 0;  // S tiles and outputs of this tile so far
        WinItem it;
        for (uint32_t k = 0; ok && next_item(k, it, ok); ++k) {
            const int from = t == 0 ? 0 : it.dB, to = t == 0 ? it.nA : it.hasB ? it.n : 0;
            const int wp = it.p[t] + rq * 32;  // position of the warp's first row
            const int pos = wp + lane < it.len ? wp + lane : -1;
            float m = -1e30f, l = 0.f;  // finite: a row that has seen nothing keeps P = 0 and l = 0
            for (int j = from; j < to; ++j, ++cs) {
                const int kb = it.tile(j) << 7, w = it.width(a, t, j);
                // the tile whole, for every row of the warp?
                const bool whole = w == 128 && kb + 127 <= wp && wp + 31 < it.len &&
                                   (a.window == 0 || kb > wp + 31 - a.window || kb + 128 <= a.sinks);
                if (kb + w > it.len && it.len < a.q_start + a.S) {
                    // rows past the sequence may hold anything: P is 0 there, and V has to be finite
                    const uint32_t gj = g + j, s = gj % ST;
                    ok = __all_sync(0xffffffffu, tc::mbar_wait(&v_full[s], (gj / ST) & 1u, err, 99));
                    if (!ok) break;
                    const int r = rq * 32 + lane;
                    if (kb + r >= it.len) {
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                reinterpret_cast<uint4*>(sV + s * TILE + c * ATOM + r * 128)[q] = make_uint4(0, 0, 0, 0);
                    }
                    tc::fence_proxy_async_smem();
                }
                ok = __all_sync(0xffffffffu, tc::mbar_wait(&s_full[t], cs & 1u, err, 98));
                if (!ok) break;
                tc::fence_after_sync();
                uint32_t v[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tc::tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&v[32 * c]));
                tc::tmem_wait_ld();
                if (!whole) {
                    // visible columns of the row as bits: lo .. hi and those below sk
                    const int hi = pos - kb, lo = a.window > 0 ? hi + 1 - a.window : 0, sk = a.window > 0 ? a.sinks - kb : 0;
                    const int whi = wp - kb, wlo = a.window > 0 ? wp + 32 - a.window - kb : 0;  // what every row sees
                    const bool in = wp + 31 < it.len;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (in && 32 * c + 31 <= whi && (32 * c >= wlo || 32 * c + 32 <= sk)) continue;
                        const uint32_t see = below(hi + 1 - 32 * c) & (~below(lo - 32 * c) | below(sk - 32 * c));
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(see >> e & 1)) v[32 * c + e] = 0xff800000u;  // -inf
                    }
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 128; e += 2)
                    mx4[(e >> 1) & 3] = fmaxf(fmaxf(mx4[(e >> 1) & 3], __uint_as_float(v[e])), __uint_as_float(v[e + 1]));
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;
                const float m_new = fmaxf(m, mx);
                const bool resc = m_new > m + 8.f;
                const float m_use = resc ? m_new : m;
                const float alpha = ex2(m - m_use);
                if (j > from && __any_sync(0xffffffffu, resc)) {
                    // the P V before has completed (S, issued behind it, has)
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        tc::tmem_ld16(tO + c, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tc::tmem_st16(tO + c, o);
                    }
                }
                m = m_use;
                const uint64_t nm2 = two(-m, -m);
                uint64_t l2[2] = {0, 0};
                auto weights = [&](auto masked) {  // columns past w are not read by the product
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (!decltype(masked)::value || 32 * c < w) {
                            uint32_t pk[16];
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                const float2 x = one_each(
                                    fma2(two(__uint_as_float(v[32 * c + e]), __uint_as_float(v[32 * c + e + 1])), scale2, nm2));
                                float2 p;
                                if (!decltype(masked)::value && C::SHARE && (e >> 1) % (C::SHARE ? C::SHARE : 1) == C::SHARE - 1)
                                    p = ex2_fma(x);
                                else p = make_float2(ex2(x.x), ex2(x.y));
                                l2[(e >> 1) & 1] = add2(l2[(e >> 1) & 1], two(p.x, p.y));
                                pk[e >> 1] = pack16<BF16>(p.x, p.y);
                            }
                            tc::tmem_st16(tS + (uint32_t)(16 * c), pk);
                        }
                        if (c & 1) {
                            tc::tmem_wait_st();
                            tc::fence_before_sync();
                            tc::mbar_arrive(c == 1 ? &p_lo[t] : &p_hi[t]);
                        }
                    }
                };
                if (whole) weights(std::false_type());
                else weights(std::true_type());
                const float2 ls = one_each(add2(l2[0], l2[1]));
                l = l * alpha + (ls.x + ls.y);
            }
            if (ok && to > from) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait(&o_done[t], co & 1u, err, 100));
                ++co;
                tc::fence_after_sync();
                const float inv_l = l > 0.f ? 1.f / l : 0.f;
                // 64 outputs of 32 rows at a time leave through shared memory by TMA
                uint8_t* stage = sm + C::OFF_OUT + warp * 4096;
#pragma unroll 1
                for (int c = 0; c < D; c += 64) {
                    uint32_t o[64];
                    tc::tmem_ld32(tO + c, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
                    tc::tmem_ld32(tO + c + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
                    tc::tmem_wait_ld();
                    if (lane == 0) tc::tma_store_wait_read();  // the stage's last store
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        uint4 x;
                        x.x = pack16<BF16>(__uint_as_float(o[8 * q + 0]) * inv_l, __uint_as_float(o[8 * q + 1]) * inv_l);
                        x.y = pack16<BF16>(__uint_as_float(o[8 * q + 2]) * inv_l, __uint_as_float(o[8 * q + 3]) * inv_l);
                        x.z = pack16<BF16>(__uint_as_float(o[8 * q + 4]) * inv_l, __uint_as_float(o[8 * q + 5]) * inv_l);
                        x.w = pack16<BF16>(__uint_as_float(o[8 * q + 6]) * inv_l, __uint_as_float(o[8 * q + 7]) * inv_l);
                        *reinterpret_cast<uint4*>(stage + lane * 128 + ((q ^ (lane & 7)) << 4)) = x;
                    }
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    const int row = it.row[t] + rq * 32;
                    if (ok && lane == 0 && c < a.D && row < a.S) tc::tma_store_4d(&tmO, stage, c, it.h[t], row, it.b);
                }
            }
            g += it.n;
        }
        if (lane == 0) tc::tma_store_wait();
        // rows of tiles past a sequence's end: zeros
        if (a.seq_lens) {
            const int64_t row16 = (int64_t)a.nq * a.D / 8;
            for (int b = 0; b < a.batch; ++b) {
                const int len = WinItem::length(a, b);
                const int done = WinItem::tiles(a, len) * 128;
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

static int window_map(CUtensorMap* m, const b2_kv_view& v, int heads, int64_t rows, uint32_t box_rows, const WinArgs& a,
                      bool bf16) {
    const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)heads, (uint64_t)rows, (uint64_t)a.batch};
    const uint64_t st[3] = {(uint64_t)v.stride_h * 2, (uint64_t)v.stride_s * 2, (uint64_t)v.stride_b * 2};
    const uint32_t box[4] = {64, 1, box_rows, 1};
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
    CUtensorMap tq, tk, tv, to;
    int rc = window_map(&tq, a.q, a.nq, a.S, 128, a, BF16);
    if (rc == B2_OK) rc = window_map(&tk, a.k, a.nkv, T, 128, a, BF16);
    if (rc == B2_OK) rc = window_map(&tv, a.v, a.nkv, T, 128, a, BF16);
    const b2_kv_view out = {a.out, (int64_t)a.S * a.nq * a.D, a.D, (int64_t)a.nq * a.D, 1};
    if (rc == B2_OK) rc = window_map(&to, out, a.nq, a.S, 32, a, BF16);
    if (rc != B2_OK) return rc;
    auto kern = window_tc_kernel<D, BF16>;
    static bool done[64];
    B2_TRY(allow_smem(kern, (int)C::SMEM, done));
    // with no more tiles than SMs a tile to each is quicker than two to half of them (77 rows of 14 heads: 5.8 us, 7.2 paired)
    const int64_t tiles = ((int64_t)a.S + 127) / 128 * (a.nq / a.nkv);
    a.single = tiles * a.nkv * a.batch <= sm_count();
    const int64_t items = (int64_t)a.batch * a.nkv * (a.single ? tiles : (tiles + 1) / 2);
    const unsigned grid = (unsigned)(items < sm_count() ? items : sm_count());
    B2_TRY(launch(kern, dim3(grid), dim3(C::THREADS), C::SMEM, s, true, tq, tk, tv, to, a, err));
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
    if (D > 256 || q_len > (1 << 30) || q_start > (1 << 30) - q_len || q.stride_d != 1 || k.stride_d != 1 || v.stride_d != 1)
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
    // 16-byte loads where every row is aligned for them
    auto rows16 = [](const b2_kv_view& x) { return aligned16(x.data) && !((x.stride_b | x.stride_h | x.stride_s) & 7); };
    const int vec = rows16(k) && rows16(v);
    cudaStream_t s = as_stream(stream);
    if (D <= 64) return bf16 ? launch_window_mma<64, true>(a, vec, s) : launch_window_mma<64, false>(a, vec, s);
    if (D <= 128) return bf16 ? launch_window_mma<128, true>(a, vec, s) : launch_window_mma<128, false>(a, vec, s);
    return bf16 ? launch_window_mma<256, true>(a, vec, s) : launch_window_mma<256, false>(a, vec, s);
}
