// paged_split.cuh -- how attention over a paged cache spreads the visible
// positions of all (sequence, kv head) pairs over the CTAs of one grid, and how
// a pair's pieces are joined.  Shared by the caches of 16-bit rows
// (paged_attn.cu) and of 4-bit rows (kv4_attn.cu).
//
// A (sequence, kv head, group of heads) is a segment of units of U positions.
// Every CTA of a grid that is resident at once takes an equal share of the
// units, in one of two ways.  Pieces: every segment is cut into pieces of the
// same size, one per CTA, when a size within an eighth (or two units) of the
// even share gives no more pieces than CTAs -- one segment end per CTA.
// Stream-K otherwise: all units end to end, cut evenly, whatever the lengths --
// up to three segment ends per CTA but no idle ones.  A CTA that covers a
// segment writes its outputs; a segment cut between CTAs leaves a partial (max,
// sum, unnormalised output) per piece in the workspace, and the CTA that
// arrives last at the segment's counter adds the pieces in order (same bits
// whoever is last).
#pragma once

#include "mma.cuh"
#include "paged.cuh"
#include "workspace.cuh"

namespace b2 {

constexpr int kPgWarps = 4;
constexpr int kPgThreads = kPgWarps * 32;

struct SplitArgs {
    const int* block_tables;
    const int* seq_lens;
    int num_blocks, block_size, max_blocks;
    BlockDiv div;
    // LIST: the blocks of its sequence that each (sequence, kv head) sees, [batch][nkv][listed]
    const int* blocks;
    int listed;
    int batch, nq, nkv, D, group, hg, gs, window, sinks;
    void* out;      // [batch][nq][D]
    float* parts;   // [2 * grid][gs][D], unnormalised partial outputs
    float2* pml;    // [2 * grid][gs], their (max, sum)
    int* counters;  // [grid], null: segments are not cut
    float2* stats;  // [batch][nq], the joined (max, sum); scores only
};

// Rows are read once: they leave the L2 first, and what the call reads again
// (logits, partial results, tables) stays (8 x 4096 with weights: 30.4 us, 32.2
// without).
__device__ __forceinline__ uint64_t read_once() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
// 16 bytes, or 16 zero bytes without reading src
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
                 "r"(there ? 16 : 0), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void store4(void* p, int64_t i, float4 v, float scale) {
    const uint2 x = make_uint2(pack16<BF16>(v.x * scale, v.y * scale), pack16<BF16>(v.z * scale, v.w * scale));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = x;
}

// What the newest token of a sequence of L tokens sees, in units of U
// positions: ns units over the first s0 positions, then units from w0 (lo
// rounded down to 16) on, of which positions lo .. L-1 count.  A sequence
// that sees nothing still has one unit, which writes its zeros.
// LIST: units over the positions of the listed blocks, end to end; which of
// them count depends on the list.  Of a sequence of nb blocks the first nb
// entries count at most (s0 says how many): units for the padding of short
// sequences would be most of the work (8 sequences of 272 tokens, 32 K/V heads, 44
// blocks of 128 listed: 11 us with, 77 without this).
template <int U, bool LIST = false>
struct Seen {
    int L, lo, s0, ns, w0, n;
    __device__ __forceinline__ void of(const SplitArgs& a, int b) {
        L = max(0, min(a.seq_lens[b], a.max_blocks * a.block_size));
        if constexpr (LIST) {
            lo = ns = w0 = 0;
            s0 = min(a.listed, L > 0 ? a.div.block(L - 1) + 1 : 0);
            n = max(1, (s0 * a.block_size + U - 1) / U);
        } else {
            lo = a.window > 0 ? max(0, L - a.window) : 0;
            s0 = min(a.sinks, lo);
            ns = (s0 + U - 1) / U;
            w0 = lo & ~15;
            n = max(1, ns + (L - w0 + U - 1) / U);
        }
    }
    __device__ __forceinline__ int base(int u) const { return u < ns ? u * U : w0 + (u - ns) * U; }
    __device__ __forceinline__ bool sees(int u, int pos) const { return u < ns ? pos < s0 : pos >= lo && pos < L; }
};

// A place in the list of all units: head group g of kv head kvh of sequence b,
// unit u of that segment.
template <int U, bool LIST = false>
struct Place {
    int b, kvh, g, u;
    Seen<U, LIST> s;
    __device__ __forceinline__ void next(const SplitArgs& a) {
        if (++u < s.n) return;
        u = 0;
        if (++g < a.hg) return;
        g = 0;
        if (++kvh < a.nkv) return;
        kvh = 0;
        if (++b < a.batch) s.of(a, b);
    }
    // First query head of the segment, and how many it has.
    __device__ __forceinline__ int head0(const SplitArgs& a) const { return kvh * a.group + g * a.gs; }
    __device__ __forceinline__ int heads(const SplitArgs& a) const { return min(a.gs, a.group - g * a.gs); }
};

struct SplitShared {
    int scan[kPgWarps], count[kPgWarps][8];
    int b, before, last;
};

// A CTA's share: units r0 .. r1 - 1, counted from the first one of its segment
// (pieced) or of all.
struct Share {
    int r0, r1;
    bool pieced;
    int upc;         // units per CTA
    int cf, pieces;  // first CTA of the segment and how many share it (pieced only)
};

// The share of CTA c and the place where it starts; false if it has none.  The
// whole CTA calls it.
template <int U, bool LIST>
__device__ __forceinline__ bool split_units(const SplitArgs& a, SplitShared& sh, Share& w, Place<U, LIST>& at) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int c = blockIdx.x, grid = (int)gridDim.x;
    const int heads = a.nkv * a.hg;
    int total, upc, first;   // units of all segments (or pieces); units per CTA; what this CTA starts with
    bool pieced = false;     // equal pieces: first counts pieces, else units
    int fb, fbefore;         // the sequence it lies in, what lies before that
    const bool can_piece = a.counters && (int64_t)a.batch * heads <= grid;
    // the k-th candidate for the size of equal pieces; those up to an eighth or two units above the even share are taken
    // (two of the 16-bit rows' 64 positions; of units of 256 that can be a third of the work: 8 x 4096 tokens in 4 bits take
    // 4 units on 232 CTAs where 2.9 on 296 are even)
    auto size_of = [&](int k) { return upc + k * ((upc + 63) / 64); };
    auto near = [&](int k) { return k * ((upc + 63) / 64) <= max(2, upc / 8); };
    if (a.batch <= 32) {
        // every warp by itself, lane b for sequence b
        Seen<U, LIST> s;
        s.n = 0;
        if (lane < a.batch) s.of(a, lane);
        total = __reduce_add_sync(~0u, s.n) * heads;
        upc = (total + grid - 1) / grid;
        int here = s.n * heads;
        if (can_piece && total <= grid) {
            pieced = true;  // a CTA for every unit
        } else if (can_piece) {
            int pick = -1;
#pragma unroll
            for (int k = 7; k >= 0; --k) {  // (the sum over the warp whatever near() says)
                const int all = (int)__reduce_add_sync(~0u, (unsigned)(s.n + size_of(k) - 1) / (unsigned)size_of(k)) * heads;
                if (all <= grid && near(k)) pick = k;
            }
            if (pick >= 0) {
                pieced = true;
                upc = size_of(pick);
                here = (int)((unsigned)(s.n + upc - 1) / (unsigned)upc) * heads;
            }
        }
        int incl = here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, incl, o);
            if (lane >= o) incl += v;
        }
        total = __shfl_sync(~0u, incl, 31);
        first = pieced ? c : c * upc;
        if (first >= total) return false;
        fb = __ffs(__ballot_sync(~0u, incl > first)) - 1;
        fbefore = __shfl_sync(~0u, incl - here, fb);
    } else {
        const int per = (a.batch + kPgThreads - 1) / kPgThreads;
        const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
        // Sum of count(units) over the sequences before this thread's own and with them, and over all.
        auto scan = [&](auto count) -> int2 {
            int mine = 0;
            for (int b = b0; b < b1; ++b) {
                Seen<U, LIST> s;
                s.of(a, b);
                mine += count(s.n);
            }
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(~0u, incl, o);
                if (lane >= o) incl += v;
            }
            __syncthreads();
            if (lane == 31) sh.scan[warp] = incl;
            __syncthreads();
            total = 0;
#pragma unroll
            for (int v = 0; v < kPgWarps; ++v) {
                if (v < warp) incl += sh.scan[v];
                total += sh.scan[v];
            }
            return make_int2(incl - mine, incl);
        };
        int2 span = scan([&](int n) { return n * heads; });
        upc = (total + grid - 1) / grid;
        if (can_piece) {
            const int size = size_of(tid & 7);
            int n = 0, pick = -1;
            for (int b = tid >> 3; b < a.batch; b += kPgThreads / 8) {
                Seen<U, LIST> s;
                s.of(a, b);
                n += (s.n + size - 1) / size * heads;
            }
            n += __shfl_xor_sync(~0u, n, 8);
            n += __shfl_xor_sync(~0u, n, 16);
            if (lane < 8) sh.count[warp][lane] = n;
            __syncthreads();
            for (int k = 7; k >= 0; --k) {
                int all = 0;
#pragma unroll
                for (int v = 0; v < kPgWarps; ++v) all += sh.count[v][k];
                if (all <= grid && near(k)) pick = k;
            }
            if (pick >= 0) {
                pieced = true;
                upc = size_of(pick);
                span = scan([&](int n) { return (n + upc - 1) / upc * heads; });
            }
        }
        first = pieced ? c : c * upc;
        if (first >= total) return false;
        if (first >= span.x && first < span.y) {  // one thread
            int b = b0, before = span.x;
            for (;; ++b) {
                Seen<U, LIST> s;
                s.of(a, b);
                const int here = (pieced ? (s.n + upc - 1) / upc : s.n) * heads;
                if (first < before + here) break;
                before += here;
            }
            sh.b = b;
            sh.before = before;
        }
        __syncthreads();
        fb = sh.b;
        fbefore = sh.before;
    }
    at.b = fb;
    at.s.of(a, at.b);
    {
        w.pieces = pieced ? (at.s.n + upc - 1) / upc : at.s.n;
        const int hh = (first - fbefore) / w.pieces, rest = first - fbefore - hh * w.pieces;
        w.cf = c - rest;
        at.u = pieced ? rest * upc : rest;
        at.kvh = hh / a.hg;
        at.g = hh - at.kvh * a.hg;
        w.r0 = pieced ? at.u : first;
        w.r1 = min(pieced ? at.s.n : total, w.r0 + upc);
    }
    w.pieced = pieced;
    w.upc = upc;
    if (!a.counters) {  // whole segments only: those that begin in the range
        if (at.u > 0) {
            w.r0 += at.s.n - at.u;
            at.u = at.s.n - 1;
            at.next(a);
        }
        if (w.r0 >= w.r1) return false;
        // the end moves to the end of the segment that holds unit r1 - 1
        Place<U, LIST> e = at;
        int r = w.r0;
        while (r < w.r1) {
            r += e.s.n;
            e.u = e.s.n - 1;
            e.next(a);
        }
        w.r1 = r;
    }
    return true;
}

// The end of a segment or of a CTA's piece of it, with its sum(row, d) (4
// outputs of a head, unnormalised) and (max, sum) ml[row] in shared memory: the
// outputs, or the piece to the workspace and, from the last of the segment's
// CTAs to arrive, the join.  r: the unit just done, piece0: the first one of
// the piece.  The whole CTA calls it.
template <int U, bool LIST, typename Store, typename Sum>
__device__ __forceinline__ void finish_piece(const SplitArgs& a, SplitShared& sh, Share& w, const Place<U, LIST>& at,
                                             int r, int piece0, const float2* ml, Sum sum, Store store) {
    const int tid = threadIdx.x, c = blockIdx.x;
    const bool done = at.u == at.s.n - 1;
    const int h0 = at.head0(a), nh = at.heads(a);
    const int64_t oat = ((int64_t)at.b * a.nq + h0) * a.D;
    const int seg0 = r - at.u;  // first unit of the segment
    const int quads = a.D / 4;
    if (done && piece0 == seg0) {
        for (int i = tid; i < nh * quads; i += kPgThreads) {
            const int row = i / quads, d = (i - row * quads) * 4;
            const float Ls = ml[row].y;
            store(oat + row * a.D + d, sum(row, d), Ls > 0.f ? 1.f / Ls : 0.f);
        }
        if (a.stats && tid < nh) a.stats[(int64_t)at.b * a.nq + h0 + tid] = ml[tid];
        return;
    }
    const int slot = 2 * c + (piece0 == seg0 ? 1 : 0);
    float* part = a.parts + (int64_t)slot * a.gs * a.D;
    for (int i = tid; i < nh * quads; i += kPgThreads) {
        const int row = i / quads, d = (i - row * quads) * 4;
        *reinterpret_cast<float4*>(part + row * a.D + d) = sum(row, d);
    }
    if (tid < nh) a.pml[(int64_t)slot * a.gs + tid] = ml[tid];
    if (!w.pieced) {
        w.cf = seg0 / w.upc;
        w.pieces = (seg0 + at.s.n - 1) / w.upc - w.cf + 1;
    }
    __syncthreads();
    if (tid == 0) {  // (the barrier orders the CTA's writes before this thread's fence)
        __threadfence();
        sh.last = atomicAdd(a.counters + w.cf, 1) == w.pieces - 1;
        __threadfence();
    }
    __syncthreads();
    if (!sh.last) return;
    // last of the segment's CTAs: its pieces in order.  Piece p is in slot 2 (cf + p), the first one in the slot after
    if (tid == 0) a.counters[w.cf] = 0;
    const float2* ml0 = a.pml + (int64_t)2 * w.cf * a.gs;
    const float* part0 = a.parts + (int64_t)2 * w.cf * a.gs * a.D;
    for (int i = tid; i < nh * quads; i += kPgThreads) {
        const int row = i / quads, d = (i - row * quads) * 4;
        float M = -1e30f, Ls = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int p = 0; p < w.pieces; ++p) {
            const int64_t sl = (int64_t)(2 * p + (p == 0)) * a.gs + row;
            const float4 x = __ldcg(reinterpret_cast<const float4*>(part0 + sl * a.D + d));
            const float2 l = __ldcg(&ml0[sl]);
            const float m = fmaxf(M, l.x), f = ex2(M - m), g = ex2(l.x - m);
            M = m;
            Ls = fmaf(Ls, f, l.y * g);
            v = make_float4(fmaf(v.x, f, x.x * g), fmaf(v.y, f, x.y * g), fmaf(v.z, f, x.z * g), fmaf(v.w, f, x.w * g));
        }
        store(oat + row * a.D + d, v, Ls > 0.f ? 1.f / Ls : 0.f);
        if (a.stats && d == 0) a.stats[(int64_t)at.b * a.nq + h0 + row] = make_float2(M, Ls);
    }
}

}  // namespace b2
