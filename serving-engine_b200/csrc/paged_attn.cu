// paged_attn.cu -- GQA attention of the newest token of each sequence over a
// paged K/V cache, with window, sinks and accumulated attention weights
// (operator API paged_decode_gqa).
//
//   out = sum_i p_i v_i,  p = softmax over the visible positions of
//   q . k_i / sqrt(D);  score_i += sum over the group's heads of p_i
#include <cmath>

#include "paged.cuh"
#include "workspace.cuh"

namespace b2 {

struct PagedArgs {
    const void* q;
    int64_t ldq;
    b2_paged_kv kv;
    void* out;
    float* scores;
    int nq, nkv, D, window, sinks;
    float scale_log2;
    float2* stats;  // [batch][nq]: (max, sum) of the softmax in the log2 domain
};

template <bool BF16>
__device__ __forceinline__ float ld16f(const void* p, int64_t i) {
    if constexpr (BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

// The positions that the newest token of a sequence of L sees, numbered 0 ..
// n-1: the first s0, then those from lo on.
struct Seen {
    int L, lo, s0, n;
    __device__ Seen(const PagedArgs& a, int b) {
        L = paged_len(a.kv, b);
        lo = a.window > 0 ? max(0, L - a.window) : 0;
        s0 = min(a.sinks, lo);
        n = s0 + L - lo;
    }
    __device__ int pos(int i) const { return i < s0 ? i : i - s0 + lo; }
};

__device__ __forceinline__ int64_t paged_row(const b2_paged_kv& kv, int b, int kvh, int pos) {
    const int blk = kv.block_tables[(int64_t)b * kv.max_blocks + pos / kv.block_size];
    if (blk < 0 || blk >= kv.num_blocks) return -1;
    return blk * kv.stride_block + (pos % kv.block_size) * kv.stride_slot + kvh * kv.stride_head;
}

// One warp per (sequence, query head), lane l holding elements l, l + 32, ..
template <bool BF16>
__global__ void __launch_bounds__(32) paged_rows_kernel(const PagedArgs a) {
    griddep_wait();
    const int h = blockIdx.x, b = blockIdx.y, kvh = h / (a.nq / a.nkv), lane = threadIdx.x;
    const Seen seen(a, b);
    float q[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        q[e] = lane + 32 * e < a.D ? ld16f<BF16>(a.q, b * a.ldq + (int64_t)h * a.D + lane + 32 * e) : 0.f;
        o[e] = 0.f;
    }
    for (int i = 0; i < seen.n; ++i) {
        const int64_t r = paged_row(a.kv, b, kvh, seen.pos(i));
        if (r < 0) continue;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < a.D) s = fmaf(q[e], ld16f<BF16>(a.kv.k, r + lane + 32 * e), s);
        s = warp_sum(s) * a.scale_log2;
        const float m_new = fmaxf(m, s);
        const float al = exp2f(m - m_new), p = exp2f(s - m_new);
        m = m_new;
        l = fmaf(l, al, p);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < a.D) o[e] = fmaf(o[e], al, p * ld16f<BF16>(a.kv.v, r + lane + 32 * e));
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int64_t at = ((int64_t)b * a.nq + h) * a.D + lane;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (lane + 32 * e >= a.D) continue;
        if constexpr (BF16) static_cast<__nv_bfloat16*>(a.out)[at + 32 * e] = __float2bfloat16_rn(o[e] * inv);
        else static_cast<__half*>(a.out)[at + 32 * e] = __float2half_rn(o[e] * inv);
    }
    if (a.scores && lane == 0) a.stats[(int64_t)b * a.nq + h] = make_float2(m, l);
}

// One warp per (sequence, kv head, 32nd of the positions): the group's weights
// of each position, in head order.
template <bool BF16>
__global__ void __launch_bounds__(32) paged_rows_scores_kernel(const PagedArgs a) {
    griddep_wait();
    const int kvh = blockIdx.x, b = blockIdx.y, g = a.nq / a.nkv, lane = threadIdx.x;
    const Seen seen(a, b);
    for (int i = blockIdx.z; i < seen.n; i += gridDim.z) {
        const int pos = seen.pos(i);
        const int64_t r = paged_row(a.kv, b, kvh, pos);
        if (r < 0) continue;
        float w = 0.f;
        for (int h = kvh * g; h < (kvh + 1) * g; ++h) {
            float s = 0.f;
            for (int d = lane; d < a.D; d += 32)
                s = fmaf(ld16f<BF16>(a.q, b * a.ldq + (int64_t)h * a.D + d), ld16f<BF16>(a.kv.k, r + d), s);
            const float2 st = a.stats[(int64_t)b * a.nq + h];
            w += exp2f(warp_sum(s) * a.scale_log2 - st.x) / st.y;
        }
        if (lane == 0) {
            const int bs = a.kv.block_size, blk = a.kv.block_tables[(int64_t)b * a.kv.max_blocks + pos / bs];
            float* sc = a.scores + ((int64_t)blk * a.nkv + kvh) * bs + pos % bs;
            *sc = pos == seen.L - 1 ? w : *sc + w;
        }
    }
}

}  // namespace b2

extern "C" size_t b2_paged_decode_workspace_bytes(int batch, int nq, int nkv, int D, int64_t max_positions,
                                                  int scored) {
    if (batch <= 0 || nq <= 0 || nkv <= 0 || nq % nkv || D <= 0 || max_positions < 0) return 0;
    return scored ? (size_t)batch * nq * sizeof(float2) : 0;
}

extern "C" int b2_paged_decode_gqa(const void* q, int64_t ldq, const b2_paged_kv* kv, void* out, float* scores,
                                   int batch, int nq, int nkv, int D, int window, int sinks, b2_workspace* ws,
                                   void* stream) {
    using namespace b2;
    if (batch <= 0) return B2_OK;
    B2_REQUIRE(q && out && nq > 0 && nkv > 0 && nq % nkv == 0 && window >= 0 && sinks >= 0);
    const int rc = check_paged(kv, nkv, D);
    if (rc != B2_OK) return rc;
    if (!aligned16(q) || !aligned16(out) || (ldq & 7) || batch > 65535 || nkv > 65535) return B2_ERR_UNSUPPORTED;
    PagedArgs a = {};
    a.q = q;
    a.ldq = ldq;
    a.kv = *kv;
    a.out = out;
    a.scores = scores;
    a.nq = nq;
    a.nkv = nkv;
    a.D = D;
    a.window = window;
    a.sinks = sinks;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)D);
    if (scores) {
        if (!ws || ws->bytes < b2_paged_decode_workspace_bytes(batch, nq, nkv, D, 0, 1)) return B2_ERR_WORKSPACE;
        a.stats = static_cast<float2*>(ws->ptr);
    }
    cudaStream_t s = as_stream(stream);
    B2_TRY(launch(kv->bf16 ? paged_rows_kernel<true> : paged_rows_kernel<false>, dim3(nq, batch), dim3(32), 0, s, true,
                  a));
    if (scores)
        B2_TRY(launch(kv->bf16 ? paged_rows_scores_kernel<true> : paged_rows_scores_kernel<false>, dim3(nkv, batch, 32),
                      dim3(32), 0, s, true, a));
    return B2_OK;
}
