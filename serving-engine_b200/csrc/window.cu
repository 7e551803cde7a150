// window.cu -- causal GQA attention of a chunk of query tokens with a sliding
// window and sinks (operator API window_prefill_gqa).
//
//   out_i = sum_j p_ij v_j,  p_i = softmax over {j <= i : i - j < W or j < K}
//   of q_i . k_j / sqrt(D)
#include <cmath>

#include "common.cuh"

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
    const int64_t warps = q_len * nq * batch;
    int64_t blocks = (warps + 7) / 8;
    if (blocks > (int64_t)sm_count() * 64) blocks = (int64_t)sm_count() * 64;
    B2_TRY(launch(bf16 ? window_rows_kernel<true> : window_rows_kernel<false>, dim3((unsigned)blocks), dim3(256), 0,
                  as_stream(stream), true, a));
    return B2_OK;
}
