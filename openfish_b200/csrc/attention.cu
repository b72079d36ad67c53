// attention.cu -- attention over packed sequences (openfish_b200_attention).
#include <math.h>
#include <stdint.h>

#include "encoder_device.cuh"

namespace {

// A sequence's rows in a tensor of `rows`, cut to the room there is.
__device__ __forceinline__ void span(const int32_t *start, const int32_t *used, int s, long long rows, int most, int *first, int *count) {
    const long long lo = min(max((long long)start[s], 0LL), rows), hi = min(max((long long)start[s + 1], lo), rows);
    long long n = hi - lo;
    if (used) n = min(n, max((long long)used[s], 0LL));
    *first = (int)lo;
    *count = (int)min(n, (long long)most);
}

// A warp to a query and head: 32 keys at a time, a lane to a key for the scores, a lane to four elements for the sum.
template <class T>
__global__ void __launch_bounds__(128) attention_simple_kernel(const openfish_b200_attention_t a) {
    const int lane = threadIdx.x & 31;
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int i = (int)(at / a.q_heads), h = (int)(at % a.q_heads);
    for (int s = blockIdx.y; s < a.sequences; s += gridDim.y) {
    int q0, nq, k0, nk;
    span(a.q_start, a.q_used, s, a.q_rows, a.max_q, &q0, &nq);
    span(a.k_start, a.k_used, s, a.k_rows, a.max_k, &k0, &nk);
    if (i >= nq) continue;
    const int kh = h / (a.q_heads / a.kv_heads);
    const T *q = static_cast<const T *>(a.q) + (long long)(q0 + i) * a.q_stride_row + h * a.q_stride_head;
    const T *k = static_cast<const T *>(a.k) + (long long)k0 * a.k_stride_row + kh * a.k_stride_head;
    const T *v = static_cast<const T *>(a.v) + (long long)k0 * a.v_stride_row + kh * a.v_stride_head;
    T *o = static_cast<T *>(a.out) + (long long)(q0 + i) * a.out_stride_row + h * a.out_stride_head;
    const int place = i + nk - nq;
    const int lo = a.window_left < 0 ? 0 : (int)max((long long)place - a.window_left, 0LL);
    const int hi = a.window_right < 0 ? nk : (int)min((long long)place + a.window_right + 1, (long long)nk);
    float top = -INFINITY, total = 0.f, acc[4] = {};
    for (int j0 = lo; j0 < hi; j0 += 32) {
        const int j = j0 + lane;
        float z = -INFINITY;
        if (j < hi) {
            z = 0.f;
            for (int d = 0; d < a.head_dim; ++d) z = fmaf(ofe::to_float(q[d]), ofe::to_float(k[(long long)j * a.k_stride_row + d]), z);
            z *= a.scale;
        }
        float m = z;
        for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        m = fmaxf(m, top);
        const float fade = top == m ? 1.f : expf(top - m), p = j < hi ? expf(z - (m == -INFINITY ? 0.f : m)) : 0.f;
        top = m;
        float t = p;
        for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
        total = total * fade + t;
        for (int c = 0; c < 4; ++c) acc[c] *= fade;
        for (int n = 0; n < 32 && j0 + n < hi; ++n) {
            const float pn = __shfl_sync(0xffffffffu, p, n);
            for (int c = 0; c < 4; ++c)
                if (c * 32 + lane < a.head_dim) acc[c] = fmaf(pn, ofe::to_float(v[(long long)(j0 + n) * a.v_stride_row + c * 32 + lane]), acc[c]);
        }
    }
    for (int c = 0; c < 4; ++c)
        if (c * 32 + lane < a.head_dim) o[c * 32 + lane] = ofe::from_float<T>(hi > lo ? acc[c] / total : 0.f);
    }
}

__device__ int g_status;  // of the kernels on this device: a wait that ran out

}  // namespace

extern "C" size_t ofb_attention_workspace(const openfish_b200_attention_t *) { return 0; }

extern "C" int ofb_attention(void *stream, const openfish_b200_attention_t *a) {
    const dim3 grid((unsigned)(((long long)a->max_q * a->q_heads + 3) / 4), a->sequences < 65535 ? a->sequences : 65535);
    if (a->dtype == OPENFISH_B200_F16) attention_simple_kernel<__half><<<grid, 128, 0, (cudaStream_t)stream>>>(*a);
    else attention_simple_kernel<__nv_bfloat16><<<grid, 128, 0, (cudaStream_t)stream>>>(*a);
    return ofe::launched();
}

extern "C" int ofb_attention_settle(void *stream, int *gave_up) { return ofe::settle((cudaStream_t)stream, g_status, gave_up); }
