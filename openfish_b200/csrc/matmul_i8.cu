// matmul_i8.cu -- product of tokens and weights in 8-bit integers (openfish_b200_matmul_i8).
//
//   out[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n]
#include <stdint.h>

#include "encoder_device.cuh"

namespace {

constexpr int kTile = 64, kDepth = 64;

template <class T>
__global__ void __launch_bounds__(256) matmul_simple_kernel(const openfish_b200_matmul_i8_t a) {
    __shared__ int sx[kTile][kDepth / 4 + 1], sw[kTile][kDepth / 4 + 1];
    const long long m0 = (long long)blockIdx.x * kTile;
    const int n0 = blockIdx.y * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.depth; k0 += kDepth) {
        for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
            const int row = i / kDepth, k = i % kDepth;
            const bool in = k0 + k < a.depth;
            reinterpret_cast<int8_t *>(&sx[row][0])[k] = in && m0 + row < a.rows ? a.x[(m0 + row) * a.x_stride + k0 + k] : 0;
            reinterpret_cast<int8_t *>(&sw[row][0])[k] = in && n0 + row < a.cols ? a.w[(n0 + row) * a.w_stride + k0 + k] : 0;
        }
        __syncthreads();
        for (int k = 0; k < kDepth / 4; ++k)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sx[ty * 4 + i][k], sw[tx * 4 + j][k], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const long long m = m0 + ty * 4 + i;
            const int n = n0 + tx * 4 + j;
            if (m >= a.rows || n >= a.cols) continue;
            float y = (float)acc[i][j] * (a.x_scale[m] * a.w_scale[n]);
            if (a.bias) y += ofe::to_float(static_cast<const T *>(a.bias)[n]);
            static_cast<T *>(a.out)[m * a.out_stride + n] = ofe::from_float<T>(y);
        }
}

}  // namespace

extern "C" size_t ofb_matmul_i8_workspace(const openfish_b200_matmul_i8_t *) { return 0; }

extern "C" int ofb_matmul_i8(void *stream, const openfish_b200_matmul_i8_t *a) {
    const dim3 grid((unsigned)((a->rows + kTile - 1) / kTile), (unsigned)((a->cols + kTile - 1) / kTile));
    if (a->dtype == OPENFISH_B200_F16) matmul_simple_kernel<__half><<<grid, 256, 0, (cudaStream_t)stream>>>(*a);
    else matmul_simple_kernel<__nv_bfloat16><<<grid, 256, 0, (cudaStream_t)stream>>>(*a);
    return ofe::launched();
}
