// encoder_device.cuh -- what the encoder's operators share: their two types, the status word of a device, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "encoder.h"

namespace ofe {

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline int cuda_status(cudaError_t e) {
    return e == cudaSuccess ? OPENFISH_B200_OK : ofb_fail(OPENFISH_B200_ERR_CUDA, cudaGetErrorString(e));
}
inline int launched() { return cuda_status(cudaGetLastError()); }
inline int sm_count(int *out) {
    int dev = 0;
    if (const int rc = cuda_status(cudaGetDevice(&dev))) return rc;
    return cuda_status(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
}
// Waits for the stream, then reads a file's status word and clears it.
inline int settle(cudaStream_t stream, const int &symbol, int *gave_up) {
    int seen = 0;
    const int none = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&seen, symbol, sizeof(seen), 0, cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e == cudaSuccess && seen) {
        e = cudaMemcpyToSymbolAsync(symbol, &none, sizeof(none), 0, cudaMemcpyHostToDevice, stream);
        if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    }
    *gave_up = seen != 0;
    return cuda_status(e);
}

}  // namespace ofe
