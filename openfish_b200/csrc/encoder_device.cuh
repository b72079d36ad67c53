// encoder_device.cuh -- what the encoder's operators share: their two types, the reports of waits that have run out, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "encoder.h"
#include "reports.h"

namespace ofe {

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Division of numbers below 2^30 by a number that the host knows: a multiplication, an addition and a shift (the quotient is
// exact: Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
struct Divider {
    uint32_t mul, shift;
    explicit Divider(uint32_t d = 1) {
        shift = 0;
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ int quotient(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
};

// Two 16-bit numbers in a register, and back.
template <class T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <class T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// Two fp32 operations in an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 y;
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%6, %7};\n\t"
        "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "=f"(y.x), "=f"(y.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 y;
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "=f"(y.x), "=f"(y.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return y;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 y;
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "=f"(y.x), "=f"(y.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return y;
}

inline int cuda_status(cudaError_t e) {
    return e == cudaSuccess ? OPENFISH_B200_OK : ofb_fail(OPENFISH_B200_ERR_CUDA, cudaGetErrorString(e));
}
inline int launched() { return cuda_status(cudaGetLastError()); }
// The current device's, and which one that is.
inline int sm_count(int *out, int *device = nullptr) {
    int dev = 0;
    if (const int rc = cuda_status(cudaGetDevice(&dev))) return rc;
    if (device) *device = dev;
    return cuda_status(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
}
// Waits for the stream, then reads a file's count of waits that have run out: whether that is news to the calling thread.
inline int settle(cudaStream_t stream, const int &symbol, Reports &reports, int *known, int *gave_up) {
    int seen = 0, dev = 0;
    *gave_up = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&seen, symbol, sizeof(seen), 0, cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e == cudaSuccess) *gave_up = reports.take(dev, known, seen);
    return cuda_status(e);
}

}  // namespace ofe
