// Eight consecutive values of a 128-value head row, as the RoPE + append kernels move them: 16 threads hold a row, and
// every load and store is 16 bytes per thread.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

// as they lie in memory: one 16-byte piece for fp16, two for f32
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ void to_f32(float (&x)[8]) const {
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
};
template <>
struct Raw8<__half> {
    uint4 raw;
    __device__ __forceinline__ void load(const __half* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void to_f32(float (&x)[8]) const {
        const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(h[j]);
            x[2 * j] = f.x, x[2 * j + 1] = f.y;
        }
    }
};
__device__ __forceinline__ void st8_as_f16(__half* p, const float (&x)[8]) {
    uint4 raw;
    __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = raw;
}
