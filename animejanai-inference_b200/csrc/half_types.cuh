/* half_types.cuh — fp16 and bf16 to fp32 and back, by type. */
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ajib {
namespace dev {

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace dev
}  // namespace ajib
