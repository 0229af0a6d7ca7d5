// Numbers of the operators' types as f32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b200 {

template <typename E> __device__ __forceinline__ float widened(E v);
template <> __device__ __forceinline__ float widened<float>(float v) { return v; }
template <> __device__ __forceinline__ float widened<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widened<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

}  // namespace b200
