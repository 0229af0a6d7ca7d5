// Waits of operators' kernels that ran out, counted on their device: a number for each translation unit, which b200rwkv_op_lost_waits adds up.
#pragma once

namespace b200 {

static __device__ unsigned lost_waits;
__device__ __forceinline__ void lost_wait() { atomicAdd(&lost_waits, 1u); }

}  // namespace b200
