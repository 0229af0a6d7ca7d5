// Launches of the operators on device memory (operators.cu), as the C entries and the engine make them.
#pragma once
#include "adapters.cuh"
#include "host.cuh"
#include "logits.cuh"

namespace b200 {

// bytes of the plan that a call of this many tokens needs (0: none)
B200_HIDDEN size_t adapters_workspace(int tokens, int adapters);
// orders the tokens of a longer call by adapter; its groups serve any number of adapters_apply calls with the same tokens
B200_HIDDEN void adapters_plan(cudaStream_t s, const AdapterParams& p);
// parts [0, nparts) of p; type: B200RWKV_TYPE_F16 / _BF16, out_type: that or _F32
B200_HIDDEN void adapters_apply(cudaStream_t s, const AdapterParams& p, int nparts, int type, int out_type);
// slice, sub, buffered and vec of p are filled in here
B200_HIDDEN void logits_rows(cudaStream_t s, LogitsParams p, int rows, int type);

}  // namespace b200
