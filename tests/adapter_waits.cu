// The tile kernels of the adapters with waits that run out: a wait ends as it should, and is then told to the threads under test as one that did not, so
// that what it was for is done.  Barriers that hang on such a wait never come: theirs end after 50 ms.  Compiled and driven by test_gpu_adapter_waits.py.
#include "../ai00_server_b200/csrc/common.cuh"

namespace b200 {

// kernel (its threads), block and thread (-1: all) whose waits run out; 0 threads: none
__device__ int g_kernel, g_block, g_thread;

__device__ __forceinline__ bool lost_try(uint32_t bar, uint32_t parity) {
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try(bar, parity))
        if (globaltimer_ns() - t0 > 50000000ull) return false;          // (a barrier that hangs on a lost wait)
    return !(g_kernel == (int)blockDim.x && g_block == (int)blockIdx.x && (g_thread < 0 || g_thread == (int)threadIdx.x));
}
// a tick is longer than any wait
__device__ __forceinline__ unsigned long long lost_timer() { return globaltimer_ns() << 32; }

}  // namespace b200

#define mbar_try lost_try
#define globaltimer_ns lost_timer
#include "../ai00_server_b200/csrc/adapter_tiles.cuh"

using namespace b200;

static int tiles_of(int tokens, int adapters) { return adapters + 1 + tokens / ADP_TILE; }

extern "C" long long waits_workspace(int tokens, int adapters, int rank) {
    return (long long)AdapterPlan::ints(tokens, adapter_groups(tokens, adapters), tiles_of(tokens, adapters)) * 4 + 16 + (long long)adt_low_bytes(tokens, rank, 2);
}

// every adapter in tiles, f16 to f32; 0, or a CUDA error
extern "C" int waits_run(int kernel, int block, int thread, int tokens, int adapters, int K, int N, int R, const void* x, const void* a, const void* b, const int* index,
                         const float* scale, const float* base, float* out, void* workspace, int out_ctas) {
    AdapterParams p;
    memset(&p, 0, sizeof(p));
    p.tokens = tokens; p.adapters = adapters; p.index = index; p.scale = scale;
    p.nparts = 1; p.rank = R; p.tile_least = 1; p.copy = 1;
    p.out_tokens = adt_out_tokens(R, 2);
    p.plan.base = (int*)workspace;
    p.plan.groups = adapter_groups(tokens, adapters);
    p.plan.tiles = tiles_of(tokens, adapters);
    p.low = (uint8_t*)workspace + ((AdapterPlan::ints(tokens, p.plan.groups, p.plan.tiles) * 4 + 15) & ~(size_t)15);
    AdapterPart& d = p.part[0];
    d.x = x; d.x_stride = K; d.a = a; d.b = b; d.base = base; d.base_stride = N; d.out = out; d.out_stride = N;
    d.K = K; d.N = N; d.R = R; d.vec = N % 4 == 0;
    cudaMemcpyToSymbol(g_kernel, &kernel, sizeof(int));
    cudaMemcpyToSymbol(g_block, &block, sizeof(int));
    cudaMemcpyToSymbol(g_thread, &thread, sizeof(int));
    cudaFuncSetAttribute(adapter_low_kernel<__half, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, adt_low_smem(R));
    cudaFuncSetAttribute(adapter_out_kernel<__half, float>, cudaFuncAttributeMaxDynamicSharedMemorySize, adt_out_smem(R, 2));
    adapter_plan_kernel<<<1, ADP_PLAN_THREADS>>>(p);
    adapter_low_kernel<__half, 2><<<dim3(ADP_CTAS * p.plan.tiles, 1), ADT_LOW_THREADS, adt_low_smem(R)>>>(p);
    adapter_out_kernel<__half, float><<<out_ctas, ADT_THREADS, adt_out_smem(R, 2)>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? (int)e : (int)cudaDeviceSynchronize();
}
