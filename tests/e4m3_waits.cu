// The kernels of 8-bit products with waits that run out: a wait ends as it should, and is then told to the threads under test as one that did not, so that what it was for is done.
// Barriers that hang on such a wait never come: theirs end after 10 ms.  Compiled and driven by test_gpu_e4m3_waits.py.
#include "../ai00_server_b200/csrc/common.cuh"

namespace b200 {

// kernel (its threads), block and thread (-1: all) whose waits run out; 0 threads: none
__device__ int g_kernel, g_block, g_thread;

__device__ __forceinline__ bool lost_try(uint32_t bar, uint32_t parity) {
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try(bar, parity))
        if (globaltimer_ns() - t0 > 20000ull) return false;             // (of the 512 tries that a wait has)
    return !(g_kernel == (int)blockDim.x && g_block == (int)blockIdx.x && (g_thread < 0 || g_thread == (int)threadIdx.x));
}
// a tick is longer than any wait
__device__ __forceinline__ unsigned long long lost_timer() { return globaltimer_ns() << 32; }

}  // namespace b200

#define mbar_try lost_try
#define globaltimer_ns lost_timer
#include "../ai00_server_b200/csrc/e4m3_linear.cuh"

#include <cstring>

using namespace b200;

static bool rows_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t width, uint32_t box_rows) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess || !f) return false;
    const cuuint64_t dim[2] = {width, rows}, step[1] = {width};
    const cuuint32_t box[2] = {E4L_KB, box_rows}, es[2] = {1, 1};
    return ((PFN_cuTensorMapEncodeTiled_v12000)f)(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dim, step, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TT>
static cudaError_t few(E4LinearParams p, const void* x, const void* w, int K, int split) {
    using C = E4Few<TT>;
    if (!rows_map(&p.tx, x, p.tokens, K, TT) || !rows_map(&p.tw, w, p.N, K, 128)) return cudaErrorUnknown;
    p.split = split;
    const cudaError_t e = cudaFuncSetAttribute(e4_few_kernel<TT, float>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((p.N + 127) / 128 * split, (p.tokens + TT - 1) / TT);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = split;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, e4_few_kernel<TT, float>, p);
}

// f32 out; form: tokens of the few-token kernel (16, 128), or 256 for the pairs (`split`: clusters); 0, or a CUDA error
extern "C" int waits_run(int kernel, int block, int thread, int form, int split, int tokens, int K, int N, const void* x, const float* xs, const void* w, const float* ws, float* out) {
    E4LinearParams p;
    memset(&p, 0, sizeof(p));
    p.xs = xs; p.ws = ws; p.out = out; p.out_stride = N; p.tokens = tokens; p.N = N; p.kblocks = (K + E4L_KB - 1) / E4L_KB; p.vec = N % 4 == 0;
    cudaMemcpyToSymbol(g_kernel, &kernel, sizeof(int));
    cudaMemcpyToSymbol(g_block, &block, sizeof(int));
    cudaMemcpyToSymbol(g_thread, &thread, sizeof(int));
    cudaError_t e;
    if (form == 16) {
        e = few<16>(p, x, w, K, split);
    } else if (form == 128) {
        e = few<128>(p, x, w, K, split);
    } else {
        using C = E4Pair;
        if (!rows_map(&p.tx, x, tokens, K, 128) || !rows_map(&p.tw, w, N, K, C::BN / 2)) return (int)cudaErrorUnknown;
        e = cudaFuncSetAttribute(e4_pair_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e == cudaSuccess) {
            e4_pair_kernel<float><<<2 * split, C::THREADS, C::SMEM>>>(p);
            e = cudaGetLastError();
        }
    }
    return e != cudaSuccess ? (int)e : (int)cudaDeviceSynchronize();
}

// waits that ran out so far
extern "C" unsigned waits_lost() {
    unsigned n = ~0u;
    cudaMemcpyFromSymbol(&n, lost_waits, sizeof(n));
    return n;
}
