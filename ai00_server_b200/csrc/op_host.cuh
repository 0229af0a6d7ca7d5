// Host side of the operators on device memory, shared by their translation units: launches, the device of a call, buffers that overlap.
#pragma once
#include <atomic>
#include <cstring>

#include "common.cuh"
#include "host.cuh"

namespace b200 {

// a kernel's dynamic shared memory, once for every device that launches it
template <auto KERN>
static void prepare(size_t bytes, bool wide_clusters = false) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    CK(cudaGetDevice(&dev));
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return;
    allow_smem(KERN, bytes);
    if (wide_clusters) CK(cudaFuncSetAttribute(KERN, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    done.fetch_or(bit, std::memory_order_release);
}

static int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0;
    CK(cudaGetDevice(&dev));
    int n = known[dev & 63].load(std::memory_order_relaxed);
    if (n == 0) {
        CK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        known[dev & 63].store(n, std::memory_order_relaxed);
    }
    return n;
}

// cluster: CTAs of a cluster where the kernel does not say
template <typename P>
static void launch(void (*kern)(P), dim3 grid, int threads, size_t smem, cudaStream_t s, const P& p, int cluster = 0) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    // starts while the kernel in front drains; every kernel here waits for that one's end before it reads anything
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    CK(cudaLaunchKernelEx(&cfg, kern, p));
}

// the calling thread's device for the length of a call
struct OnDevice {
    int before = 0;
    explicit OnDevice(int device) {
        CK(cudaGetDevice(&before));
        if (before != device) CK(cudaSetDevice(device));
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// rows of a buffer: bytes between them and of each (a row is no longer than their distance)
struct RowSpan {
    uintptr_t at, step, width, end;
    RowSpan(const void* p, long long rows, long long stride, long long cols, int size)
        : at((uintptr_t)p), step((uintptr_t)(stride * size)), width((uintptr_t)(cols * size)), end(at + (uintptr_t)(rows - 1) * step + width) {}
    bool dense() const { return step == width || end - at == width; }
};
// some byte is in both, as far as can be told: rows at one distance are compared modulo it (columns of a wider buffer may lie side by side), rows without gaps
// as a whole, with each other and with rows that have some; of two at different distances nothing is said
static bool overlap(const RowSpan& a, const RowSpan& b) {
    if (a.at >= b.end || b.at >= a.end) return false;
    if (a.at == b.at || (a.dense() && b.dense())) return true;
    if (b.dense()) return overlap(b, a);
    if (a.dense()) {                                 // (one that starts in front reaches the first row; one in a gap has a row behind it)
        const uintptr_t d = a.at < b.at ? 0 : (a.at - b.at) % b.step;
        return d < b.width || b.step - d < a.end - a.at;
    }
    if (a.step != b.step) return false;
    const uintptr_t d = a.at <= b.at ? (b.at - a.at) % a.step : (a.step - (a.at - b.at) % a.step) % a.step;
    return d < a.width || a.step - d < b.width;
}

// waits of adapters that ran out on the current device (operators.cu)
B200_HIDDEN unsigned adapters_lost_waits();

}  // namespace b200
