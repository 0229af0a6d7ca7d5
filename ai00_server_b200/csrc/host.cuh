// Errors of the host side, shared by the translation units of the library: a failing call throws Error, the C entries turn it into a status
// and keep its text for the calling thread (b200rwkv_last_error).
#pragma once
#include <cuda_runtime.h>

#include <mutex>
#include <stdexcept>
#include <string>

#include "../../include/b200rwkv.h"

#define B200_HIDDEN __attribute__((visibility("hidden")))

namespace b200 {

struct Error : std::runtime_error {
    int code;
    Error(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

// the calling thread's last error text (engine.cu)
B200_HIDDEN std::string& last_error_text();
// the device watchdog's record, empty without one (engine.cu)
B200_HIDDEN std::string watchdog_report();

}  // namespace b200

#define CK(call)                                                                                         \
    do {                                                                                                 \
        cudaError_t e_ = (call);                                                                         \
        if (e_ != cudaSuccess)                                                                           \
            throw b200::Error(B200RWKV_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_) + " @" +   \
                                               __FILE__ + ":" + std::to_string(__LINE__) + watchdog_report()); \
    } while (0)
#define REQUIRE(cond, code, msg)                 \
    do {                                         \
        if (!(cond)) throw b200::Error((code), (msg)); \
    } while (0)

// Error text is thread-local: the reference makes engine calls from two tasks (infer / softmax, run.rs:1232-1237) and a
// per-engine string would race between them.  b200rwkv_last_error() returns the message of the calling thread's last failure.
#define API_BEGIN(e)                            \
    std::string* errp_ = &b200::last_error_text();    \
    (void)(e);                                  \
    try {
#define API_END                                  \
    }                                            \
    catch (const b200::Error& ex) {                    \
        *errp_ = ex.what();                      \
        return ex.code;                          \
    }                                            \
    catch (const std::exception& ex) {           \
        *errp_ = ex.what();                      \
        return B200RWKV_ERR_INVALID;             \
    }                                            \
    catch (...) {                                \
        *errp_ = "unknown exception";            \
        return B200RWKV_ERR_INVALID;             \
    }                                            \
    return B200RWKV_OK;

namespace b200 {

// dynamic shared memory a kernel may be launched with.  The limit belongs to the process, not to an engine: it is only ever raised, so that a
// narrower model loaded later leaves the launches of a wider one valid
template <typename K>
static void allow_smem(K* kern, size_t bytes) {
    static std::mutex mu;
    std::lock_guard<std::mutex> lk(mu);
    cudaFuncAttributes a;
    CK(cudaFuncGetAttributes(&a, kern));
    if ((size_t)a.maxDynamicSharedSizeBytes < bytes) CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
}

}  // namespace b200
