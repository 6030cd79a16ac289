// errwords.cuh — host side of bounded waits: where kernels tell a wait that ran
// out, so that the calls after it refuse without a synchronisation to look.
#pragma once

#include <cuda_runtime.h>
#include <string.h>

#include <atomic>
#include <mutex>
#include <string>

#include "common.cuh"

namespace concord {

// The error words of one family of kernels (a static object; constants until it is used): a device's own, `symbol`, and its
// copy in host memory, which the kernels write to and the host reads.
class ErrorWords {
    static constexpr int DEVICES = 64;
    const void* symbol_;
    const char *kernels_, *clear_;          // "attention kernel", and the function that clears
    std::atomic<int*> words_{nullptr};
    std::mutex mu_;

public:
    ErrorWords(const void* symbol, const char* kernels, const char* clear) : symbol_(symbol), kernels_(kernels), clear_(clear) {}

    // the current device's word in host memory; nullptr: none to be had
    volatile int* host() {
        int d = 0;
        if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= DEVICES) return nullptr;
        int* w = words_.load();
        if (!w) {
            std::lock_guard<std::mutex> g(mu_);
            w = words_.load();
            if (!w) {
                // (an allocation is no work on a stream: it may come first in a capture)
                cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
                cudaThreadExchangeStreamCaptureMode(&mode);
                void* p = nullptr;
                const cudaError_t e = cudaHostAlloc(&p, DEVICES * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
                cudaThreadExchangeStreamCaptureMode(&mode);
                if (e != cudaSuccess) {
                    cudaGetLastError();
                    return nullptr;
                }
                memset(p, 0, DEVICES * sizeof(int));
                words_.store(w = static_cast<int*>(p));
            }
        }
        return w + d;
    }

    // both words as a kernel takes them; refuses while a wait that ran out is told
    int take(int** err, int** err_host, const char* name) {
        volatile int* h = host();
        void* p = nullptr;
        if (!h || cudaGetSymbolAddress(&p, symbol_) != cudaSuccess)
            return fail(CONCORD_ELAUNCH, std::string(name) + ": device set-up failed");
        if (*h)
            return fail(CONCORD_ETIMEOUT, std::string(name) + ": a wait inside an earlier " + kernels_ + " ran out (code " +
                                              std::to_string(*h) + "), its results hold NaN; " + clear_ + "(1) clears this");
        *err = static_cast<int*>(p);
        if (cudaHostGetDevicePointer(&p, const_cast<int*>(h), 0) != cudaSuccess)
            return fail(CONCORD_ELAUNCH, std::string(name) + ": device set-up failed");
        *err_host = static_cast<int*>(p);
        return CONCORD_OK;
    }

    // the code that is told (0: none; -1: no device), cleared with `reset`; synchronises
    int read(int reset) {
        volatile int* h = host();
        void* p = nullptr;
        int v = 0;
        if (!h || cudaGetSymbolAddress(&p, symbol_) != cudaSuccess ||
            cudaMemcpy(&v, p, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess)
            return -1;
        if (!v) v = *h;
        if (reset) {
            if (cudaMemset(p, 0, sizeof(int)) != cudaSuccess) return -1;
            *h = 0;
        }
        return v;
    }
};

}  // namespace concord
