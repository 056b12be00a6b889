#include "kernels/sm100/wait_status.h"

#include "core/check.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

namespace b200ccl::kernels {

namespace {

constexpr int kDevices = 64;
std::atomic<unsigned*> all_words{nullptr};

}  // namespace

unsigned* wait_status_word(WaitsOf what, int device) {
    static unsigned* words = [] {
        // (Allocating is allowed beside a capture: nothing of it belongs to the graph.)
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        B2_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
        void* p = nullptr;
        const cudaError_t st = cudaHostAlloc(&p, kWaitsOf * kDevices * sizeof(unsigned), cudaHostAllocMapped | cudaHostAllocPortable);
        cudaThreadExchangeStreamCaptureMode(&mode);
        B2_CUDA(st);
        std::fill_n(static_cast<unsigned*>(p), kWaitsOf * kDevices, 0u);
        all_words.store(static_cast<unsigned*>(p));
        return static_cast<unsigned*>(p);
    }();
    return words + static_cast<int>(what) * kDevices + device % kDevices;
}

bool waits_failed(WaitsOf what, int device) {
    B2_REQUIRE(device >= 0, "no such device");
    unsigned* words = all_words.load();  // (null before the first call of all)
    return words != nullptr && __atomic_exchange_n(words + static_cast<int>(what) * kDevices + device % kDevices, 0u, __ATOMIC_RELAXED) != 0u;
}

}  // namespace b200ccl::kernels
