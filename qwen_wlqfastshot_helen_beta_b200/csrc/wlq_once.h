// A setting that belongs to a device, such as a kernel's dynamic shared memory
// limit: made at the first launch on each device and remembered, so that a
// decoding step's launches do not pay for it on the host again.
#pragma once

#include <cuda_runtime_api.h>

#include <atomic>
#include <cstdint>

namespace wlq {

class OncePerDevice {
  public:
    // Calls set() unless it has succeeded for this device before.  A failure
    // is returned and not remembered; two threads may both call it.
    template <typename Set>
    cudaError_t run(int device, Set set) {
        const bool known = device >= 0 && device < 64;
        const uint64_t bit = known ? uint64_t{1} << device : 0;
        if (done_.load(std::memory_order_acquire) & bit) return cudaSuccess;
        const cudaError_t e = set();
        if (e == cudaSuccess) done_.fetch_or(bit, std::memory_order_release);
        return e;
    }

  private:
    std::atomic<uint64_t> done_{0};
};

}  // namespace wlq
