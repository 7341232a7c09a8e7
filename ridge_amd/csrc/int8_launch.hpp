// int8_launch.hpp -- launches of the 8-bit operators' kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

namespace ridge {

// Enqueues a kernel; the launch's own status. hipGetLastError behind <<< >>> would give back,
// and clear, what any earlier call of the program has left: a kernel that runs would be
// reported as failed.
template <typename... Args>
hipError_t launchKernel(void (*kernel)(Args...), unsigned blocks, int threads, hipStream_t stream,
                        const std::enable_if_t<true, Args>&... args) {
    void* addresses[] = {const_cast<void*>(static_cast<const void*>(&args))...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(blocks), dim3((unsigned)threads), addresses, 0,
                           stream);
}

}  // namespace ridge
