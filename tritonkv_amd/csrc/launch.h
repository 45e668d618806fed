// Kernel launches of the page-pool entry points.
#pragma once

#include <hip/hip_runtime.h>

namespace tkv {

// Launches kernel on st; a TKV status (0, or the hipError_t).  The runtime's call
// itself, not the <<<>>> form, which keeps the configuration in a stack of its own
// first: 2.2 against 2.5 us of host time a launch.
template <class... P>
inline int launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t st, P... args) {
  void* list[] = {const_cast<void*>(static_cast<const void*>(&args))...};
  return (int)hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, list, lds, st);
}

}  // namespace tkv
