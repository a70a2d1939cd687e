// A kernel launch whose own error is reported (not one that an earlier call left).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>

namespace sca::kern {

// What a kernel reads or writes has an address: a tensor without memory (a fake one, as tracers use) has none.
inline void need_memory(const void* p, const char* what) {
  if (!p) throw std::invalid_argument(std::string(what) + " has no memory");
}

// A launch holds fewer than 2^32 threads along x.  Asked before the first launch of a call, so that a call is refused whole.
inline void need_blocks(int64_t blocks, int threads, const char* what) {
  if (blocks > int64_t(0xffffffff) / threads) throw std::invalid_argument(std::string(what) + ": too large for one call");
}

template <class... P, class... A>
void launch_kernel(void (*fn)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t s, A&&... args) {
  static_assert(sizeof...(P) == sizeof...(A), "one argument for each parameter");
  std::tuple<std::decay_t<P>...> held(std::forward<A>(args)...);
  std::apply(
      [&](auto&... x) {
        void* ptrs[] = {const_cast<void*>(static_cast<const void*>(&x))...};
        hipError_t e = hipSuccess;
        if (lds > 64 * 1024)  // beyond the default limit of a launch
          e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
        if (e == hipSuccess) e = hipLaunchKernel(reinterpret_cast<const void*>(fn), grid, block, ptrs, lds, s);
        if (e != hipSuccess) throw std::runtime_error(std::string("kernel launch failed: ") + hipGetErrorString(e));
      },
      held);
}

}  // namespace sca::kern
