/*
 * row_device.h - what the kernels of the row operators share.
 */
#ifndef CUTT_ROW_DEVICE_H
#define CUTT_ROW_DEVICE_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <tuple>
#include <type_traits>

namespace cutt {

// Reports the launch call's own result (hipGetLastError would also report, and clear, what an earlier call of the
// application left behind).
template <typename... KArgs, typename... Args>
int launchRows(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t lds, void* stream, Args... args) {
  static_assert(sizeof...(KArgs) == sizeof...(Args), "one argument per kernel parameter");
  std::tuple<std::remove_const_t<KArgs>...> held{args...};
  void* ptrs[sizeof...(KArgs)];
  int i = 0;
  std::apply([&](auto&... v) { ((ptrs[i++] = (void*)&v), ...); }, held);
  return (int)hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, ptrs, lds, (hipStream_t)stream);
}

}  // namespace cutt

#endif  // CUTT_ROW_DEVICE_H
