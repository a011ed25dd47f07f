/*
 * row_device.h - what the kernels of the row operators share.
 */
#ifndef CUTT_ROW_DEVICE_H
#define CUTT_ROW_DEVICE_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <tuple>
#include <type_traits>

#include "hip_layer.h"

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

// n / d for a divisor made by cuttHipMakeDivisor(d), n below 2^31.
__device__ __forceinline__ uint32_t divide(uint32_t n, const cuttHipDivisor& d) { return (__umulhi(n, d.mul) + n * d.add) >> d.shift; }

// N elements that lie anywhere: a vector whose accesses assume no more alignment than its element's.  16 bytes per lane are one
// load or store instruction at any address.
template <typename T, int N>
struct VecOf {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
using Vec = typename VecOf<T, N>::type;

// N elements in a lane's registers, taken from and put to memory in one access.
template <typename T, int N>
struct Pack {
  Vec<T, N> v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const Vec<T, N>*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Vec<T, N>*>(p) = v; }
  __device__ __forceinline__ T get(int i) const { return v[i]; }
  __device__ __forceinline__ void set(int i, T x) { v[i] = x; }
  // zeros unless `keep`
  __device__ __forceinline__ void zeroUnless(bool keep) {
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T) * N / 4)));
    v = __builtin_bit_cast(Vec<T, N>, keep ? __builtin_bit_cast(Words, v) : Words(0));
  }
};
template <typename T>
struct Pack<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ T get(int) const { return v; }
  __device__ __forceinline__ void set(int, T x) { v = x; }
  __device__ __forceinline__ void zeroUnless(bool keep) { v = keep ? v : T(0); }
};

}  // namespace cutt

#endif  // CUTT_ROW_DEVICE_H
