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

// Whether rows are more than the memory-side cache (256 MB) holds.  Then what is read cannot have been left there by whoever wrote it, nor what is
// written be found there, and accesses past the caches are faster; below it they cost the next kernel more than they give.  MI355X, 8 choices, 4096
// bfloat16: dispatch of 8192 tokens (537 MB of rows) 105 us past the caches, 118 through them, combine 104 and 119; dispatch and a combine that reads its
// rows right after it, 134 MB: 58 us past, 52 through, 537 MB: 211 and 253.
inline bool pastCaches(uint64_t rows, uint64_t rowBytes) { return rows * rowBytes > ((uint64_t)256 << 20); }

// n / d for a divisor made by cuttHipMakeDivisor(d), n below 2^31.
__device__ __forceinline__ uint32_t divide(uint32_t n, const cuttHipDivisor& d) { return (__umulhi(n, d.mul) + n * d.add) >> d.shift; }

// x of the lanes up to this one combined by an associative f whose neutral element is 0, for the lanes of a wavefront (all of them
// take part).  Data move between lanes in the vector unit: four steps inside rows of 16 lanes, then the last lane of a row to the
// next row and the last lane of the lower half to the upper half.
template <typename F>
__device__ __forceinline__ uint32_t scanOverWave(uint32_t x, F f) {
#define CUTT_STEP(ctrl, rows) x = f(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false))
  CUTT_STEP(0x111, 0xf);  // row_shr:1
  CUTT_STEP(0x112, 0xf);
  CUTT_STEP(0x114, 0xf);
  CUTT_STEP(0x118, 0xf);
  CUTT_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
  CUTT_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef CUTT_STEP
  return x;
}

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
  // NT: past the caches (non-temporal), for what is used once
  template <bool NT = false>
  __device__ __forceinline__ void load(const T* p) {
    const Vec<T, N>* const q = reinterpret_cast<const Vec<T, N>*>(p);
    if constexpr (NT) v = __builtin_nontemporal_load(q);
    else v = *q;
  }
  template <bool NT = false>
  __device__ __forceinline__ void store(T* p) const {
    Vec<T, N>* const q = reinterpret_cast<Vec<T, N>*>(p);
    if constexpr (NT) __builtin_nontemporal_store(v, q);
    else *q = v;
  }
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
  template <bool NT = false>
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  template <bool NT = false>
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ T get(int) const { return v; }
  __device__ __forceinline__ void set(int, T x) { v = x; }
  __device__ __forceinline__ void zeroUnless(bool keep) { v = keep ? v : T(0); }
};

}  // namespace cutt

#endif  // CUTT_ROW_DEVICE_H
