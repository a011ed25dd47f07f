/*
 * product_device.h - what the kernels of the products share: matrix instructions, tiles of operands in LDS and the fragments that the
 * instructions take from them.
 *
 * All products use D = A * B + C of 16 x 16 results: lane l holds of A row l & 15, of B column l & 15, and of both the same k's: those of the
 * lane's quarter l / 16.  Which k's these are is free as long as A and B agree.  D: column l & 15, rows 4 * (l / 16) + 0..3.
 */
#ifndef CUTT_PRODUCT_DEVICE_H
#define CUTT_PRODUCT_DEVICE_H

#include "row_device.h"

namespace cutt {

typedef float Acc __attribute__((ext_vector_type(4)));

template <typename T, int N>
struct AlignedVecOf {
  typedef T type __attribute__((ext_vector_type(N)));
};
// N elements at an address that is a multiple of their size.
template <typename T, int N>
using AlignedVec = typename AlignedVecOf<T, N>::type;

// Elements of 16 bytes.
template <typename T>
constexpr int kPer16 = 16 / sizeof(T);
template <typename T>
using Chunk = AlignedVec<T, kPer16<T>>;

// Products of 16 bytes of k's per lane: 32 k's in one instruction of the 16-bit types, 16 in four of the 32-bit type.
__device__ __forceinline__ Acc multiply(Chunk<__bf16> a, Chunk<__bf16> b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ Acc multiply(Chunk<_Float16> a, Chunk<_Float16> b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ Acc multiply(float a, float b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ Acc multiply(Chunk<float> a, Chunk<float> b, Acc c) {
#pragma unroll
  for (int j = 0; j < 4; j++) c = multiply(a[j], b[j], c);
  return c;
}

// The first `valid` of 16 bytes of elements at p, zeros behind them; nothing else is read.
template <typename T>
__device__ __forceinline__ Chunk<T> loadChunk(const T* p, int valid) {
  constexpr int E = kPer16<T>;
  Chunk<T> v = {};
  if (valid >= E) {
    v = __builtin_bit_cast(Chunk<T>, *reinterpret_cast<const Vec<T, E>*>(p));
  } else if (valid > 0) {
#pragma unroll
    for (int i = 0; i < E; i++)
      if (i < valid) v[i] = p[i];
  }
  return v;
}

// x of lane l combined with those of the lanes that differ from it in bits 4 and 5.
template <typename F>
__device__ __forceinline__ float overQuarters(float x, F f) {
  x = f(x, __shfl_xor(x, 16));
  return f(x, __shfl_xor(x, 32));
}

}  // namespace cutt

#endif  // CUTT_PRODUCT_DEVICE_H
