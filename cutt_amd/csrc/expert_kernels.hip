/*
 * expert_kernels.hip - rows sorted by expert and back (cutt_rows.h): the stable counting sort of a router's
 * choices, the move of the tokens' rows to their experts, the weighted sum back, and the gradients of both.
 */
#include "row_device.h"
#include "row_layer.h"

using namespace cutt;

namespace {

// ---------------------------------------------------------------------------
// Sort: one workgroup counts, adds up and places.
// ---------------------------------------------------------------------------
constexpr uint32_t kSortThreads = 512, kSortWaves = kSortThreads / 64;

// The expert of choice i among the `experts`, or `experts` if it is none of them.
template <typename Id>
__device__ __forceinline__ uint32_t expertOf(const cuttHipSortArgs& a, uint32_t i) {
  const uint64_t e = (uint64_t)(int64_t) static_cast<const Id*>(a.ids)[i] - (uint64_t)(int64_t)a.firstExpert;  // (wraps)
  return e < a.experts ? (uint32_t)e : a.experts;
}

// Lanes of the wavefront whose key is this lane's.
__device__ __forceinline__ uint64_t sameKey(uint32_t key, uint32_t bits) {
  uint64_t same = ~0ull;
  for (uint32_t b = 0; b < bits; b++) {
    const bool one = (key >> b) & 1;
    const uint64_t set = __ballot(one);
    same &= one ? set : ~set;
  }
  return same;
}

template <typename Id>
__global__ __launch_bounds__(kSortThreads) void expertSortKernel(cuttHipSortArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t* const next = lds;                     // [experts + 1] row of an expert's next choice
  uint32_t* const seen = lds + a.experts + 1;     // [waves][experts + 1]
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = a.experts;
  for (uint32_t i = tid; i <= E; i += kSortThreads) next[i] = 0;
  __syncthreads();
  for (uint32_t i = tid; i < a.n; i += kSortThreads) atomicAdd(&next[expertOf<Id>(a, i)], 1u);
  __syncthreads();
  if (tid == 0) {
    uint32_t at = 0;
    for (uint32_t e = 0; e < E; e++) {
      const uint32_t c = next[e];
      a.counts[e] = (int32_t)c;
      a.offsets[e] = (int32_t)at;
      next[e] = at;
      at += (c + a.align - 1) / a.align * a.align;
    }
    a.offsets[E] = (int32_t)at;
  }
  for (uint32_t r = tid; r < a.rows; r += kSortThreads) a.source[r] = -1;
  const uint32_t bits = 32 - __builtin_clz(E);
  for (uint32_t base = 0; base < a.n; base += kSortThreads) {
    __syncthreads();
    for (uint32_t i = tid; i < kSortWaves * (E + 1); i += kSortThreads) seen[i] = 0;
    __syncthreads();
    const uint32_t i = base + tid;
    const uint32_t e = i < a.n ? expertOf<Id>(a, i) : E;
    const uint64_t same = sameKey(e, bits);
    const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
    if (rank == 0) seen[wave * (E + 1) + e] = __popcll(same);
    __syncthreads();
    uint32_t row = next[e] + rank;
    for (uint32_t w = 0; w < wave; w++) row += seen[w * (E + 1) + e];
    if (i < a.n) {
      const bool there = e < E && row < a.rows;
      a.position[i] = there ? (int32_t)row : -1;
      if (there) a.source[row] = (int32_t)i;
    }
    __syncthreads();
    for (uint32_t x = tid; x < E; x += kSortThreads)
      for (uint32_t w = 0; w < kSortWaves; w++) next[x] += seen[w * (E + 1) + x];
  }
}

// ---------------------------------------------------------------------------
// Rows to experts and back, one workgroup per row.
// ---------------------------------------------------------------------------
constexpr uint32_t kRowThreads = 256;
constexpr uint32_t kMaxBlocks = 1u << 22;  // (workgroups x lanes have to fit 32 bits)

__device__ __forceinline__ bool rowAt(const cuttHipExpertArgs& a, uint64_t choice, uint32_t& row) {
  row = (uint32_t)a.position[choice];
  return row < a.rows;
}

template <typename T>
__device__ void clearEmptyRows(const cuttHipExpertArgs& a, T* y, uint64_t stride, uint64_t first, uint64_t step) {
  for (uint64_t r = first; r < a.rows; r += step) {
    if (a.source[r] >= 0) continue;
    for (uint32_t c = threadIdx.x; c < a.width; c += kRowThreads) y[r * stride + c] = T(0);
  }
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void dispatchKernel(cuttHipExpertArgs a, const T* x, uint64_t xStride, T* y, uint64_t yStride) {
  for (uint64_t t = blockIdx.x; t < a.tokens; t += gridDim.x)
    for (uint32_t k = 0; k < a.choices; k++) {
      uint32_t row;
      if (!rowAt(a, t * a.choices + k, row)) continue;
      for (uint32_t c = threadIdx.x; c < a.width; c += kRowThreads) y[row * yStride + c] = x[t * xStride + c];
    }
  clearEmptyRows(a, y, yStride, blockIdx.x, gridDim.x);
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void combineKernel(cuttHipExpertArgs a, const T* y, uint64_t yStride, T* out, uint64_t outStride) {
  for (uint64_t t = blockIdx.x; t < a.tokens; t += gridDim.x)
    for (uint32_t c = threadIdx.x; c < a.width; c += kRowThreads) {
      float sum = 0;
      for (uint32_t k = 0; k < a.choices; k++) {
        uint32_t row;
        if (!rowAt(a, t * a.choices + k, row)) continue;
        const float v = (float)y[row * yStride + c];
        sum += a.weights ? a.weights[t * a.choices + k] * v : v;
      }
      out[t * outStride + c] = (T)sum;
    }
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void combineBackwardKernel(cuttHipExpertArgs a, const T* y, uint64_t yStride, const T* dout, uint64_t doutStride,
                                                                     T* dy, uint64_t dyStride, float* dweights) {
  __shared__ float part[kRowThreads];
  for (uint64_t t = blockIdx.x; t < a.tokens; t += gridDim.x)
    for (uint32_t k = 0; k < a.choices; k++) {
      uint32_t row;
      const bool there = rowAt(a, t * a.choices + k, row);
      float sum = 0;
      if (there)
        for (uint32_t c = threadIdx.x; c < a.width; c += kRowThreads) {
          const float g = (float)dout[t * doutStride + c];
          if (dweights) sum += g * (float)y[row * yStride + c];
          if (dy) dy[row * dyStride + c] = (T)(a.weights[t * a.choices + k] * g);
        }
      if (!dweights) continue;
      part[threadIdx.x] = sum;
      for (uint32_t n = kRowThreads / 2; n; n /= 2) {
        __syncthreads();
        if (threadIdx.x < n) part[threadIdx.x] += part[threadIdx.x + n];
      }
      if (threadIdx.x == 0) dweights[t * a.choices + k] = part[0];
      __syncthreads();
    }
  if (dy) clearEmptyRows(a, dy, dyStride, blockIdx.x, gridDim.x);
}

uint32_t blocksFor(uint64_t n) { return (uint32_t)(n < 1 ? 1 : n < kMaxBlocks ? n : kMaxBlocks); }

}  // namespace

extern "C" size_t cuttHipSortWorkspace(uint32_t, uint32_t) { return 0; }

extern "C" int cuttHipExpertSort(const cuttHipSortArgs* a, void* stream) {
  const size_t lds = (size_t)(kSortWaves + 1) * (a->experts + 1) * 4;
  return a->idBytes == 8 ? launchRows(expertSortKernel<int64_t>, 1, kSortThreads, lds, stream, *a)
                         : launchRows(expertSortKernel<int32_t>, 1, kSortThreads, lds, stream, *a);
}

extern "C" int cuttHipDispatch(const cuttHipExpertArgs* a, uint32_t elemSize, const void* x, uint64_t xStride, void* y, uint64_t yStride, void* stream) {
  const dim3 grid(blocksFor(a->tokens > a->rows ? a->tokens : a->rows));
  switch (elemSize) {
    case 1: return launchRows(dispatchKernel<uint8_t>, grid, kRowThreads, 0, stream, *a, (const uint8_t*)x, xStride, (uint8_t*)y, yStride);
    case 2: return launchRows(dispatchKernel<uint16_t>, grid, kRowThreads, 0, stream, *a, (const uint16_t*)x, xStride, (uint16_t*)y, yStride);
    case 4: return launchRows(dispatchKernel<uint32_t>, grid, kRowThreads, 0, stream, *a, (const uint32_t*)x, xStride, (uint32_t*)y, yStride);
    default: return launchRows(dispatchKernel<uint64_t>, grid, kRowThreads, 0, stream, *a, (const uint64_t*)x, xStride, (uint64_t*)y, yStride);
  }
}

namespace {

template <typename T>
int combine(const cuttHipExpertArgs* a, const void* y, uint64_t yStride, void* out, uint64_t outStride, void* stream) {
  return launchRows(combineKernel<T>, blocksFor(a->tokens), kRowThreads, 0, stream, *a, (const T*)y, yStride, (T*)out, outStride);
}

template <typename T>
int combineBackward(const cuttHipExpertArgs* a, const void* y, uint64_t yStride, const void* dout, uint64_t doutStride, void* dy, uint64_t dyStride,
                    float* dweights, void* stream) {
  return launchRows(combineBackwardKernel<T>, blocksFor(a->tokens > a->rows ? a->tokens : a->rows), kRowThreads, 0, stream, *a, (const T*)y, yStride,
                (const T*)dout, doutStride, (T*)dy, dyStride, dweights);
}

}  // namespace

extern "C" int cuttHipCombine(const cuttHipExpertArgs* a, int type, const void* y, uint64_t yStride, void* out, uint64_t outStride, void* stream) {
  switch (type) {
    case CUTT_ROW_F32: return combine<float>(a, y, yStride, out, outStride, stream);
    case CUTT_ROW_F16: return combine<_Float16>(a, y, yStride, out, outStride, stream);
    default: return combine<__bf16>(a, y, yStride, out, outStride, stream);
  }
}

extern "C" int cuttHipCombineBackward(const cuttHipExpertArgs* a, int type, const void* y, uint64_t yStride, const void* dout, uint64_t doutStride,
                                      void* dy, uint64_t dyStride, float* dweights, void* stream) {
  switch (type) {
    case CUTT_ROW_F32: return combineBackward<float>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
    case CUTT_ROW_F16: return combineBackward<_Float16>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
    default: return combineBackward<__bf16>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
  }
}
