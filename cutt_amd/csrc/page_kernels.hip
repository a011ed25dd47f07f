/*
 * page_kernels.hip - rows in pages (cutt_rows.h): the tables of pages and the slots of new tokens from the requests'
 * lengths, and the move of keys and values to their slots and back.
 */
#include "row_device.h"
#include "row_layer.h"

using namespace cutt;

namespace {

constexpr uint32_t kThreads = 256, kMaxBlocks = 1u << 22;

// Sums of lengths stop at 2^31 - 1.  (Capping a sum of such numbers is associative, so the order of a scan does not matter.)
__device__ __forceinline__ uint32_t capped(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }

__device__ __forceinline__ uint32_t pagesFor(uint32_t tokens, uint32_t pageSize) { return (tokens + pageSize - 1) / pageSize; }

// One thread goes through the requests.
__global__ void pageTablesKernel(cuttHipTablesArgs a) {
  uint32_t start = 0, taken = 0;
  for (uint32_t b = 0; b < a.requests; b++) {
    const uint32_t cached = max(a.cached[b], 0), added = max(a.added[b], 0);
    const uint32_t owned = pagesFor(cached, a.pageSize), want = pagesFor(capped(cached, added), a.pageSize);
    a.starts[b] = (int32_t)start;
    for (uint32_t j = owned; j < want && j < a.tableWidth; j++) {
      const uint64_t at = (uint64_t)taken + (j - owned);
      a.tables[(uint64_t)b * a.tableWidth + j] = at < a.freeCount ? a.freePages[at] : -1;
    }
    start = capped(start, added);
    taken = capped(taken, want - owned);
  }
  a.starts[a.requests] = (int32_t)start;
  a.used[0] = (int32_t)taken;
}

__global__ __launch_bounds__(kThreads) void pageSlotsKernel(cuttHipTablesArgs a) {
  for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < a.tokens; i += (uint64_t)gridDim.x * kThreads) {
    int64_t slot = -1;
    int32_t position = -1;
    if (i < (uint32_t)a.starts[a.requests]) {
      uint32_t lo = 0, hi = a.requests;  // starts[lo] <= i < starts[hi]
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if ((uint32_t)a.starts[mid] <= i) lo = mid;
        else hi = mid;
      }
      const uint32_t p = capped(max(a.cached[lo], 0), (uint32_t)i - (uint32_t)a.starts[lo]), j = p / a.pageSize;
      position = (int32_t)p;
      const int32_t page = j < a.tableWidth ? a.tables[(uint64_t)lo * a.tableWidth + j] : -1;
      if (page >= 0) slot = (int64_t)page * a.pageSize + (p - j * a.pageSize);
    }
    a.slots[i] = slot;
    if (a.positions) a.positions[i] = position;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pageMoveKernel(cuttHipPageArgs a) {
  const uint64_t perToken = (uint64_t)a.heads * a.width;
  T* const rows = (T*)a.rows[blockIdx.y];
  T* const cache = (T*)a.cache[blockIdx.y];
  for (uint64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int64_t slot = a.slots[t];
    const bool there = slot >= 0 && slot < (int64_t)a.pages * a.pageSize;
    if (!there && !a.load) continue;
    const uint64_t at = there ? slot / a.pageSize * a.pageStride + slot % a.pageSize * a.slotStride : 0;
    for (uint64_t i = threadIdx.x; i < perToken; i += kThreads) {
      const uint64_t h = i / a.width, c = i % a.width;
      T& row = rows[t * a.tokenStride + h * a.headStride + c];
      T* const cell = cache + (at + h * a.cacheHeadStride + c);
      if (!a.load) *cell = row;
      else row = there ? *cell : T(0);
    }
  }
}

}  // namespace

extern "C" int cuttHipPageTables(const cuttHipTablesArgs* a, void* stream) {
  if (int e = launchRows(pageTablesKernel, 1, 1, 0, stream, *a)) return e;
  if (!a->tokens) return 0;
  const uint32_t blocks = (a->tokens + kThreads - 1) / kThreads;
  return launchRows(pageSlotsKernel, blocks < kMaxBlocks ? blocks : kMaxBlocks, kThreads, 0, stream, *a);
}

extern "C" int cuttHipPageMove(const cuttHipPageArgs* a, void* stream) {
  const dim3 grid(a->tokens < kMaxBlocks ? a->tokens : kMaxBlocks, a->rows[1] ? 2 : 1);
  switch (a->elemSize) {
    case 1: return launchRows(pageMoveKernel<uint8_t>, grid, kThreads, 0, stream, *a);
    case 2: return launchRows(pageMoveKernel<uint16_t>, grid, kThreads, 0, stream, *a);
    case 4: return launchRows(pageMoveKernel<uint32_t>, grid, kThreads, 0, stream, *a);
    default: return launchRows(pageMoveKernel<uint64_t>, grid, kThreads, 0, stream, *a);
  }
}
