/*
 * page_kernels.hip - rows in pages (cutt_rows.h): the tables of pages and the slots of new tokens from the requests'
 * lengths, and the move of keys and values to their slots and back.  (Times in the comments as in expert_kernels.hip.)
 */
#include "row_device.h"
#include "row_layer.h"

using namespace cutt;

namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;

// Sums of lengths stop at 2^31 - 1.  (Capping a sum of such numbers is associative, so the order of a scan does not matter.)
__device__ __forceinline__ uint32_t capped(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }

__device__ __forceinline__ uint32_t pagesFor(uint32_t tokens, uint32_t pageSize) { return (tokens + pageSize - 1) / pageSize; }

// What the tables need to know of a request.
struct Request {
  uint32_t cached, added, owned, need;
  __device__ __forceinline__ Request(const cuttHipTablesArgs& a, uint32_t b) {
    cached = max(a.cached[b], 0);
    added = max(a.added[b], 0);
    owned = min(pagesFor(cached, a.pageSize), a.tableWidth);
    need = min(pagesFor(capped(cached, added), a.pageSize), a.tableWidth) - owned;
  }
};

// ---------------------------------------------------------------------------
// Page tables.  A workgroup scans the lengths of up to kScan requests: how many new tokens and new pages there are before each.
// Tokens and pages then find their request by a search in LDS.
//
// Bound by the launch and a chain of latencies (lengths, scan, search, table, store): 256 requests of one token 4.4 us, 96 requests with 98352 tokens (1.2
// MB) 4.5, 2048 requests 6.8.  More requests than one scan takes (kScan, 25 KB of LDS): two launches, the first with one workgroup that scans part after part and writes all
// tables: 11 us for 2049, 15 for 4096, 50 for 20000.
// ---------------------------------------------------------------------------
constexpr uint32_t kPerThread = 8, kScan = kThreads * kPerThread;

struct Scan {
  uint32_t tokens[kScan + 1];  // before request i of the scan; behind the last one, all
  uint32_t pages[kScan + 1];
  uint32_t cached[kScan];
  uint32_t waveTokens[kWaves], wavePages[kWaves];
};

// Fills s for the requests first .. first + n - 1, whose predecessors have the given numbers of tokens and pages.  All threads of the workgroup.
__device__ __forceinline__ void scanRequests(const cuttHipTablesArgs& a, uint32_t first, uint32_t n, uint32_t tokensBefore, uint32_t pagesBefore, Scan& s) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t each = (n + kThreads - 1) / kThreads, from = threadIdx.x * each;  // consecutive requests of this thread
  uint32_t tokens[kPerThread], pages[kPerThread], allTokens = 0, allPages = 0;
#pragma unroll
  for (uint32_t i = 0; i < kPerThread; i++) {
    tokens[i] = pages[i] = 0;
    if (i < each && from + i < n) {
      const Request r(a, first + from + i);
      tokens[i] = r.added;
      pages[i] = r.need;
      s.cached[from + i] = r.cached;
    }
    allTokens = capped(allTokens, tokens[i]);
    allPages = capped(allPages, pages[i]);
  }
  const uint32_t upToTokens = scanOverWave(allTokens, capped), upToPages = scanOverWave(allPages, capped);
  if (lane == 63) {
    s.waveTokens[wave] = upToTokens;
    s.wavePages[wave] = upToPages;
  }
  uint32_t t = __shfl_up(upToTokens, 1), p = __shfl_up(upToPages, 1);
  if (lane == 0) t = p = 0;
  __syncthreads();
  for (uint32_t w = 0; w < wave; w++) {
    t = capped(t, s.waveTokens[w]);
    p = capped(p, s.wavePages[w]);
  }
  t = capped(t, tokensBefore);
  p = capped(p, pagesBefore);
#pragma unroll
  for (uint32_t i = 0; i < kPerThread; i++) {
    if (i < each && from + i < n) {
      s.tokens[from + i] = t;
      s.pages[from + i] = p;
    }
    t = capped(t, tokens[i]);
    p = capped(p, pages[i]);
  }
  if (threadIdx.x == kThreads - 1) {  // (its requests are the last ones, or there are none behind the last)
    s.tokens[n] = t;
    s.pages[n] = p;
  }
  __syncthreads();
}

// The last request whose number is not above x; sums[0] <= x < sums[n].
__device__ __forceinline__ uint32_t requestOf(const uint32_t* sums, uint32_t n, uint32_t x) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int32_t freePage(const cuttHipTablesArgs& a, uint32_t at) { return at < a.freeCount ? a.freePages[at] : -1; }

// Writes the new entries of the scanned requests' tables; `thread` of `threads` takes every `threads`-th page.
__device__ __forceinline__ void assignPages(const cuttHipTablesArgs& a, uint32_t first, uint32_t n, const Scan& s, uint32_t thread, uint32_t threads) {
  for (uint64_t at = (uint64_t)s.pages[0] + thread; at < s.pages[n]; at += threads) {
    const uint32_t i = requestOf(s.pages, n, (uint32_t)at), b = first + i;
    const uint32_t j = min(pagesFor(s.cached[i], a.pageSize), a.tableWidth) + ((uint32_t)at - s.pages[i]);
    if (j < a.tableWidth) a.tables[(uint64_t)b * a.tableWidth + j] = freePage(a, (uint32_t)at);  // (always, unless sums were capped)
  }
}

// The requests are few enough for one scan: every workgroup makes it for itself and takes its share of the tokens and the pages.  A new token's page
// comes from the free list, not from the table, whose new entries another workgroup may still have to write.
__global__ __launch_bounds__(kThreads) void pageTablesKernel(cuttHipTablesArgs a) {
  __shared__ Scan s;
  const uint32_t n = a.requests, thread = blockIdx.x * kThreads + threadIdx.x, threads = gridDim.x * kThreads;
  scanRequests(a, 0, n, 0, 0, s);
  if (blockIdx.x == 0) {
    for (uint32_t b = threadIdx.x; b <= n; b += kThreads) a.starts[b] = (int32_t)s.tokens[b];
    if (threadIdx.x == 0) a.used[0] = (int32_t)s.pages[n];
  }
  for (uint64_t i = thread; i < a.tokens; i += threads) {
    int64_t slot = -1;
    int32_t position = -1;
    if (i < s.tokens[n]) {
      const uint32_t b = requestOf(s.tokens, n, (uint32_t)i);
      const uint32_t cached = s.cached[b], owned = pagesFor(cached, a.pageSize);
      const uint32_t p = capped(cached, (uint32_t)i - s.tokens[b]), j = p / a.pageSize;
      position = (int32_t)p;
      if (j < a.tableWidth) {
        const int32_t page = j < owned ? a.tables[(uint64_t)b * a.tableWidth + j] : freePage(a, capped(s.pages[b], j - owned));
        if (page >= 0) slot = (int64_t)page * a.pageSize + (p - j * a.pageSize);
      }
    }
    a.slots[i] = slot;
    if (a.positions) a.positions[i] = position;
  }
  assignPages(a, 0, n, s, thread, threads);
}

// Any number of requests: one workgroup scans them part by part and writes the tables, a second launch looks the tokens up.
__global__ __launch_bounds__(kThreads) void pageTablesLongKernel(cuttHipTablesArgs a) {
  __shared__ Scan s;
  uint32_t tokens = 0, pages = 0;
  for (uint32_t first = 0; first < a.requests; first += kScan) {
    const uint32_t n = min(a.requests - first, kScan);
    scanRequests(a, first, n, tokens, pages, s);
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) a.starts[first + i] = (int32_t)s.tokens[i];
    assignPages(a, first, n, s, threadIdx.x, kThreads);
    tokens = s.tokens[n];
    pages = s.pages[n];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    a.starts[a.requests] = (int32_t)tokens;
    a.used[0] = (int32_t)pages;
  }
}

__global__ __launch_bounds__(kThreads) void pageSlotsKernel(cuttHipTablesArgs a) {
  const uint32_t* const starts = reinterpret_cast<const uint32_t*>(a.starts);
  const uint32_t all = starts[a.requests];
  for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < a.tokens; i += (uint64_t)gridDim.x * kThreads) {
    int64_t slot = -1;
    int32_t position = -1;
    if (i < all) {
      const uint32_t b = requestOf(starts, a.requests, (uint32_t)i);
      const uint32_t p = capped(max(a.cached[b], 0), (uint32_t)i - starts[b]), j = p / a.pageSize;
      position = (int32_t)p;
      const int32_t page = j < a.tableWidth ? a.tables[(uint64_t)b * a.tableWidth + j] : -1;
      if (page >= 0) slot = (int64_t)page * a.pageSize + (p - j * a.pageSize);
    }
    a.slots[i] = slot;
    if (a.positions) a.positions[i] = position;
  }
}

// ---------------------------------------------------------------------------
// Rows to their slots and back.  Bound by memory: every row is read once and written once.  131072 tokens, 8 heads of 128 bfloat16, keys and values
// (1075 MB), out of pages [page, head, slot] to [head, token] 176 us (6.1 TB/s), into them from a projection's output 199 us, into pages
// [page, slot, head] 214; 256 tokens 2.6 us.
// ---------------------------------------------------------------------------
constexpr uint32_t kMaxBlocks = 1u << 20;
constexpr int kPerLane = 2;  // vectors a lane keeps in flight; that load: 180 us with one, 175 with two, 190 with four, 197 with eight

struct PageMove {
  uint32_t tokens, rowBytes;
  uint32_t heads, vecs;                 // vectors per row
  uint32_t groupTokens, groupItems;     // a workgroup's tokens at a time, and their vectors
  cuttHipDivisor byVecs, byInner;       // inner: what runs faster of a group's tokens and heads
  uint32_t pages, pageSize;
  int wideSlots;                        // pages * pageSize is 2^31 or more
  cuttHipDivisor byPage;
  const int64_t* slots;
  uint8_t* rows[2];
  uint8_t* cache[2];
  uint64_t tokenStride, headStride, pageStride, slotStride, cacheHeadStride;  // in bytes
};

// A workgroup takes a few tokens' rows of all heads at a time, N bytes per lane.  TOKENS_INNER: neighbouring lanes go from a row to the next
// token's of the same head, else to the next head's: as the written side has them.  131072 tokens, 8 heads of 80 bfloat16, whose rows share lines, pages
// [page, slot, head]: into pages of one slot 130 us so and 151 the other way, out of them into [head, token] 128 and 155, out of pages of 16 slots 125 and
// 151; [page, head, slot] into [token, head] 125 and 134.  Rows on the grid hardly care: that last one of 128 elements 169 us so, 167 the other way.
template <int N, bool LOAD, bool TOKENS_INNER, bool NT>
__global__ __launch_bounds__(kThreads) void pageMoveKernel(PageMove a) {
  uint8_t* const rows = a.rows[blockIdx.y];
  uint8_t* const cache = a.cache[blockIdx.y];
  const uint64_t allSlots = (uint64_t)a.pages * a.pageSize;
  for (uint64_t group = (uint64_t)blockIdx.x * a.groupTokens; group < a.tokens; group += (uint64_t)gridDim.x * a.groupTokens)
    for (uint32_t item = threadIdx.x; item < a.groupItems; item += kThreads * kPerLane) {
      Pack<uint8_t, N> v[kPerLane];
      uint8_t *row[kPerLane], *cell[kPerLane];
      bool mine[kPerLane], there[kPerLane];
      int64_t slot[kPerLane];
      uint32_t head[kPerLane], at[kPerLane];
#pragma unroll
      for (int u = 0; u < kPerLane; u++) {
        const uint32_t i = min(item + u * kThreads, a.groupItems - 1), q = divide(i, a.byVecs), outer = divide(q, a.byInner);
        const uint32_t inner = q - outer * (TOKENS_INNER ? a.groupTokens : a.heads);
        head[u] = TOKENS_INNER ? outer : inner;
        const uint64_t token = group + (TOKENS_INNER ? inner : outer);
        mine[u] = item + u * kThreads < a.groupItems && token < a.tokens;
        at[u] = min((i - q * a.vecs) * N, a.rowBytes - N);
        const uint64_t t = min(token, (uint64_t)a.tokens - 1);
        slot[u] = a.slots[t];
        row[u] = rows + (t * a.tokenStride + head[u] * a.headStride + at[u]);
      }
#pragma unroll
      for (int u = 0; u < kPerLane; u++) {
        there[u] = (uint64_t)slot[u] < allSlots;
        const uint64_t s = there[u] ? slot[u] : 0;
        const uint64_t page = a.wideSlots ? s / a.pageSize : divide((uint32_t)s, a.byPage);
        cell[u] = cache + (page * a.pageStride + (s - page * a.pageSize) * a.slotStride + head[u] * a.cacheHeadStride + at[u]);
        if (LOAD) {
          v[u] = {};
          if (mine[u] && there[u]) v[u].template load<NT>(cell[u]);
        } else {
          v[u].template load<NT>(row[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < kPerLane; u++) {
        if (LOAD) {
          if (mine[u]) v[u].template store<NT>(row[u]);
        } else {
          if (mine[u] && there[u]) v[u].template store<NT>(cell[u]);
        }
      }
    }
}

template <int N, bool NT>
int movePages(const PageMove& a, bool load, bool tokensInner, dim3 grid, void* stream) {
  auto kernel = load ? (tokensInner ? pageMoveKernel<N, true, true, NT> : pageMoveKernel<N, true, false, NT>)
                     : (tokensInner ? pageMoveKernel<N, false, true, NT> : pageMoveKernel<N, false, false, NT>);
  return launchRows(kernel, grid, kThreads, 0, stream, a);
}

}  // namespace

extern "C" int cuttHipPageTables(const cuttHipTablesArgs* a, void* stream) {
  const uint64_t most = a->tokens > a->requests ? a->tokens : a->requests;
  const uint64_t groups = (most + kThreads - 1) / kThreads;
  if (a->requests <= kScan)
    return launchRows(pageTablesKernel, groups < 1 ? 1 : groups < 1024 ? groups : 1024, kThreads, 0, stream, *a);
  if (int e = launchRows(pageTablesLongKernel, 1, kThreads, 0, stream, *a)) return e;
  if (!a->tokens) return 0;
  return launchRows(pageSlotsKernel, groups < kMaxBlocks ? groups : kMaxBlocks, kThreads, 0, stream, *a);
}

extern "C" int cuttHipPageMove(const cuttHipPageArgs* a, void* stream) {
  PageMove m;
  const uint64_t size = a->elemSize;
  m.tokens = a->tokens;
  m.rowBytes = (uint32_t)(a->width * size);
  m.heads = a->heads;
  const uint32_t n = m.rowBytes >= 16 ? 16 : m.rowBytes % 4 == 0 ? 4 : 1;
  m.vecs = (m.rowBytes + n - 1) / n;
  const uint32_t perToken = m.vecs * m.heads;
  m.groupTokens = kThreads * kPerLane / perToken;
  if (m.groupTokens < 1) m.groupTokens = 1;
  if (m.groupTokens > m.tokens) m.groupTokens = m.tokens;
  m.groupItems = m.groupTokens * perToken;
  const bool tokensInner = cuttHipTokensInner(a);
  m.byVecs = cuttHipMakeDivisor(m.vecs);
  m.byInner = cuttHipMakeDivisor(tokensInner ? m.groupTokens : m.heads);
  m.pages = a->pages;
  m.pageSize = a->pageSize;
  m.wideSlots = (uint64_t)a->pages * a->pageSize > 0x7fffffffull;
  m.byPage = cuttHipMakeDivisor(a->pageSize);
  m.slots = a->slots;
  for (int i = 0; i < 2; i++) {
    m.rows[i] = (uint8_t*)a->rows[i];
    m.cache[i] = (uint8_t*)a->cache[i];
  }
  m.tokenStride = a->tokenStride * size;
  m.headStride = a->headStride * size;
  m.pageStride = a->pageStride * size;
  m.slotStride = a->slotStride * size;
  m.cacheHeadStride = a->cacheHeadStride * size;
  const uint32_t groups = (m.tokens + m.groupTokens - 1) / m.groupTokens;
  const dim3 grid(groups < kMaxBlocks ? groups : kMaxBlocks, a->rows[1] ? 2 : 1);
  const bool load = a->load != 0;
  if (n == 4) return movePages<4, false>(m, load, tokensInner, grid, stream);
  if (n == 1) return movePages<1, false>(m, load, tokensInner, grid, stream);
  if (pastCaches(m.tokens, (uint64_t)m.rowBytes * m.heads * (a->rows[1] ? 2 : 1))) return movePages<16, true>(m, load, tokensInner, grid, stream);
  return movePages<16, false>(m, load, tokensInner, grid, stream);
}
