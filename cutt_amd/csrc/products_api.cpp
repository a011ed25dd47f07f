/*
 * products_api.cpp - the exported products (cutt_products.h): argument checks, then one call into the
 * kernels' layer (product_layer.h).  Pure host C++; nothing here allocates or throws.
 */
#include "../../include/cutt_products.h"

#include <cmath>

#include "product_layer.h"
#include "row_checks.h"

namespace {

bool productSizes(int rows, int groups, int inner, int outer) {
  return rows >= 0 && groups >= 1 && groups <= CUTT_MAX_EXPERTS && inner >= 1 && outer >= 1;
}

// The stride of an axis of n entries as the kernels' layer takes it: that of a single entry is never used and may be anything.
uint64_t strideOf(long long stride, int n) { return n > 1 ? (uint64_t)stride : 0; }

bool attendSizes(int queries, int heads, int keyHeads, int width, int pageSize, int tableWidth, int window) {
  return queries >= 0 && heads >= 1 && heads <= CUTT_MAX_HEADS && keyHeads >= 1 && heads % keyHeads == 0 && (long long)queries * heads <= INT_MAX && width >= 1 &&
         width <= CUTT_MAX_HEAD_WIDTH && pageSize >= 1 && tableWidth >= 1 && window >= 0;
}

}  // namespace

extern "C" cuttResult cuttGroupedProduct(int rows, int groups, int inner, int outer, cuttRowType type, int transposed, hipStream_t stream,
                                         const int* offsets, const void* x, long long xStride, const void* w, const long long* wStrides, void* y,
                                         long long yStride) {
  const size_t size = sizeOf(type);
  if (!size || !productSizes(rows, groups, inner, outer) || !wStrides) return CUTT_INVALID_PARAMETER;
  const unsigned long long extent[2] = {(unsigned long long)groups, (unsigned long long)(transposed ? outer : inner)};
  Span o, from, weights, to;
  Axes axes;
  if (!values(offsets, (unsigned long long)groups + 1, 4, o) || !rowsRead(x, rows, xStride, inner, size, from) ||
      !strided(w, 2, extent, wStrides, false, transposed ? inner : outer, size, weights, axes) || !rowsWritten(y, rows, yStride, outer, size, to))
    return CUTT_INVALID_PARAMETER;
  if (overlap(to, from) || overlap(to, weights) || overlap(to, o)) return CUTT_INVALID_PARAMETER;
  if (rows == 0) return CUTT_SUCCESS;
  cuttHipProductArgs a;
  a.rows = (uint32_t)rows;
  a.groups = (uint32_t)groups;
  a.inner = (uint32_t)inner;
  a.outer = (uint32_t)outer;
  a.offsets = offsets;
  a.x = x;
  a.w = w;
  a.y = y;
  a.xStride = strideOf(xStride, rows);
  a.yStride = strideOf(yStride, rows);
  a.wGroup = strideOf(wStrides[0], groups);
  a.wRow = strideOf(wStrides[1], transposed ? outer : inner);
  return launched(cuttHipGroupedProduct(&a, (int)type, transposed != 0, stream));
}

extern "C" cuttResult cuttGroupedProductWeights(int rows, int groups, int inner, int outer, cuttRowType type, hipStream_t stream, const int* offsets,
                                                const void* x, long long xStride, const void* dy, long long dyStride, void* dw,
                                                const long long* dwStrides) {
  const size_t size = sizeOf(type);
  if (!size || !productSizes(rows, groups, inner, outer) || !dwStrides) return CUTT_INVALID_PARAMETER;
  const unsigned long long extent[2] = {(unsigned long long)groups, (unsigned long long)inner};
  Span o, from, grad, to;
  Axes axes;
  if (!values(offsets, (unsigned long long)groups + 1, 4, o) || !rowsRead(x, rows, xStride, inner, size, from) ||
      !rowsRead(dy, rows, dyStride, outer, size, grad) || !strided(dw, 2, extent, dwStrides, true, outer, size, to, axes))
    return CUTT_INVALID_PARAMETER;
  if (overlap(to, from) || overlap(to, grad) || overlap(to, o)) return CUTT_INVALID_PARAMETER;
  cuttHipProductArgs a;
  a.rows = (uint32_t)rows;
  a.groups = (uint32_t)groups;
  a.inner = (uint32_t)inner;
  a.outer = (uint32_t)outer;
  a.offsets = offsets;
  a.x = x;
  a.w = dy;
  a.y = dw;
  a.xStride = strideOf(xStride, rows);
  a.wRow = strideOf(dyStride, rows);
  a.wGroup = strideOf(dwStrides[0], groups);
  a.yStride = strideOf(dwStrides[1], inner);
  return launched(cuttHipGroupedWeights(&a, (int)type, stream));
}

extern "C" size_t cuttAttendPagesWorkspace(int queries, int heads, int keyHeads, int width, int pageSize, int tableWidth, int window) {
  if (!attendSizes(queries, heads, keyHeads, width, pageSize, tableWidth, window)) return 0;
  return cuttHipAttendWorkspace((uint32_t)queries, (uint32_t)heads, (uint32_t)keyHeads, (uint32_t)width, (uint32_t)pageSize, (uint32_t)tableWidth,
                                (uint32_t)window);
}

extern "C" cuttResult cuttAttendPages(int queries, int requests, int heads, int keyHeads, int width, cuttRowType type, int pages, int pageSize,
                                      int tableWidth, int window, float scale, hipStream_t stream, const int* tables, const int* owners,
                                      const int* positions, const void* q, const long long* qStrides, const void* kCache, const void* vCache,
                                      const long long* cacheStrides, void* out, const long long* outStrides, float* logSums, void* workspace,
                                      size_t workspaceBytes) {
  const size_t size = sizeOf(type);
  if (!size || !attendSizes(queries, heads, keyHeads, width, pageSize, tableWidth, window) || requests < 0 || pages < 0 || !std::isfinite(scale) ||
      !qStrides || !cacheStrides || !outStrides)
    return CUTT_INVALID_PARAMETER;
  const size_t space = cuttAttendPagesWorkspace(queries, heads, keyHeads, width, pageSize, tableWidth, window);
  if (workspaceBytes < space) return CUTT_INVALID_PARAMETER;
  const unsigned long long n = (unsigned long long)queries, rowExtent[2] = {n, (unsigned long long)heads};
  const unsigned long long cacheExtent[3] = {(unsigned long long)pages, (unsigned long long)pageSize, (unsigned long long)keyHeads};
  Span in[6], to[3];
  Axes axes;
  if (!values(tables, (unsigned long long)requests * (unsigned long long)tableWidth, 4, in[0]) || !values(owners, owners ? n : 0, 4, in[1]) ||
      !values(positions, n, 4, in[2]) || !strided(q, 2, rowExtent, qStrides, false, width, size, in[3], axes) ||
      !strided(kCache, 3, cacheExtent, cacheStrides, false, width, size, in[4], axes) ||
      !strided(vCache, 3, cacheExtent, cacheStrides, false, width, size, in[5], axes) || !strided(out, 2, rowExtent, outStrides, true, width, size, to[0], axes) ||
      !values(logSums, logSums ? n * (unsigned long long)heads : 0, 4, to[1]) || !values(workspace, space / 4, 4, to[2]))
    return CUTT_INVALID_PARAMETER;
  for (int i = 0; i < 3; i++) {
    for (int j = 0; j < 6; j++)
      if (overlap(to[i], in[j])) return CUTT_INVALID_PARAMETER;
    for (int j = 0; j < i; j++)
      if (overlap(to[i], to[j])) return CUTT_INVALID_PARAMETER;
  }
  if (queries == 0) return CUTT_SUCCESS;
  cuttHipAttendArgs a;
  a.queries = (uint32_t)queries;
  a.requests = (uint32_t)requests;
  a.heads = (uint32_t)heads;
  a.keyHeads = (uint32_t)keyHeads;
  a.width = (uint32_t)width;
  a.pages = (uint32_t)pages;
  a.pageSize = (uint32_t)pageSize;
  a.tableWidth = (uint32_t)tableWidth;
  a.window = (uint32_t)window;
  a.scale = scale;
  a.tables = tables;
  a.owners = owners;
  a.positions = positions;
  a.q = q;
  a.k = kCache;
  a.v = vCache;
  a.out = out;
  a.logSums = logSums;
  a.qStride = strideOf(qStrides[0], queries);
  a.qHead = strideOf(qStrides[1], heads);
  a.outStride = strideOf(outStrides[0], queries);
  a.outHead = strideOf(outStrides[1], heads);
  a.pageStride = strideOf(cacheStrides[0], pages);
  a.slotStride = strideOf(cacheStrides[1], pageSize);
  a.cacheHead = strideOf(cacheStrides[2], keyHeads);
  a.workspace = workspace;
  return launched(cuttHipAttend(&a, (int)type, stream));
}
