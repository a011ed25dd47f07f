/*
 * product_layer.h - the C-ABI layer between the products' host code (products_api.cpp) and their kernels
 * (product_kernels.hip, attend_kernels.hip).  Plain C types; a stream travels as void*.  Every function launches and returns 0, or
 * the hipError_t value of a refused launch.  The arguments have been checked (cutt_products.h).
 */
#ifndef CUTT_PRODUCT_LAYER_H
#define CUTT_PRODUCT_LAYER_H

#include "../../include/cutt_products.h"
#include "row_layer.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Strides in elements; that of an axis with one entry is 0. */
typedef struct cuttHipProductArgs {
  uint32_t rows, groups, inner, outer; /* rows and groups above 0 */
  const int32_t* offsets;
  const void *x, *w;                   /* w: the second factor, dy for the weights' gradient */
  void* y;                             /* dw for the weights' gradient */
  uint64_t xStride, yStride;           /* (yStride of dw: from row to row of a group) */
  uint64_t wGroup, wRow;               /* (wGroup of dw: from group to group of dw; wRow: the row stride of dy) */
} cuttHipProductArgs;

int cuttHipGroupedProduct(const cuttHipProductArgs* a, int type, int transposed, void* stream);
int cuttHipGroupedWeights(const cuttHipProductArgs* a, int type, void* stream);

typedef struct cuttHipAttendArgs {
  uint32_t queries, requests, heads, keyHeads, width;
  uint32_t pages, pageSize, tableWidth, window; /* window 0: none */
  float scale;
  const int32_t *tables, *owners, *positions;   /* owners null: query i belongs to request i */
  const void *q, *k, *v;
  void* out;
  float* logSums;                               /* null: not wanted */
  uint64_t qStride, qHead, outStride, outHead;  /* elements; that of an axis with one entry is 0 */
  uint64_t pageStride, slotStride, cacheHead;
  void* workspace;
} cuttHipAttendArgs;

size_t cuttHipAttendWorkspace(uint32_t queries, uint32_t heads, uint32_t keyHeads, uint32_t width, uint32_t pageSize, uint32_t tableWidth, uint32_t window);
int cuttHipAttend(const cuttHipAttendArgs* a, int type, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CUTT_PRODUCT_LAYER_H */
