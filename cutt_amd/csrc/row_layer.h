/*
 * row_layer.h - the C-ABI layer between the row operators' host code (rows_api.cpp) and their kernels
 * (expert_kernels.hip, page_kernels.hip).  Plain C types; a stream travels as void*.  Every function launches and
 * returns 0, or the hipError_t value of a refused launch.  The arguments have been checked (cutt_rows.h): sizes are in range,
 * nothing that has to be there is null.
 */
#ifndef CUTT_ROW_LAYER_H
#define CUTT_ROW_LAYER_H

#include <stddef.h>
#include <stdint.h>

#include "hip_layer.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types as in cutt_rows.h: 0 = 32-bit, 1 = 16-bit, 2 = bfloat16. */
enum { CUTT_ROW_F32 = 0, CUTT_ROW_F16 = 1, CUTT_ROW_BF16 = 2 };

typedef struct cuttHipSortArgs {
  uint32_t n;             /* choices in all: tokens * choices, below 2^31 */
  int32_t firstExpert;
  uint32_t experts, align;
  uint32_t rows;
  uint32_t idBytes;       /* 4 or 8 */
  const void* ids;
  int32_t *counts, *offsets, *position, *source;
  uint32_t* workspace;
} cuttHipSortArgs;

size_t cuttHipSortWorkspace(uint32_t n, uint32_t experts);
int cuttHipExpertSort(const cuttHipSortArgs* a, void* stream);

/* Rows to experts and back.  Strides in elements. */
typedef struct cuttHipExpertArgs {
  uint32_t tokens, choices, rows, width;
  const int32_t *position, *source;
  const float* weights;   /* null: all ones */
} cuttHipExpertArgs;

int cuttHipDispatch(const cuttHipExpertArgs* a, uint32_t elemSize, const void* x, uint64_t xStride, void* y, uint64_t yStride,
                    void* stream);
int cuttHipCombine(const cuttHipExpertArgs* a, int type, const void* y, uint64_t yStride, void* out, uint64_t outStride, void* stream);
/* dy null or dweights null: not wanted */
int cuttHipCombineBackward(const cuttHipExpertArgs* a, int type, const void* y, uint64_t yStride, const void* dout,
                           uint64_t doutStride, void* dy, uint64_t dyStride, float* dweights, void* stream);

typedef struct cuttHipTablesArgs {
  uint32_t requests, pageSize, tableWidth, freeCount, tokens;
  const int32_t *cached, *added, *freePages;
  int32_t *tables, *starts, *used;
  int64_t* slots;
  int32_t* positions;     /* null: not wanted */
} cuttHipTablesArgs;

int cuttHipPageTables(const cuttHipTablesArgs* a, void* stream);

/* heads * width * elemSize is below 2^31. */
typedef struct cuttHipPageArgs {
  uint32_t tokens, heads, width, elemSize;
  uint32_t pages, pageSize;
  const int64_t* slots;
  void* rows[2];          /* k, v; rows[1] null: only k */
  void* cache[2];
  uint64_t tokenStride, headStride;                /* of rows, in elements */
  uint64_t pageStride, slotStride, cacheHeadStride; /* of the caches, in elements */
  int load;               /* 0: rows to the cache, 1: back */
} cuttHipPageArgs;

/* Whether neighbouring lanes go from a row to the next token's of the same head rather than to the next head's: as those come closer on the side that is
 * written, where lines that two rows share have to be put together (pageMoveKernel).  The next token's slot is the next one of its
 * page, or the next page where a page has one slot.  The stride of an axis with one entry is 0, and either order is then the same. */
static inline int cuttHipTokensInner(const cuttHipPageArgs* a) {
  if (a->load) return a->tokenStride < a->headStride;
  return (a->pageSize > 1 ? a->slotStride : a->pageStride) < a->cacheHeadStride;
}

int cuttHipPageMove(const cuttHipPageArgs* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CUTT_ROW_LAYER_H */
