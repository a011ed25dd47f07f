/*
 * rows_api.cpp - the exported row operators (cutt_rows.h): argument checks, then one call into the
 * kernels' layer (row_layer.h).  Pure host C++; nothing here allocates or throws.
 */
#include <climits>
#include <cstdint>

#include "../../include/cutt_rows.h"
#include "row_layer.h"

namespace {

typedef unsigned __int128 Wide;

// Byte ranges beyond this are no device buffer's (and keep the kernels' 64-bit offsets exact).
constexpr Wide kMaxBytes = (Wide)1 << 62;

// A device buffer as a call's arguments describe it: from its first to its last byte, as rows of `row` bytes every `pitch` bytes; one piece (values, a
// row, a row that is read again and again) has no pitch.
struct Span {
  uintptr_t at = 0;
  Wide bytes = 0;
  Wide row = 0, pitch = 0;
};

// Whether two buffers may share a byte.  Rows lie apart if they do so modulo a number that divides both pitches (one piece takes any): they are then columns side
// by side in the rows of a larger buffer.  Exact for equal pitches and for one piece; other pitches may be taken for overlapping where they are not.
bool overlap(const Span& a, const Span& b) {
  if (!a.bytes || !b.bytes || a.at >= b.at + b.bytes || b.at >= a.at + a.bytes) return false;
  Wide pitch = a.pitch;
  for (Wide r = b.pitch; r;) {  // the greatest common divisor
    const Wide rest = pitch % r;
    pitch = r;
    r = rest;
  }
  if (!pitch) return true;
  const Wide apart = (b.at >= a.at ? b.at - a.at : pitch - (a.at - b.at) % pitch) % pitch;  // from a's columns to b's
  return !(apart >= a.row && apart + b.row <= pitch);
}

bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// `count` contiguous values of `size` bytes.
bool values(const void* p, unsigned long long count, size_t size, Span& s) {
  s = {(uintptr_t)p, (Wide)count * size, (Wide)count * size, 0};
  return count == 0 || (p && aligned(p, size) && s.bytes <= kMaxBytes);
}

// The axes of a strided buffer that have more than one entry, the smallest stride first; in elements.
struct Axes {
  int n = 0;
  unsigned long long extent[3];
  Wide stride[3];
};

// Extents and strides in elements along each of n axes over `width` contiguous elements.  Strides are 0 and more; of what is written each has to lead past
// everything that the smaller ones reach, so that no two entries share an element.
bool strided(const void* p, int n, const unsigned long long* extent, const long long* stride, bool written, unsigned long long width, size_t size, Span& s,
             Axes& axes) {
  s = {(uintptr_t)p, 0, 0, 0};
  axes.n = 0;
  Wide last = 0;
  for (int i = 0; i < n; i++)
    if (extent[i] == 0) return true;
  if (width == 0) return true;
  if (!p || !aligned(p, size)) return false;
  for (int i = 0; i < n; i++) {
    if (extent[i] == 1) continue;
    if (stride[i] < 0) return false;
    last += (Wide)(extent[i] - 1) * (Wide)stride[i];
    if (last > kMaxBytes) return false;
    int at = axes.n++;
    for (; at > 0 && axes.stride[at - 1] > (Wide)stride[i]; at--) {
      axes.extent[at] = axes.extent[at - 1];
      axes.stride[at] = axes.stride[at - 1];
    }
    axes.extent[at] = extent[i];
    axes.stride[at] = (Wide)stride[i];
  }
  Wide reach = width;
  for (int i = 0; written && i < axes.n; i++) {
    if (axes.stride[i] < reach) return false;
    reach += (axes.extent[i] - 1) * axes.stride[i];
  }
  s.bytes = s.row = (last + width) * size;
  if (n == 1 && extent[0] > 1) {
    s.row = (Wide)width * size;
    s.pitch = (Wide)stride[0] * size;
  }
  return s.bytes <= kMaxBytes;
}

bool rowsRead(const void* p, unsigned long long count, long long stride, unsigned long long width, size_t size, Span& s) {
  Axes axes;
  return strided(p, 1, &count, &stride, false, width, size, s, axes);
}
bool rowsWritten(const void* p, unsigned long long count, long long stride, unsigned long long width, size_t size, Span& s) {
  Axes axes;
  return strided(p, 1, &count, &stride, true, width, size, s, axes);
}

// Whether two buffers of the same written axes, the second one `apart` bytes behind the first, share a byte: whether `apart` is less than a row off a sum of
// steps along the axes.  What the smaller strides reach either way, with a row, stays within one step of an axis, so that only the two multiples of its stride
// around what is left to go can lead there.
bool meet(__int128 apart, const Axes& axes, int n, unsigned long long width, size_t size) {
  if (n == 0) return (apart < 0 ? -apart : apart) < (__int128)width * (__int128)size;
  const __int128 stride = (__int128)(axes.stride[n - 1] * size), most = axes.extent[n - 1] - 1;
  __int128 steps = apart / stride;
  if (steps * stride > apart) steps--;  // (rounded down)
  for (int i = 0; i < 2; i++, steps++)
    if (steps <= most && -steps <= most && meet(apart - steps * stride, axes, n - 1, width, size)) return true;
  return false;
}

size_t sizeOf(cuttRowType type) { return type == CUTT_F32 ? 4 : type == CUTT_F16 || type == CUTT_BF16 ? 2 : 0; }

bool opaqueSize(size_t s) { return s == 1 || s == 2 || s == 4 || s == 8; }

cuttResult launched(int e) { return e == 0 ? CUTT_SUCCESS : CUTT_INTERNAL_ERROR; }

// The sizes that the calls on sorted rows share.
bool rowSizes(int tokens, int choices, int rows, int width) {
  return tokens >= 0 && choices >= 1 && rows >= 0 && width >= 1 && (long long)tokens * choices <= INT_MAX;
}

cuttHipExpertArgs rowArgs(int tokens, int choices, int rows, int width, const int* position, const int* source, const float* weights) {
  cuttHipExpertArgs a;
  a.tokens = (uint32_t)tokens;
  a.choices = (uint32_t)choices;
  a.rows = (uint32_t)rows;
  a.width = (uint32_t)width;
  a.position = position;
  a.source = source;
  a.weights = weights;
  return a;
}

// The weighted sum of every token's rows, which the gradient of dispatch is too.
cuttResult sumRows(int tokens, int choices, int rows, int width, cuttRowType type, hipStream_t stream, const int* position,
                   const float* weights, bool weighted, const void* y, long long yStride, void* out, long long outStride) {
  const size_t size = sizeOf(type);
  if (!size || !rowSizes(tokens, choices, rows, width)) return CUTT_INVALID_PARAMETER;
  const unsigned long long n = (unsigned long long)tokens * choices;
  Span p, w, from, to;
  if (!values(position, n, 4, p) || !values(weights, weighted ? n : 0, 4, w) || !rowsRead(y, rows, yStride, width, size, from) ||
      !rowsWritten(out, tokens, outStride, width, size, to))
    return CUTT_INVALID_PARAMETER;
  if (overlap(to, from) || overlap(to, p) || overlap(to, w)) return CUTT_INVALID_PARAMETER;
  if (tokens == 0) return CUTT_SUCCESS;
  const cuttHipExpertArgs a = rowArgs(tokens, choices, rows, width, position, nullptr, weighted ? weights : nullptr);
  return launched(cuttHipCombine(&a, (int)type, y, (uint64_t)yStride, out, (uint64_t)outStride, stream));
}

cuttResult movePages(bool load, int tokens, int heads, int width, size_t sizeofType, int pages, int pageSize, hipStream_t stream,
                     const long long* slots, const void* k, const void* v, const long long* rowStrides, const void* kCache, const void* vCache,
                     const long long* cacheStrides) {
  if (tokens < 0 || heads < 1 || width < 1 || !opaqueSize(sizeofType) || pages < 0 || pageSize < 1 || !rowStrides || !cacheStrides)
    return CUTT_INVALID_PARAMETER;
  if ((Wide)heads * (Wide)width * sizeofType > INT_MAX) return CUTT_INVALID_PARAMETER;
  const unsigned long long rowExtent[2] = {(unsigned long long)tokens, (unsigned long long)heads};
  const unsigned long long cacheExtent[3] = {(unsigned long long)pages, (unsigned long long)pageSize, (unsigned long long)heads};
  Span s, row[2], cache[2];
  Axes rowAxes, cacheAxes;  // (the same for both tensors)
  if (!values(slots, tokens, 8, s)) return CUTT_INVALID_PARAMETER;
  const void* const rowsAt[2] = {k, v};
  const void* const cacheAt[2] = {kCache, vCache};
  const int tensors = v || vCache ? 2 : 1;  // (one of the two may be null if it has no entries)
  for (int i = 0; i < tensors; i++)
    if (!strided(rowsAt[i], 2, rowExtent, rowStrides, load, width, sizeofType, row[i], rowAxes) ||
        !strided(cacheAt[i], 3, cacheExtent, cacheStrides, !load, width, sizeofType, cache[i], cacheAxes))
      return CUTT_INVALID_PARAMETER;
  for (int i = 0; i < tensors; i++) {
    for (int j = 0; j < tensors; j++)
      if (overlap(row[i], cache[j])) return CUTT_INVALID_PARAMETER;
    if (overlap(load ? row[i] : cache[i], s)) return CUTT_INVALID_PARAMETER;
  }
  const Span* const out = load ? row : cache;
  const Axes& outAxes = load ? rowAxes : cacheAxes;
  if (out[0].bytes && out[1].bytes && meet((__int128)out[1].at - (__int128)out[0].at, outAxes, outAxes.n, width, sizeofType)) return CUTT_INVALID_PARAMETER;
  if (tokens == 0 || (!load && pages == 0)) return CUTT_SUCCESS;
  cuttHipPageArgs a;
  a.tokens = (uint32_t)tokens;
  a.heads = (uint32_t)heads;
  a.width = (uint32_t)width;
  a.elemSize = (uint32_t)sizeofType;
  a.pages = (uint32_t)pages;
  a.pageSize = (uint32_t)pageSize;
  a.slots = (const int64_t*)slots;
  for (int i = 0; i < 2; i++) {
    a.rows[i] = const_cast<void*>(rowsAt[i]);
    a.cache[i] = const_cast<void*>(pages ? cacheAt[i] : rowsAt[i]);  // (a cache without pages is never touched and may be null)
  }
  // (the stride of an axis with one entry is never used: it may be anything)
  a.tokenStride = tokens > 1 ? (uint64_t)rowStrides[0] : 0;
  a.headStride = heads > 1 ? (uint64_t)rowStrides[1] : 0;
  a.pageStride = pages > 1 ? (uint64_t)cacheStrides[0] : 0;
  a.slotStride = pageSize > 1 ? (uint64_t)cacheStrides[1] : 0;
  a.cacheHeadStride = heads > 1 ? (uint64_t)cacheStrides[2] : 0;
  a.load = load;
  return launched(cuttHipPageMove(&a, stream));
}

}  // namespace

extern "C" long long cuttExpertRows(int tokens, int choices, int experts, int align) {
  if (tokens < 0 || choices < 1 || experts < 1 || experts > CUTT_MAX_EXPERTS || align < 1) return -1;
  const long long n = (long long)tokens * choices;
  if (n > INT_MAX) return -1;
  const long long rows = n + (n < experts ? n : experts) * (long long)(align - 1);
  return rows > INT_MAX ? -1 : rows;
}

extern "C" size_t cuttExpertSortWorkspace(int tokens, int choices, int experts) {
  if (cuttExpertRows(tokens, choices, experts, 1) < 0) return 0;
  return cuttHipSortWorkspace((uint32_t)tokens * (uint32_t)choices, (uint32_t)experts);
}

extern "C" cuttResult cuttExpertSort(int tokens, int choices, int firstExpert, int experts, int align, int rows, size_t sizeofId,
                                     hipStream_t stream, const void* ids, int* counts, int* offsets, int* position, int* source, void* workspace,
                                     size_t workspaceBytes) {
  if (cuttExpertRows(tokens, choices, experts, align) < 0 || rows < 0 || (sizeofId != 4 && sizeofId != 8)) return CUTT_INVALID_PARAMETER;
  const unsigned long long n = (unsigned long long)tokens * choices;
  const size_t space = cuttExpertSortWorkspace(tokens, choices, experts);
  if (workspaceBytes < space) return CUTT_INVALID_PARAMETER;
  Span in, out[5];
  if (!values(ids, n, sizeofId, in) || !values(counts, experts, 4, out[0]) || !values(offsets, (unsigned long long)experts + 1, 4, out[1]) ||
      !values(position, n, 4, out[2]) || !values(source, rows, 4, out[3]) || !values(workspace, space / 4, 4, out[4]))
    return CUTT_INVALID_PARAMETER;
  for (int i = 0; i < 5; i++) {
    if (overlap(in, out[i])) return CUTT_INVALID_PARAMETER;
    for (int j = 0; j < i; j++)
      if (overlap(out[i], out[j])) return CUTT_INVALID_PARAMETER;
  }
  cuttHipSortArgs a;
  a.n = (uint32_t)n;
  a.firstExpert = firstExpert;
  a.experts = (uint32_t)experts;
  a.align = (uint32_t)align;
  a.rows = (uint32_t)rows;
  a.idBytes = (uint32_t)sizeofId;
  a.ids = ids;
  a.counts = counts;
  a.offsets = offsets;
  a.position = position;
  a.source = source;
  a.workspace = (uint32_t*)workspace;
  return launched(cuttHipExpertSort(&a, stream));
}

extern "C" cuttResult cuttExpertDispatch(int tokens, int choices, int rows, int width, size_t sizeofType, hipStream_t stream, const int* position,
                                         const int* source, const void* x, long long xStride, void* y, long long yStride) {
  if (!opaqueSize(sizeofType) || !rowSizes(tokens, choices, rows, width)) return CUTT_INVALID_PARAMETER;
  const unsigned long long n = (unsigned long long)tokens * choices;
  Span p, s, from, to;
  if (!values(position, n, 4, p) || !values(source, rows, 4, s) || !rowsRead(x, tokens, xStride, width, sizeofType, from) ||
      !rowsWritten(y, rows, yStride, width, sizeofType, to))
    return CUTT_INVALID_PARAMETER;
  if (overlap(to, from) || overlap(to, p) || overlap(to, s)) return CUTT_INVALID_PARAMETER;
  if (rows == 0) return CUTT_SUCCESS;
  const cuttHipExpertArgs a = rowArgs(tokens, choices, rows, width, position, source, nullptr);
  return launched(cuttHipDispatch(&a, (uint32_t)sizeofType, x, (uint64_t)xStride, y, (uint64_t)yStride, stream));
}

extern "C" cuttResult cuttExpertDispatchBackward(int tokens, int choices, int rows, int width, cuttRowType type, hipStream_t stream,
                                                 const int* position, const void* dy, long long dyStride, void* dx, long long dxStride) {
  return sumRows(tokens, choices, rows, width, type, stream, position, nullptr, false, dy, dyStride, dx, dxStride);
}

extern "C" cuttResult cuttExpertCombine(int tokens, int choices, int rows, int width, cuttRowType type, hipStream_t stream, const int* position,
                                        const float* weights, const void* y, long long yStride, void* out, long long outStride) {
  return sumRows(tokens, choices, rows, width, type, stream, position, weights, true, y, yStride, out, outStride);
}

extern "C" cuttResult cuttExpertCombineBackward(int tokens, int choices, int rows, int width, cuttRowType type, hipStream_t stream,
                                                const int* position, const int* source, const float* weights, const void* y, long long yStride,
                                                const void* dout, long long doutStride, void* dy, long long dyStride, float* dweights) {
  const size_t size = sizeOf(type);
  if (!size || !rowSizes(tokens, choices, rows, width)) return CUTT_INVALID_PARAMETER;
  const unsigned long long n = (unsigned long long)tokens * choices;
  // (a buffer of no entries may be null without being left out)
  if (!dy && rows != 0 && !dweights && n != 0) return CUTT_INVALID_PARAMETER;
  const bool anyRows = rows != 0 && dy, anyWeights = n != 0 && dweights;
  // What only the other gradient needs is neither checked nor passed on.
  Span p, s, w, yIn, dIn, dyOut, dwOut;
  if (!values(position, n, 4, p) || !rowsRead(dout, tokens, doutStride, width, size, dIn)) return CUTT_INVALID_PARAMETER;
  if (anyRows && (!values(source, rows, 4, s) || !values(weights, n, 4, w) || !rowsWritten(dy, rows, dyStride, width, size, dyOut)))
    return CUTT_INVALID_PARAMETER;
  if (anyWeights && (!values(dweights, n, 4, dwOut) || !rowsRead(y, rows, yStride, width, size, yIn))) return CUTT_INVALID_PARAMETER;
  const Span reads[] = {p, s, w, yIn, dIn};
  for (const Span& r : reads)
    if (overlap(dyOut, r) || overlap(dwOut, r)) return CUTT_INVALID_PARAMETER;
  if (overlap(dyOut, dwOut)) return CUTT_INVALID_PARAMETER;
  if (!anyRows && !anyWeights) return CUTT_SUCCESS;
  const cuttHipExpertArgs a = rowArgs(tokens, choices, rows, width, position, anyRows ? source : nullptr, anyRows ? weights : nullptr);
  return launched(cuttHipCombineBackward(&a, (int)type, anyWeights ? y : nullptr, (uint64_t)yStride, dout, (uint64_t)doutStride, anyRows ? dy : nullptr, (uint64_t)dyStride,
                                         anyWeights ? dweights : nullptr, stream));
}

extern "C" cuttResult cuttPageTables(int requests, int pageSize, int tableWidth, int freeCount, int tokens, hipStream_t stream, const int* cached,
                                     const int* added, const int* freePages, int* tables, int* starts, int* used, long long* slots, int* positions) {
  if (requests < 0 || pageSize < 1 || tableWidth < 1 || freeCount < 0 || tokens < 0) return CUTT_INVALID_PARAMETER;
  const unsigned long long n = (unsigned long long)requests;
  Span in[3], out[5];
  if (!values(cached, n, 4, in[0]) || !values(added, n, 4, in[1]) || !values(freePages, freeCount, 4, in[2]) ||
      !values(tables, n * (unsigned long long)tableWidth, 4, out[0]) || !values(starts, n + 1, 4, out[1]) || !values(used, 1, 4, out[2]) ||
      !values(slots, tokens, 8, out[3]) || !values(positions, positions ? tokens : 0, 4, out[4]))
    return CUTT_INVALID_PARAMETER;
  for (int i = 0; i < 5; i++) {
    for (int j = 0; j < 3; j++)
      if (overlap(out[i], in[j])) return CUTT_INVALID_PARAMETER;
    for (int j = 0; j < i; j++)
      if (overlap(out[i], out[j])) return CUTT_INVALID_PARAMETER;
  }
  cuttHipTablesArgs a;
  a.requests = (uint32_t)requests;
  a.pageSize = (uint32_t)pageSize;
  a.tableWidth = (uint32_t)tableWidth;
  a.freeCount = (uint32_t)freeCount;
  a.tokens = (uint32_t)tokens;
  a.cached = cached;
  a.added = added;
  a.freePages = freePages;
  a.tables = tables;
  a.starts = starts;
  a.used = used;
  a.slots = (int64_t*)slots;
  a.positions = positions;
  return launched(cuttHipPageTables(&a, stream));
}

extern "C" cuttResult cuttPageStore(int tokens, int heads, int width, size_t sizeofType, int pages, int pageSize, hipStream_t stream,
                                    const long long* slots, const void* k, const void* v, const long long* rowStrides, void* kCache, void* vCache,
                                    const long long* cacheStrides) {
  return movePages(false, tokens, heads, width, sizeofType, pages, pageSize, stream, slots, k, v, rowStrides, kCache, vCache, cacheStrides);
}

extern "C" cuttResult cuttPageLoad(int tokens, int heads, int width, size_t sizeofType, int pages, int pageSize, hipStream_t stream,
                                   const long long* slots, void* k, void* v, const long long* rowStrides, const void* kCache, const void* vCache,
                                   const long long* cacheStrides) {
  return movePages(true, tokens, heads, width, sizeofType, pages, pageSize, stream, slots, k, v, rowStrides, kCache, vCache, cacheStrides);
}
