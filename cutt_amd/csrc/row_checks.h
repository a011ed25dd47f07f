/*
 * row_checks.h - the argument checks that the row operators' and the products' host code share (rows_api.cpp, products_api.cpp): what a buffer's
 * arguments describe, and whether two buffers share a byte.  Pure host C++; nothing here allocates or throws.
 */
#ifndef CUTT_ROW_CHECKS_H
#define CUTT_ROW_CHECKS_H

#include <climits>
#include <cstdint>

#include "../../include/cutt_rows.h"

namespace {

typedef unsigned __int128 Wide;

// Byte ranges beyond this are no device buffer's (and keep the kernels' 64-bit offsets exact).
constexpr Wide kMaxBytes = (Wide)1 << 62;

// A device buffer as a call's arguments describe it: from its first to its last byte, as rows of `row` bytes every `pitch` bytes (the largest stride; a row is what the others reach); one
// piece (values, a row, a row that is read again and again) has no pitch.
struct Span {
  uintptr_t at = 0;
  Wide bytes = 0;
  Wide row = 0, pitch = 0;
};

// Whether two buffers may share a byte.  Rows lie apart if they do so modulo a number that divides both pitches (one piece takes any): they are then columns side
// by side in the rows of a larger buffer.  Exact for equal pitches and for one piece; other pitches may be taken for overlapping where they are not.
inline bool overlap(const Span& a, const Span& b) {
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

inline bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// `count` contiguous values of `size` bytes.
inline bool values(const void* p, unsigned long long count, size_t size, Span& s) {
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
inline bool strided(const void* p, int n, const unsigned long long* extent, const long long* stride, bool written, unsigned long long width, size_t size, Span& s,
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
  if (axes.n) {
    s.pitch = axes.stride[axes.n - 1] * size;
    s.row -= (Wide)(axes.extent[axes.n - 1] - 1) * s.pitch;
  }
  return s.bytes <= kMaxBytes;
}

inline bool rowsRead(const void* p, unsigned long long count, long long stride, unsigned long long width, size_t size, Span& s) {
  Axes axes;
  return strided(p, 1, &count, &stride, false, width, size, s, axes);
}
inline bool rowsWritten(const void* p, unsigned long long count, long long stride, unsigned long long width, size_t size, Span& s) {
  Axes axes;
  return strided(p, 1, &count, &stride, true, width, size, s, axes);
}

// Whether two buffers of the same written axes, the second one `apart` bytes behind the first, share a byte: whether `apart` is less than a row off a sum of
// steps along the axes.  What the smaller strides reach either way, with a row, stays within one step of an axis, so that only the two multiples of its stride
// around what is left to go can lead there.
inline bool meet(__int128 apart, const Axes& axes, int n, unsigned long long width, size_t size) {
  if (n == 0) return (apart < 0 ? -apart : apart) < (__int128)width * (__int128)size;
  const __int128 stride = (__int128)(axes.stride[n - 1] * size), most = axes.extent[n - 1] - 1;
  __int128 steps = apart / stride;
  if (steps * stride > apart) steps--;  // (rounded down)
  for (int i = 0; i < 2; i++, steps++)
    if (steps <= most && -steps <= most && meet(apart - steps * stride, axes, n - 1, width, size)) return true;
  return false;
}

inline size_t sizeOf(cuttRowType type) { return type == CUTT_F32 ? 4 : type == CUTT_F16 || type == CUTT_BF16 ? 2 : 0; }

inline bool opaqueSize(size_t s) { return s == 1 || s == 2 || s == 4 || s == 8; }

inline cuttResult launched(int e) { return e == 0 ? CUTT_SUCCESS : CUTT_INTERNAL_ERROR; }

}  // namespace

#endif  // CUTT_ROW_CHECKS_H
