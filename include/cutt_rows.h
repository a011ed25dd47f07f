/*
 * cutt_rows.h - rows that move to places which only the GPU knows: tokens sorted by expert and back,
 * and keys and values that live in pages.  Beside the plan API of cutt.h, whose permutations the host
 * knows when it plans; the reference has no counterpart.
 *
 * Conventions:
 *   - a row is `width` contiguous elements; row strides are in elements, `width` and more for what is written, 0 and more for
 *     what is read; integers in device buffers are 32-bit unless said otherwise;
 *   - rows that only move are opaque (sizeofType 1, 2, 4 or 8 bytes per element) and keep their bits;
 *     rows that are summed have a cuttRowType, are summed in 32 bits and rounded once, to nearest even;
 *   - every call only launches kernels on `stream`, on the current device: it allocates nothing, keeps nothing,
 *     copies nothing and does not synchronise, and can be captured into a HIP graph (make the call once before
 *     the capture, so that the library's code object is loaded).  The caller orders work of other streams;
 *   - buffers are aligned to their elements; any such address and any stride will do, multiples of 16 bytes are
 *     fastest.  What a call writes must not overlap what it reads; columns side by side in one buffer of rows (equal strides,
 *     or a single row on either side) do not;
 *   - no buffer's contents can make a call touch memory outside the buffers as their sizes, strides and
 *     counts describe them: positions, slots, experts and pages out of range count as absent;
 *   - the results do not depend on timing: equal inputs give equal bits.  The one exception is a place that the caller's numbers
 *     name twice for writing (a row in two positions, a slot of two tokens): each of its elements is then one of those
 *     that were to go there, not said which, nor that its neighbours have the same origin.
 *
 * All functions return CUTT_SUCCESS, CUTT_INVALID_PARAMETER (null, misaligned or overlapping buffers, sizes out of range;
 * nothing was launched) or CUTT_INTERNAL_ERROR (the HIP runtime refused a launch).
 */
#ifndef CUTT_ROWS_H
#define CUTT_ROWS_H

#include "cutt.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of rows that are summed. */
typedef enum cuttRowType_t {
  CUTT_F32 = 0,
  CUTT_F16 = 1,
  CUTT_BF16 = 2
} cuttRowType;

#define CUTT_MAX_EXPERTS 1024

/* ---- rows sorted by expert and back ---------------------------------------
 *
 * A router gives each of `tokens` tokens `choices` experts.  Choice k of token t has the number
 * a = t * choices + k.  `rows` rows hold the choices sorted by expert, in the order of their numbers
 * within an expert, every expert's segment starting at a multiple of `align` rows:
 *
 *   counts[e]    choices of expert firstExpert + e, 0 <= e < experts
 *   offsets[0] = 0, offsets[e + 1] = offsets[e] + counts[e] rounded up to align
 *   position[a]  the row of choice a; -1 if its expert is not one of the `experts` (another device's, or none) or
 *                its row would not be below `rows`
 *   source[r]    the choice in row r, -1 if the row is empty
 */

/* Rows that suffice whatever the experts chosen are: tokens * choices + min(experts, tokens * choices) * (align - 1).  -1 if the
 * arguments are out of range (as for cuttExpertSort). */
long long cuttExpertRows(int tokens, int choices, int experts, int align);

/* Bytes of workspace that cuttExpertSort needs for these sizes (0: none, or arguments out of range). */
size_t cuttExpertSortWorkspace(int tokens, int choices, int experts);

/*
 *   tokens >= 0, choices >= 1, 1 <= experts <= CUTT_MAX_EXPERTS, align >= 1, rows >= 0; cuttExpertRows(...) < 2^31
 *   sizeofId          4 or 8: ids are 32-bit or 64-bit signed integers
 *   ids               [tokens, choices]
 *   counts            [experts]            offsets  [experts + 1]
 *   position          [tokens, choices]    source   [rows]
 *   workspace         cuttExpertSortWorkspace bytes, aligned to 4; its contents need no preparation and mean nothing afterwards.  Calls that
 *                     may overlap on the GPU need one each
 * offsets[experts] > rows says that rows did not suffice.
 */
cuttResult cuttExpertSort(int tokens, int choices, int firstExpert, int experts, int align, int rows, size_t sizeofId,
                          hipStream_t stream, const void* ids, int* counts, int* offsets, int* position, int* source,
                          void* workspace, size_t workspaceBytes);

/*
 * y[position[t, k], :] = x[t, :], and zeros in every row with source < 0.
 *   x [tokens, width] with row stride xStride, y [rows, width] with row stride yStride
 * position and source are those of one cuttExpertSort, here and below; rows whose source is >= 0 but that no position names are not written.
 */
cuttResult cuttExpertDispatch(int tokens, int choices, int rows, int width, size_t sizeofType, hipStream_t stream,
                              const int* position, const int* source, const void* x, long long xStride, void* y,
                              long long yStride);

/* Its gradient: dx[t, :] = sum over k of dy[position[t, k], :], k ascending; absent rows count as zeros. */
cuttResult cuttExpertDispatchBackward(int tokens, int choices, int rows, int width, cuttRowType type, hipStream_t stream,
                                      const int* position, const void* dy, long long dyStride, void* dx,
                                      long long dxStride);

/*
 * out[t, :] = sum over k of weights[t, k] * y[position[t, k], :], k ascending.
 *   weights           [tokens, choices] in 32-bit floating point
 * A choice without a row contributes nothing, whatever its weight; a row with weight 0 is multiplied all the same.
 */
cuttResult cuttExpertCombine(int tokens, int choices, int rows, int width, cuttRowType type, hipStream_t stream,
                             const int* position, const float* weights, const void* y, long long yStride, void* out,
                             long long outStride);

/*
 * Its gradients:
 *   dy[position[t, k], :] = weights[t, k] * dout[t, :], and zeros in every row with source < 0
 *   dweights[t, k] = sum of dout[t, :] * y[position[t, k], :], 0 for a choice without a row
 * Either may be left out: dy = NULL (then weights and source are not used and may be NULL), or dweights = NULL
 * (then y is not used and may be NULL); not both.
 */
cuttResult cuttExpertCombineBackward(int tokens, int choices, int rows, int width, cuttRowType type, hipStream_t stream,
                                     const int* position, const int* source, const float* weights, const void* y,
                                     long long yStride, const void* dout, long long doutStride, void* dy,
                                     long long dyStride, float* dweights);

/* ---- rows in pages ----------------------------------------------------------
 *
 * A cache of `pages` pages of `pageSize` slots.  Request b owns the pages tables[b, 0], tables[b, 1], ...; its token at
 * position p lives in slot tables[b, p / pageSize] * pageSize + p % pageSize.
 */

/*
 * Takes pages for the new tokens of every request from a list of free ones and names the new tokens' slots.  With
 * owned = ceil(cached / pageSize) and want = ceil((cached + added) / pageSize), both tableWidth at most, request b gets want - owned
 * pages, the requests one after the other from the front of freePages:
 *   tables[b, j]      for owned <= j < want: the next free page, -1 past the list's end; other entries stay
 *   starts[b]         new tokens of the requests before b; starts[requests] = all of them
 *   used[0]           pages wanted from the list; more than freeCount if it did not suffice
 *   slots[i]          for the i-th new token (requests one after the other): its slot as a 64-bit number; -1 if its page is
 *                     absent (a table entry below 0, or beyond the table's width) and for starts[requests] <= i < tokens
 *   positions[i]      its position in its request, -1 for i >= starts[requests].  NULL: not wanted
 *
 * The list itself stays: the caller takes used[0] entries off its front before the next call.  A captured call reads the same
 * buffers at every replay; its caller moves the list up between replays (entries below 0 are no pages and may fill its end).
 *
 *   requests, freeCount, tokens >= 0, pageSize >= 1, tableWidth >= 1
 *   cached, added     [requests]; values below 0 count as 0; sums and positions are 2^31 - 1 at most
 *   tables            [requests, tableWidth], read and written
 */
cuttResult cuttPageTables(int requests, int pageSize, int tableWidth, int freeCount, int tokens, hipStream_t stream,
                          const int* cached, const int* added, const int* freePages, int* tables, int* starts, int* used,
                          long long* slots, int* positions);

/*
 * Rows into pages: for every token t and head h, with s = slots[t],
 *   kCache[s / pageSize, s % pageSize, h, :] = k[t, h, :], the same for v.  Tokens whose slot is not in
 * 0 .. pages * pageSize - 1 are left out.  The others' slots should differ, as cuttPageTables makes them from pages that differ: a slot that two
 * tokens name may end up with elements of either, in k and in v (see above).
 * A token's heads * width * sizeofType bytes are fewer than 2^31.
 *
 *   slots             [tokens], 64-bit
 *   rowStrides[2]     elements from token to token and from head to head of k and v
 *   cacheStrides[3]   elements from page to page, slot to slot and head to head of the caches; any order of the three
 *                     ([pages, pageSize, heads, width], [pages, heads, pageSize, width], ...)
 *                     What is written must not lie on top of itself: each stride of its axes of more than one entry leads past all that the
 *                     smaller ones reach, and the two written tensors share no element (they may interleave)
 *                     k and v share width and strides, and so do their caches; where they do not, each moves in a call of its own
 *   v, vCache         NULL both: only k moves (a buffer of no tokens or of no pages may be NULL by itself)
 * The strides are host arrays, read during the call.
 */
cuttResult cuttPageStore(int tokens, int heads, int width, size_t sizeofType, int pages, int pageSize, hipStream_t stream,
                         const long long* slots, const void* k, const void* v, const long long* rowStrides, void* kCache,
                         void* vCache, const long long* cacheStrides);

/* Rows out of pages: k[t, h, :] = kCache[s / pageSize, s % pageSize, h, :], the same for v; zeros for tokens whose slot is not in
 * 0 .. pages * pageSize - 1.  Arguments as for cuttPageStore. */
cuttResult cuttPageLoad(int tokens, int heads, int width, size_t sizeofType, int pages, int pageSize, hipStream_t stream,
                        const long long* slots, void* k, void* v, const long long* rowStrides, const void* kCache,
                        const void* vCache, const long long* cacheStrides);

#ifdef __cplusplus
}
#endif

#endif /* CUTT_ROWS_H */
