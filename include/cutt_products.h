/*
 * cutt_products.h - products on the rows that cutt_rows.h lays out: rows sorted by expert times their experts' weights, with
 * the gradients, and attention over keys and values in pages.  The reference has no counterpart.
 *
 * Conventions, as for the row operators:
 *   - a row is contiguous; strides are in elements; integers in device buffers are 32-bit; all floating buffers of a call have
 *     its cuttRowType unless said otherwise;
 *   - products of 16-bit types are exact and summed in 32 bits, those of CUTT_F32 are multiplied and summed in 32 bits; results are rounded
 *     once, to nearest even;
 *   - every call only launches kernels on `stream`, on the current device: it allocates nothing, keeps nothing, copies nothing and
 *     does not synchronise, and can be captured into a HIP graph (make the call once before the capture).  The caller orders
 *     work of other streams;
 *   - buffers are aligned to their elements; any such address and any stride will do, multiples of 16 bytes are fastest.  What a
 *     call writes must not overlap what it reads; columns of one buffer (equal largest strides, all of a buffer's other axes within a
 *     column) do not;
 *   - no buffer's contents can make a call touch memory outside the buffers as their sizes, strides and counts describe them;
 *   - the results do not depend on timing: equal inputs give equal bits.
 *
 * All functions return CUTT_SUCCESS, CUTT_INVALID_PARAMETER (null, misaligned or overlapping buffers, sizes out of range;
 * nothing was launched) or CUTT_INTERNAL_ERROR (the HIP runtime refused a launch).
 */
#ifndef CUTT_PRODUCTS_H
#define CUTT_PRODUCTS_H

#include "cutt_rows.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rows grouped by expert ------------------------------------------------
 *
 * Group e has the rows offsets[e] <= r < offsets[e + 1], as cuttExpertSort makes them.  Offsets beyond 0 .. rows count as the nearer of the two, and a
 * group whose end is not above its start has no rows.  (Offsets that descend can make groups share rows: what these and the groups behind them
 * get is then not said.)
 */

/*
 * y[r, :] = x[r, :] * w[e] for every row of every group.  Rows of no group are left as they were.
 *   rows >= 0, 1 <= groups <= CUTT_MAX_EXPERTS, inner >= 1, outer >= 1
 *   offsets           [groups + 1]
 *   x                 [rows, inner] with row stride xStride         y  [rows, outer] with row stride yStride
 *   w                 [groups, inner, outer], or transposed != 0: [groups, outer, inner], whose rows are multiplied instead
 *   wStrides[2]       elements from group to group and from row to row of w; a host array, read during the call
 * The gradient for x is the same product of y's gradient with w, inner and outer exchanged and the other value of transposed.
 */
cuttResult cuttGroupedProduct(int rows, int groups, int inner, int outer, cuttRowType type, int transposed, hipStream_t stream, const int* offsets,
                              const void* x, long long xStride, const void* w, const long long* wStrides, void* y, long long yStride);

/*
 * The gradient for the weights: dw[e, i, j] = sum over the rows r of group e of x[r, i] * dy[r, j]; zeros for a group without rows.
 *   x                 [rows, inner] with row stride xStride         dy  [rows, outer] with row stride dyStride
 *   dw                [groups, inner, outer]
 *   dwStrides[2]      elements from group to group and from row to row of dw: rows must not lie on top of each other
 * For weights that are used transposed, exchange x and dy, inner and outer.  Fastest where all rows of x, and all of dy, span less than 2^30 bytes.
 */
cuttResult cuttGroupedProductWeights(int rows, int groups, int inner, int outer, cuttRowType type, hipStream_t stream, const int* offsets, const void* x,
                                     long long xStride, const void* dy, long long dyStride, void* dw, const long long* dwStrides);

/* ---- attention over pages ---------------------------------------------------- */

#define CUTT_MAX_HEAD_WIDTH 256
#define CUTT_MAX_HEADS 65536

/* Bytes of workspace that cuttAttendPages needs for these sizes (0: none, or arguments out of range).  Fewer queries may need more than many: ask for the sizes of every
 * call, or take the largest of all that may come. */
size_t cuttAttendPagesWorkspace(int queries, int heads, int keyHeads, int width, int pageSize, int tableWidth, int window);

/*
 * Queries of new tokens over the cached keys and values of their requests, which lie in pages as in cutt_rows.h (store the new tokens' own first).  Made for one or a few queries of
 * a request, which follow each other; prompts are right but not fast, as their queries read the keys and values again, a few queries at a time.
 * Query i belongs to request b = owners[i] and has the position p = positions[i].  It sees the tokens at the positions
 *   first .. p,   first = max(0, p - window + 1), or 0 without a window,
 * as far as they have a page in tables[b]: those beyond the table's width or of a page that is absent (an entry not in 0 .. pages - 1) are not seen.
 * Head h uses the keys and values of key head h / (heads / keyHeads).  With s_t = scale * (q[i, h, :] . k[t, :]) over the tokens t that it sees:
 *   logSums[i, h]     log of the sum of exp(s_t)
 *   out[i, h, :]      sum of exp(s_t - logSums[i, h]) * v[t, :]
 * A query that sees nothing (a position below 0, an owner not in 0 .. requests - 1), or whose scores are all -infinity, gets zeros, and -infinity; one with a score of
 * +infinity NaN, and +infinity.  Infinite values that are seen make their element infinite, both signs or NaN make it NaN (so may an infinity whose weight is below 2^-126 of
 * the largest).  Keys and values that are not seen have no part in it, whatever they hold.
 *
 *   queries, requests, pages >= 0, keyHeads >= 1, heads <= CUTT_MAX_HEADS a multiple of it, queries * heads < 2^31
 *   1 <= width <= CUTT_MAX_HEAD_WIDTH, pageSize, tableWidth >= 1, scale finite
 *   window            tokens that a query sees at most, itself among them; 0: all
 *   tables            [requests, tableWidth]
 *   owners            [queries], or NULL: query i belongs to request i
 *   positions         [queries], as cuttPageTables gives them
 *   q                 [queries, heads, width], qStrides[2] from query to query and from head to head
 *   kCache, vCache    cacheStrides[3] from page to page, slot to slot and head to head, of both
 *   out               [queries, heads, width], outStrides[2]
 *   logSums           [queries, heads] in 32-bit floating point, or NULL: not wanted.  (Results over two caches can be joined by them.)
 *   workspace         cuttAttendPagesWorkspace bytes, aligned to 4; its contents need no preparation and mean nothing afterwards.  Calls that may overlap
 *                     on the GPU need one each
 * Scores, their exponentials and the sums are in 32 bits, but that the 16-bit types multiply values with exponentials in two parts of the type: to within 2^-16 of each
 * (CUTT_BF16), or 2^-22 of each and 2^-40 of the largest (CUTT_F16).  The sums are divided at the end: values have to stay below 2^120 over the number of tokens.  The strides are host
 * arrays, read during the call.
 */
cuttResult cuttAttendPages(int queries, int requests, int heads, int keyHeads, int width, cuttRowType type, int pages, int pageSize, int tableWidth,
                           int window, float scale, hipStream_t stream, const int* tables, const int* owners, const int* positions, const void* q,
                           const long long* qStrides, const void* kCache, const void* vCache, const long long* cacheStrides, void* out,
                           const long long* outStrides, float* logSums, void* workspace, size_t workspaceBytes);

#ifdef __cplusplus
}
#endif

#endif /* CUTT_PRODUCTS_H */
