/* Calls every row operator with random arguments, extremes among them, on a stand-in for the kernels' layer: what is refused must not reach it, and
 * what reaches it must lie inside buffers that the arguments describe.  Built with sanitizers by tests/test_rows_api.py; no GPU. */
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "cutt_rows.h"
#include "row_layer.h"

typedef unsigned __int128 Wide;
static int gCalls = 0;
static void need(bool ok, const char* what) {
  if (!ok) {
    std::printf("wrong: %s\n", what);
    std::exit(1);
  }
}
static void rows(const void* p, uint64_t count, uint64_t stride, uint64_t width, uint64_t size, const char* what) {
  if (!count || !width) return;
  need(p && (uintptr_t)p % size == 0, what);
  need(((Wide)(count - 1) * (count > 1 ? stride : 0) + width) * size <= (Wide)1 << 62, what);
}

extern "C" size_t cuttHipSortWorkspace(uint32_t n, uint32_t experts) { return n > 4096 ? (size_t)experts * 400 : 0; }
extern "C" int cuttHipExpertSort(const cuttHipSortArgs* a, void*) {
  gCalls++;
  need(a->n <= INT_MAX && a->experts >= 1 && a->experts <= CUTT_MAX_EXPERTS && a->align >= 1, "sort sizes");
  need((uint64_t)a->n + (uint64_t)(a->n < a->experts ? a->n : a->experts) * (a->align - 1) <= INT_MAX, "sort rows");
  need((a->idBytes == 4 || a->idBytes == 8) && a->counts && a->offsets, "sort buffers");
  need(!a->n || (a->ids && a->position && (uintptr_t)a->ids % a->idBytes == 0), "sort choices");
  need(!a->rows || a->source, "sort source");
  need(!cuttHipSortWorkspace(a->n, a->experts) || a->workspace, "sort workspace");
  return 0;
}
static void expertArgs(const cuttHipExpertArgs* a) {
  need((uint64_t)a->tokens * a->choices <= INT_MAX && a->choices >= 1 && a->width >= 1 && a->rows <= INT_MAX, "sizes");
  need(!a->tokens || a->position, "position");
}
extern "C" int cuttHipDispatch(const cuttHipExpertArgs* a, uint32_t size, const void* x, uint64_t xs, void* y, uint64_t ys, void*) {
  gCalls++;
  expertArgs(a);
  need(a->rows && a->source, "dispatch source");
  rows(x, a->tokens, xs, a->width, size, "dispatch x");
  rows(y, a->rows, ys, a->width, size, "dispatch y");
  need(a->rows < 2 || ys >= a->width, "dispatch y stride");
  return 0;
}
extern "C" int cuttHipCombine(const cuttHipExpertArgs* a, int type, const void* y, uint64_t ys, void* out, uint64_t os, void*) {
  gCalls++;
  expertArgs(a);
  need(a->tokens && type >= 0 && type <= 2, "combine");
  const uint64_t size = type == CUTT_ROW_F32 ? 4 : 2;
  rows(y, a->rows, ys, a->width, size, "combine y");
  rows(out, a->tokens, os, a->width, size, "combine out");
  need(a->tokens < 2 || os >= a->width, "combine out stride");
  return 0;
}
extern "C" int cuttHipCombineBackward(const cuttHipExpertArgs* a, int type, const void* y, uint64_t ys, const void* dout, uint64_t ds, void* dy, uint64_t dys,
                                      float* dw, void*) {
  gCalls++;
  expertArgs(a);
  need(dy || dw, "nothing to do reached the layer");
  need(!dy || (a->rows && a->source && (!a->tokens || a->weights)), "backward dy");
  need(!dw || a->tokens, "backward dw");
  need(dy || (!a->weights && !a->source), "buffers that were not checked");
  need(dw || !y, "rows that were not checked");
  const uint64_t size = type == CUTT_ROW_F32 ? 4 : 2;
  rows(dout, a->tokens, ds, a->width, size, "backward dout");
  if (dy) rows(dy, a->rows, dys, a->width, size, "backward dy");
  if (dw) rows(y, a->rows, ys, a->width, size, "backward y");
  return 0;
}
extern "C" int cuttHipPageTables(const cuttHipTablesArgs* a, void*) {
  gCalls++;
  need(a->starts && a->used && a->pageSize >= 1 && a->tableWidth >= 1, "tables");
  need(!a->requests || (a->cached && a->added && a->tables), "tables requests");
  need(!a->tokens || a->slots, "tables slots");
  need(!a->freeCount || a->freePages, "tables free");
  return 0;
}
extern "C" int cuttHipPageMove(const cuttHipPageArgs* a, void*) {
  gCalls++;
  need(a->tokens && a->heads && a->width && a->slots && a->rows[0], "pages");
  need((uint64_t)a->heads * a->width * a->elemSize <= INT_MAX, "pages token");
  need(!a->pages || a->cache[0], "pages cache");
  need((a->rows[1] != nullptr) == (a->cache[1] != nullptr), "pages second tensor");
  const Wide row = (Wide)(a->tokens - 1) * a->tokenStride + (Wide)(a->heads - 1) * a->headStride + a->width;
  need(row * a->elemSize <= (Wide)1 << 62, "pages rows");
  if (a->pages) {
    const Wide cache = (Wide)(a->pages - 1) * a->pageStride + (Wide)(a->pageSize - 1) * a->slotStride + (Wide)(a->heads - 1) * a->cacheHeadStride + a->width;
    need(cache * a->elemSize <= (Wide)1 << 62, "pages cells");
  }
  return 0;
}

int main() {
  std::mt19937_64 rng(1);
  auto pick = [&](std::initializer_list<long long> v) { return *(v.begin() + rng() % v.size()); };
  auto size = [&] { return (int)pick({1, 2, 3, 4, 7, 8, 16, 100, 1000, 5, 64, 0, -1, 1 << 20, INT_MAX, INT_MIN}); };
  auto small = [&] { return (int)pick({1, 2, 3, 4, 8, 16, 100, 0, 5, 64, 1 << 20}); };
  auto ptr = [&] { return (char*)(uintptr_t)(rng() % 24 == 0 ? 0 : 0x100000000000ull * (1 + rng() % 60) + (uint64_t)pick({0, 0, 0, 0, 4, 8, 2, 64, 1 << 20})); };
  auto stride = [&] { return pick({0, 1, 2, 16, 64, 100, 128, 4096, 1 << 20, 1ll << 40, LLONG_MAX, -1, LLONG_MIN}); };
  int ok = 0, before;
  const int rounds = 400000;
  for (int i = 0; i < rounds; i++) {
    before = gCalls;
    cuttResult r = CUTT_SUCCESS;
    const int t = rng() % 2 ? small() : size(), k = rng() % 2 ? small() : size(), n = rng() % 2 ? small() : size(), w = rng() % 2 ? small() : size();
    const size_t es = (size_t)pick({1, 2, 4, 8, 2, 4, 3, 0});
    const cuttRowType type = (cuttRowType)pick({0, 1, 2, 0, 1, 2, 3});
    switch (rng() % 8) {
      case 0: {
        const int first = size(), align = small();
        r = cuttExpertSort(t, k, first, n, align, w, es, nullptr, ptr(), (int*)ptr(), (int*)ptr(), (int*)ptr(), (int*)ptr(), ptr(), (size_t)pick({0, 1 << 20}));
        break;
      }
      case 1: r = cuttExpertDispatch(t, k, n, w, es, nullptr, (int*)ptr(), (int*)ptr(), ptr(), stride(), ptr(), stride()); break;
      case 2: r = cuttExpertDispatchBackward(t, k, n, w, type, nullptr, (int*)ptr(), ptr(), stride(), ptr(), stride()); break;
      case 3: r = cuttExpertCombine(t, k, n, w, type, nullptr, (int*)ptr(), (float*)ptr(), ptr(), stride(), ptr(), stride()); break;
      case 4:
        r = cuttExpertCombineBackward(t, k, n, w, type, nullptr, (int*)ptr(), (int*)ptr(), (float*)ptr(), ptr(), stride(), ptr(), stride(), ptr(), stride(),
                                      (float*)ptr());
        break;
      case 5: r = cuttPageTables(t, k, n, w, small(), nullptr, (int*)ptr(), (int*)ptr(), (int*)ptr(), (int*)ptr(), (int*)ptr(), (int*)ptr(), (long long*)ptr(), (int*)ptr()); break;
      default: {
        const long long rs[2] = {stride(), stride()}, cs[3] = {stride(), stride(), stride()};
        char* const v = rng() % 2 ? ptr() : nullptr;
        char* const vc = rng() % 8 ? (v ? ptr() : nullptr) : ptr();
        const long long* const rp = rng() % 30 ? rs : nullptr;
        if (rng() % 2) r = cuttPageStore(t, k, w, es, n, small(), nullptr, (long long*)ptr(), ptr(), v, rp, ptr(), vc, cs);
        else r = cuttPageLoad(t, k, w, es, n, small(), nullptr, (long long*)ptr(), ptr(), v, rp, ptr(), vc, cs);
      }
    }
    if (r != CUTT_SUCCESS) {
      need(r == CUTT_INVALID_PARAMETER, "a refusal's code");
      need(gCalls == before, "a refused call reached the layer");
    } else {
      ok++;
    }
  }
  need(gCalls > rounds / 100, "hardly any call was accepted");
  std::printf("rows api ok, %d of %d accepted, %d launched\n", ok, rounds, gCalls);
  return 0;
}
