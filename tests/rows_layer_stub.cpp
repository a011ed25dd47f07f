/* A stand-in for the row operators' kernel layer that launches nothing and keeps what it was last asked for: which calls rows_api.cpp accepts can
 * then be seen with made-up addresses on any machine.  Built and loaded by tests/test_rows_accepted.py. */
#include "row_layer.h"

extern "C" {
int stubLaunches = 0;
cuttHipExpertArgs stubRows;
cuttHipPageArgs stubPages;

size_t cuttHipSortWorkspace(uint32_t n, uint32_t experts) { return n > 4096 ? (size_t)experts * 400 : 0; }
int cuttHipExpertSort(const cuttHipSortArgs*, void*) { return stubLaunches++, 0; }
int cuttHipDispatch(const cuttHipExpertArgs* a, uint32_t, const void*, uint64_t, void*, uint64_t, void*) { return stubRows = *a, stubLaunches++, 0; }
int cuttHipCombine(const cuttHipExpertArgs* a, int, const void*, uint64_t, void*, uint64_t, void*) { return stubRows = *a, stubLaunches++, 0; }
int cuttHipCombineBackward(const cuttHipExpertArgs* a, int, const void*, uint64_t, const void*, uint64_t, void*, uint64_t, float*, void*) {
  return stubRows = *a, stubLaunches++, 0;
}
int cuttHipPageTables(const cuttHipTablesArgs*, void*) { return stubLaunches++, 0; }
int cuttHipPageMove(const cuttHipPageArgs* a, void*) { return stubPages = *a, stubLaunches++, 0; }
int stubTokensInner() { return cuttHipTokensInner(&stubPages); }
}
