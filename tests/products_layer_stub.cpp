/* A stand-in for the products' kernel layer that launches nothing and keeps what it was last asked for: which calls products_api.cpp accepts, and what
 * it passes on, can then be seen with made-up addresses on any machine.  Built and loaded by tests/test_products_api.py. */
#include "product_layer.h"

extern "C" {
int stubLaunches = 0, stubResult = 0;
unsigned long long stubSpace = 0;
cuttHipProductArgs stubProduct;
cuttHipAttendArgs stubAttend;

int cuttHipGroupedProduct(const cuttHipProductArgs* a, int, int, void*) { return stubProduct = *a, stubLaunches++, stubResult; }
int cuttHipGroupedWeights(const cuttHipProductArgs* a, int, void*) { return stubProduct = *a, stubLaunches++, stubResult; }
size_t cuttHipAttendWorkspace(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return (size_t)stubSpace; }
int cuttHipAttend(const cuttHipAttendArgs* a, int, void*) { return stubAttend = *a, stubLaunches++, stubResult; }
}
