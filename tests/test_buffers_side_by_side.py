"""Buffers of several axes in the columns of one: what shares no byte is accepted where the rows' largest strides are equal, and what is accepted shares none.  On a stand-in for
the kernels' layer that launches nothing."""
import itertools

import numpy as np

from test_products_api import ATTEND, B, BAD, D, F, OK, PRODUCT, WEIGHTS, stub, stub_lib  # noqa: F401  (fixtures)


def bytes_of(at, extents, strides, width, size=2):
    """The bytes of a strided buffer at an address, its strides in elements."""
    starts = [at + size * sum(i * s for i, s in zip(index, strides)) for index in itertools.product(*map(range, extents))]
    return {a + i for a in starts for i in range(width * size)}


def test_queries_and_results_in_the_rows_of_one_buffer(stub):  # noqa: F811
    """4 queries of 8 heads of 16: 128 elements in rows of 288, the results beside them."""
    for apart in (0, 2, 126, 127, 128, 129, 144, 160, 161, 180, 287, 288, 288 + 128, 288 + 127, 4 * 288):
        for out in (F + 2 * apart, F - 2 * apart):
            call = {**ATTEND, "q": F, "qs": (288, 16), "out": out, "os": (288, 16)}
            shared = bytes_of(F, (4, 8), (288, 16), 16) & bytes_of(out, (4, 8), (288, 16), 16)
            assert stub.cuttAttendPages(*call.values()) == (BAD if shared else OK), (apart, out - F)
            assert stub.launches() == (0 if shared else 1)


def test_results_beside_keys_in_pages(stub):  # noqa: F811
    """A page's 16 slots of 2 heads are 512 elements, in pages of 1024; results of a query, 128 elements, in the other half."""
    for at, answer in ((512, OK), (511, BAD), (1024 - 128, OK), (1024 - 127, BAD), (640, OK), (0, BAD), (1536, OK)):
        assert stub.cuttAttendPages(*{**ATTEND, "cs": (1024, 32, 16), "os": (1024, 16), "out": D + 2 * at}.values()) == answer, at


def test_weights_beside_rows(stub):  # noqa: F811
    """Groups of 16 x 24 weights every 1024 elements, and rows of results behind each; gradients the same."""
    for at, answer in ((384, OK), (383, BAD), (1000, OK), (1001, BAD)):
        assert stub.cuttGroupedProduct(*{**PRODUCT, "w": D, "ws": (1024, 24), "y": D + 2 * at, "ys": 1024}.values()) == answer, at
        assert stub.cuttGroupedProductWeights(*{**WEIGHTS, "dw": D, "ws": (1024, 24), "dy": D + 2 * at, "ds": 1024}.values()) == answer, at


def test_what_is_accepted_shares_no_byte(stub):  # noqa: F811
    rng = np.random.default_rng(3)
    accepted = 0
    for _ in range(4000):
        queries, heads, width = (int(rng.integers(1, n)) for n in (5, 4, 6))
        inner = width + int(rng.integers(0, 3))
        outer = [int(rng.integers(0, 40)), inner * heads + int(rng.integers(0, 30))]
        strides = [(o, inner) if rng.integers(2) else (inner, o) for o in outer]
        if rng.integers(2):
            strides[0] = strides[1]
        at = int(rng.integers(-90, 90)) * 2
        call = {**ATTEND, "queries": queries, "heads": heads, "key_heads": 1, "width": width, "q": B + at, "qs": strides[0], "out": B, "os": strides[1],
                "positions": F}
        code = stub.cuttAttendPages(*call.values())
        stub.launches()
        if code == OK:
            accepted += 1
            assert not bytes_of(B + at, (queries, heads), strides[0], width) & bytes_of(B, (queries, heads), strides[1], width), call
    assert accepted > 400
