"""Which calls the row operators accept, on a stand-in for the kernels' layer: nothing is launched, so the addresses can be made up."""
import ctypes
import itertools
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, BAD = 0, 2
A, B, C, D, E, F, G = (0x10000000 * i for i in range(1, 8))


@pytest.fixture(scope="module")
def stub_lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("stub") / "librows.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wall", "-Wextra", "-I" + os.path.join(ROOT, "cutt_amd", "csrc"),
                           os.path.join(ROOT, "tests", "rows_layer_stub.cpp"), os.path.join(ROOT, "cutt_amd", "csrc", "rows_api.cpp"), "-o", out])
    return ctypes.CDLL(out)


@pytest.fixture
def rows(cutt, stub_lib, monkeypatch):
    """The binding on the stand-in; `rows.launches()` counts what got through since the last look."""
    for name in dir(cutt):
        if name.startswith(("cuttExpert", "cuttPage")):
            f, real = getattr(stub_lib, name), getattr(cutt.lib(), name)
            f.argtypes, f.restype = real.argtypes, real.restype
    monkeypatch.setattr(cutt.api, "_lib", stub_lib)
    count = ctypes.c_int.in_dll(stub_lib, "stubLaunches")
    count.value = 0

    def launches():
        n, count.value = count.value, 0
        return n

    monkeypatch.setattr(cutt, "launches", launches, raising=False)
    return cutt


def bytes_of(at, rows, pitch, width):
    return {at + r * pitch + i for r in range(rows) for i in range(width)}


# ---- rows side by side -----------------------------------------------------------
def test_rows_side_by_side_from_one_row_on(rows):
    """Input and output as columns of one buffer, for every pair of row counts: refused where a byte is shared, and only there."""
    for tokens, count in itertools.product((1, 2, 3), (1, 2, 5)):
        for at in range(-104, 320, 6):  # 16 elements of 2 bytes, 48 from row to row
            shared = bytes_of(D + at, tokens, 96, 32) & bytes_of(D, count, 96, 32)
            want = BAD if shared else OK
            assert rows.cuttExpertDispatch(tokens, 2, count, 16, 2, 0, A, B, D + at, 48, D, 48) == want, (tokens, count, at)
            assert rows.cuttExpertCombine(count, 2, tokens, 16, 2, 0, A, B, D + at, 48, D, 48) == want, (tokens, count, at)
            assert rows.launches() == (0 if shared else 2)


def test_one_row_for_all_beside_the_rows(rows):
    """A row that is read for every token (stride 0) in the columns beside the output; 16 columns of 48."""
    for at in range(0, 192, 4):
        shared = bytes_of(D + at, 1, 0, 32) & bytes_of(D, 8, 96, 32)
        assert rows.cuttExpertDispatch(5, 2, 8, 16, 2, 0, A, B, D + at, 0, D, 48) == (BAD if shared else OK), at


def test_rows_of_two_pitches(rows):
    """What is accepted shares no byte, whatever the two pitches are; a pitch that divides the other is told apart exactly."""
    for xs, ys in itertools.product((0, 16, 32, 48, 64, 96), repeat=2):
        if ys < 16:
            continue
        for tokens, count, at in itertools.product((1, 4), (1, 3), range(-400, 400, 16)):
            shared = bytes_of(D + at, tokens, 2 * xs, 32) & bytes_of(D, count, 2 * ys, 32)
            code = rows.cuttExpertDispatch(tokens, 2, count, 16, 2, 0, A, B, D + at, xs, D, ys)
            assert code == BAD or not shared, (xs, ys, tokens, count, at)
            if tokens == 1 or count == 1 or xs == ys or xs == 0:
                assert code == (BAD if shared else OK), (xs, ys, tokens, count, at)


def test_values_in_the_columns_beside_the_rows(rows):
    """Contiguous values inside a gap between rows are apart from them, values that reach the next row are not."""
    assert rows.cuttExpertDispatch(4, 1, 8, 16, 2, 0, D + 32, B, C, 16, D, 48) == OK  # 16 bytes of positions in a gap of 64
    assert rows.cuttExpertDispatch(4, 1, 8, 16, 2, 0, D + 80, B, C, 16, D, 48) == OK
    assert rows.cuttExpertDispatch(4, 1, 8, 16, 2, 0, D + 84, B, C, 16, D, 48) == BAD
    assert rows.cuttExpertDispatch(40, 1, 8, 16, 2, 0, D + 32, B, C, 16, D, 48) == BAD  # longer than the gap


# ---- gradients of combine, one of them left out ---------------------------------------
BACKWARD = dict(tokens=4, choices=2, rows=8, width=16, type=2, stream=0, position=A, source=B, weights=C, y=D, ys=16, dout=E, douts=16, dy=F, dys=16,
                dweights=G)


def test_buffers_of_the_gradient_that_is_left_out(rows):
    """Without dy neither source nor weights are used, without dweights y is not: null, misaligned or on top of another one, whatever the number of rows."""
    for count in (0, 8):
        for weights in (0, C + 1, G, F):
            call = {**BACKWARD, "rows": count, "dy": 0, "source": weights, "weights": weights, "dys": -3}
            assert rows.cuttExpertCombineBackward(*call.values()) == OK, (count, weights)
            assert rows.launches() == 1
        assert rows.cuttExpertCombineBackward(*{**BACKWARD, "rows": count, "dweights": 0, "y": F, "ys": -1}.values()) == OK
        assert rows.launches() == (1 if count else 0)
    for count, left in itertools.product((0, 8), ({}, {"source": 0}, {"weights": 0}, {"weights": C + 2})):
        assert rows.cuttExpertCombineBackward(*{**BACKWARD, "rows": count, **left}.values()) == (BAD if left and count else OK)
    assert rows.cuttExpertCombineBackward(*{**BACKWARD, "dy": 0, "dweights": 0}.values()) == BAD


def test_gradients_of_no_tokens(rows):
    none = {**BACKWARD, "tokens": 0, "position": 0, "weights": 0, "dout": 0}
    assert rows.cuttExpertCombineBackward(*{**none, "dweights": 0, "y": 0}.values()) == OK and rows.launches() == 1  # empty rows to clear
    assert rows.cuttExpertCombineBackward(*{**none, "dy": 0, "source": 0}.values()) == OK and rows.launches() == 0


# ---- rows in pages -----------------------------------------------------------------
PAGES = dict(tokens=4, heads=2, width=16, size=2, pages=4, page=16, stream=0, slots=A, k=B, v=C, rows=(32, 16), kc=D, vc=E, cache=(512, 32, 16))


def pages_field(stub_lib, name):
    """A field of what the layer was last asked to move."""
    class Args(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_uint32) for n in ("tokens", "heads", "width", "elemSize", "pages", "pageSize")] + [("slots", ctypes.c_void_p)] +
                    [(n, ctypes.c_void_p * 2) for n in ("rows", "cache")] +
                    [(n, ctypes.c_uint64) for n in ("tokenStride", "headStride", "pageStride", "slotStride", "cacheHeadStride")] + [("load", ctypes.c_int)])
    return getattr(Args.in_dll(stub_lib, "stubPages"), name)


def test_empty_buffers_may_be_null(rows, stub_lib):
    """Keys and values of no tokens, or a cache of no pages: null without a say in whether values move too."""
    for call in (rows.cuttPageStore, rows.cuttPageLoad):
        for null in ({"k": 0, "v": 0}, {"v": 0}, {"k": 0, "v": 0, "slots": 0}, {"k": 0, "v": 0, "vc": 0}):
            assert call(*{**PAGES, "tokens": 0, **null}.values()) == OK, null
        assert call(*{**PAGES, "tokens": 0, "k": 0, "v": 0, "vc": E + 1}.values()) == BAD  # (what has entries is checked)
        assert rows.launches() == 0
        for null in ({"kc": 0, "vc": 0}, {"kc": 0}, {"vc": 0}):
            assert call(*{**PAGES, "pages": 0, **null}.values()) == OK, null
            assert rows.launches() == (1 if call is rows.cuttPageLoad else 0)
            if call is rows.cuttPageLoad:  # zeros for keys and values
                assert list(pages_field(stub_lib, "rows")) == [B, C] and pages_field(stub_lib, "pages") == 0
        for null in ({"k": 0}, {"v": 0}, {"vc": 0}, {"kc": 0}):
            assert call(*{**PAGES, **null}.values()) == BAD, null


def cells(at, extents, strides, width, size):
    """Every byte of every row, as often as it is named."""
    return [at + (sum(i * s for i, s in zip(index, strides)) + w) * size + b for index in itertools.product(*map(range, extents)) for w in range(width)
            for b in range(size)]


def test_page_moves_write_every_element_once(rows):
    """Strides of the written side: what is accepted names no byte twice, and strides in any order that nest are accepted."""
    nested = 0
    for heads, tokens, pages, page in ((2, 4, 2, 3), (3, 2, 3, 1), (1, 3, 2, 2), (2, 1, 1, 4)):
        for strides in itertools.product((0, 2, 3, 4, 6, 8, 12), repeat=3):
            args = (heads, 3, 2, pages, page, 0, A)
            twice = len(cells(0, (pages, page, heads), strides, 3, 2)) != len(set(cells(0, (pages, page, heads), strides, 3, 2)))
            code = rows.cuttPageStore(tokens, *args, B, 0, (24, 3), D, 0, strides)
            assert code == BAD if twice else True, (heads, pages, page, strides)
            reach, fits = 3, True
            for stride, extent in sorted((s, e) for s, e in zip(strides, (pages, page, heads)) if e > 1):
                fits, reach = fits and stride >= reach, reach + (extent - 1) * stride
            assert code == (OK if fits else BAD), (heads, pages, page, strides)
            nested += fits
            two = strides[:2]
            code = rows.cuttPageLoad(tokens, *args, B, 0, two, D, 0, (0, 0, 0))
            named = cells(0, (tokens, heads), two, 3, 2)
            assert code == BAD if len(named) != len(set(named)) else True, (tokens, heads, two)
    assert nested > 50


def test_page_moves_write_two_tensors(rows):
    """Keys and values that are written: refused exactly where they share a byte, interleaved ones included."""
    layouts = [((2, 3, 2), (48, 16, 8)), ((2, 3, 2), (48, 8, 24)), ((3, 2, 2), (8, 24, 48)), ((2, 1, 3), (40, 0, 10)), ((1, 1, 1), (0, 0, 0)), ((2, 2, 2), (100, 37, 9))]
    for (pages, page, heads), strides in layouts:
        first = set(cells(0, (pages, page, heads), strides, 4, 2))
        for apart in range(-340, 340, 2):
            shared = any(b + apart in first for b in first)
            code = rows.cuttPageStore(5, heads, 4, 2, pages, page, 0, A, B, C, (32, 4), D, D + apart, strides)
            assert code == (BAD if shared else OK), (strides, apart)
            two = (strides[0], strides[2])
            rows_named = set(cells(0, (pages, heads), two, 4, 2))
            shared = any(b + apart in rows_named for b in rows_named)
            code = rows.cuttPageLoad(pages, heads, 4, 2, 7, 3, 0, A, D, D + apart, two, B, C, (64, 16, 8))
            assert code == (BAD if shared else OK), (two, apart)
    assert rows.cuttPageLoad(*{**PAGES, "v": B}.values()) == BAD and rows.cuttPageStore(*{**PAGES, "vc": D}.values()) == BAD
    # what is only read may be the same for both
    assert rows.cuttPageStore(*{**PAGES, "v": B}.values()) == OK and rows.cuttPageLoad(*{**PAGES, "vc": D}.values()) == OK
    # keys and values beside each other in every slot, far apart and beyond 32 bits
    for far in (1 << 20, 1 << 33, 1 << 50):
        wide = {**PAGES, "cache": (far * 64, far, 32)}
        assert rows.cuttPageStore(*{**wide, "kc": D, "vc": D + 32}.values()) == OK
        assert rows.cuttPageStore(*{**wide, "kc": D, "vc": D + 2 * far}.values()) == BAD
        assert rows.cuttPageStore(*{**wide, "kc": D, "vc": D + 2 * far * 16}.values()) == OK  # behind the last slot of a page


def test_order_of_the_lanes(rows, stub_lib):
    """Lanes go to the next token or to the next head, whichever comes closer on the written side; behind a page's only slot that is the next page."""
    def inner(call, **change):
        assert call(*{**PAGES, **change}.values()) == OK, change
        return stub_lib.stubTokensInner()

    by_slot, by_head, pages_by_slot, pages_by_head = (32, 16), (16, 64), (512, 32, 16), (512, 16, 256)
    for other in (by_slot, by_head):
        assert inner(rows.cuttPageStore, rows=other, cache=pages_by_slot) == 0 and inner(rows.cuttPageStore, rows=other, cache=pages_by_head) == 1
        assert inner(rows.cuttPageStore, rows=other, page=1, cache=(32, -5, 16)) == 0 and inner(rows.cuttPageStore, rows=other, page=1, cache=(16, 99, 64)) == 1
    for other, page in ((pages_by_slot, 16), (pages_by_head, 16), ((32, 32, 16), 1)):
        assert inner(rows.cuttPageLoad, rows=by_slot, cache=other, page=page) == 0 and inner(rows.cuttPageLoad, rows=by_head, cache=other, page=page) == 1


# ---- the binding ---------------------------------------------------------------------
def test_sizes_beyond_32_bits_are_refused(rows):
    """A size is refused whatever its lower 32 bits say."""
    calls = [(rows.cuttExpertSort, (4, 2, 0, 8, 1, 8, 4, 0, A, B, C, D, E), (0, 1, 2, 3, 4, 5, 6)), (rows.cuttExpertDispatch, (4, 2, 8, 16, 2, 0, A, B, C, 16, D, 16), range(5)),
             (rows.cuttExpertDispatchBackward, (4, 2, 8, 16, 2, 0, A, C, 16, D, 16), range(5)),
             (rows.cuttExpertCombine, (4, 2, 8, 16, 2, 0, A, B, C, 16, D, 16), range(5)), (rows.cuttExpertCombineBackward, tuple(BACKWARD.values()), range(5)),
             (rows.cuttPageTables, (4, 16, 8, 8, 32, 0, A, B, C, D, E, F, G, 0), range(5)), (rows.cuttPageStore, tuple(PAGES.values()), range(6)),
             (rows.cuttPageLoad, tuple(PAGES.values()), range(6))]
    for call, args, sizes in calls:
        assert call(*args) == OK and rows.launches() == 1, call
        for i in sizes:
            for more in (2 ** 32, -2 ** 32, 2 ** 63, 2 ** 64, 3 * 2 ** 64):
                assert call(*args[:i], args[i] + more, *args[i + 1:]) == BAD, (call, i, more)
    assert rows.launches() == 0
    assert rows.cuttExpertSort(4, 2, -2 ** 31, 8, 1, 8, 4, 0, A, B, C, D, E) == OK and rows.cuttExpertSort(4, 2, 2 ** 31 - 1, 8, 1, 8, 4, 0, A, B, C, D, E) == OK
    for i in range(4):
        sizes = [3, 2, 8, 16]
        assert rows.cuttExpertRows(*sizes) == 6 + 6 * 15
        sizes[i] += 2 ** 32
        assert rows.cuttExpertRows(*sizes) == -1
    assert rows.cuttExpertSortWorkspace(2 ** 13 + 2 ** 32, 1, 8) == 0 and rows.cuttExpertSortWorkspace(2 ** 13, 1, 8) > 0
