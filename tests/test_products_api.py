"""The products' boundary without a GPU: exported under their declared names, refusals before any device access, and, on a stand-in for
the kernels' layer that launches nothing, what is accepted and passed on.  Also the oracle of the GPU tests against hand-made values."""
import ctypes
import itertools
import os
import re
import subprocess

import numpy as np
import pytest

import product_oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")
OK, BAD, FAILED = 0, 2, 4
# Addresses are compared and checked for alignment, never read, on the paths taken here.
A, B, C, D, E, F, G, H, I = (0x10000000 * i for i in range(1, 10))


def test_every_declared_function_is_exported_and_bound(cutt):
    text = re.sub(r"/\*.*?\*/", " ", open(os.path.join(INCLUDE, "cutt_products.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(cutt[A-Z]\w*)\s*\(", text))
    assert len(names) == 4
    lib = ctypes.CDLL(cutt.lib_path())
    for n in names:
        assert hasattr(lib, n) and callable(getattr(cutt, n)), n
    assert cutt.CUTT_MAX_HEADS == 65536 and re.search(r"CUTT_MAX_HEADS\s+65536", text)
    assert cutt.CUTT_MAX_HEAD_WIDTH == 256 and re.search(r"CUTT_MAX_HEAD_WIDTH\s+256", text)


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "caller.c"
    src.write_text('#include "cutt_products.h"\n'
                   "int main(void) { return cuttAttendPagesWorkspace(1, 3, 2, 64, 16, 4, 0) == 0 && cuttGroupedProduct(0, 0, 1, 1, CUTT_F32, 0, 0, 0, 0, 0, 0, 0, "
                   "0, 0) == CUTT_INVALID_PARAMETER ? 0 : 1; }\n")
    exe = str(tmp_path / "caller")
    libdir = os.path.join(ROOT, "cutt_amd")
    subprocess.check_call(["gcc", "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror", "-I", INCLUDE, str(src), "-o", exe, "-L", libdir, "-lcutt",
                           "-Wl,-rpath," + libdir, "-Wl,-rpath-link,/opt/rocm/lib"])
    assert subprocess.run([exe], timeout=120).returncode == 0


PRODUCT = dict(rows=32, groups=4, inner=16, outer=24, type=2, transposed=0, stream=0, offsets=A, x=B, xs=16, w=C, ws=(384, 24), y=D, ys=24)
WEIGHTS = dict(rows=32, groups=4, inner=16, outer=24, type=2, stream=0, offsets=A, x=B, xs=16, dy=C, ds=24, dw=D, ws=(384, 24))
ATTEND = dict(queries=4, requests=4, heads=8, key_heads=2, width=16, type=2, pages=6, page=16, table=8, window=0, scale=0.25, stream=0, tables=A, owners=0,
              positions=B, q=C, qs=(128, 16), k=D, v=E, cs=(512, 32, 16), out=F, os=(128, 16), logs=G, work=H, space=1 << 30)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(groups=0), dict(groups=1025), dict(inner=0), dict(outer=0), dict(type=3), dict(type=-1), dict(offsets=0),
                                    dict(offsets=A + 2), dict(x=0), dict(x=B + 1), dict(xs=-1), dict(w=0), dict(w=C + 1), dict(ws=None), dict(ws=(-1, 24)),
                                    dict(ws=(384, -24)), dict(y=0), dict(y=D + 1), dict(ys=23), dict(ys=-24), dict(y=B), dict(y=C + 3070), dict(y=A), dict(ys=2 ** 62),
                                    dict(xs=2 ** 62), dict(ws=(2 ** 62, 24)), dict(rows=2 ** 31), dict(outer=2 ** 32 + 24)])
def test_product_refuses(cutt, change):
    assert cutt.cuttGroupedProduct(*{**PRODUCT, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(rows=-1), dict(groups=0), dict(groups=1025), dict(inner=0), dict(outer=0), dict(type=3), dict(offsets=0), dict(offsets=A + 1),
                                    dict(x=0), dict(xs=-1), dict(dy=0), dict(dy=C + 1), dict(ds=-1), dict(dw=0), dict(dw=D + 1), dict(ws=None), dict(ws=(384, 23)),
                                    dict(ws=(383, 24)), dict(ws=(0, 24)), dict(ws=(-384, 24)), dict(dw=B), dict(dw=C), dict(dw=A), dict(ws=(2 ** 62, 24))])
def test_weights_refuse(cutt, change):
    assert cutt.cuttGroupedProductWeights(*{**WEIGHTS, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(queries=-1), dict(requests=-1), dict(heads=0), dict(heads=7), dict(key_heads=0), dict(key_heads=3), dict(width=0), dict(width=257),
                                    dict(type=3), dict(pages=-1), dict(page=0), dict(table=0), dict(window=-1), dict(scale=float("inf")), dict(scale=float("nan")),
                                    dict(tables=0), dict(tables=A + 2), dict(owners=I + 1), dict(positions=0), dict(positions=B + 2), dict(q=0), dict(q=C + 1), dict(qs=None),
                                    dict(qs=(-128, 16)), dict(k=0), dict(v=0), dict(v=E + 1), dict(cs=None), dict(cs=(512, -32, 16)), dict(out=0), dict(out=F + 1),
                                    dict(os=None), dict(os=(128, 15)), dict(os=(127, 16)), dict(logs=G + 2), dict(out=C), dict(out=D + 64), dict(out=E), dict(logs=A),
                                    dict(logs=F), dict(logs=B), dict(out=A), dict(owners=F), dict(queries=2 ** 30), dict(cs=(2 ** 62, 32, 16)),
                                    dict(heads=65538, os=(2 ** 21, 16), qs=(2 ** 21, 16))])
def test_attend_refuses(cutt, change):
    assert cutt.cuttAttendPages(*{**ATTEND, **change}.values()) == BAD


def test_strides_are_as_many_as_axes(cutt):
    with pytest.raises(ValueError):
        cutt.cuttAttendPages(*{**ATTEND, "cs": (32, 16)}.values())
    with pytest.raises(ValueError):
        cutt.cuttGroupedProduct(*{**PRODUCT, "ws": (384, 24, 1)}.values())


def test_workspace_of_sizes_out_of_range(cutt):
    for bad in ((-1, 8, 2, 16, 16, 8, 0), (4, 8, 3, 16, 16, 8, 0), (4, 8, 2, 257, 16, 8, 0), (4, 8, 2, 16, 0, 8, 0), (4, 8, 2, 16, 16, 0, 0), (4, 8, 2, 16, 16, 8, -1),
                (2 ** 31, 8, 2, 16, 16, 8, 0), (4, 65538, 2, 16, 16, 8, 0)):
        assert cutt.cuttAttendPagesWorkspace(*bad) == 0


def test_no_queries_need_no_workspace(cutt):
    for sizes in ((8, 2, 16, 16, 8), (64, 8, 128, 64, 2048), (16, 16, 256, 16, 4096)):
        assert cutt.cuttAttendPagesWorkspace(0, *sizes, 0) == 0
    nothing = dict(queries=0, table=4096, positions=0, q=0, out=0, logs=0, work=0, space=0)
    assert cutt.cuttAttendPages(*{**ATTEND, **nothing}.values()) == OK


# ---- on a stand-in for the kernels' layer -----------------------------------------
class ProductArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("rows", "groups", "inner", "outer")] + [(n, ctypes.c_void_p) for n in ("offsets", "x", "w", "y")] + \
        [(n, ctypes.c_uint64) for n in ("xStride", "yStride", "wGroup", "wRow")]


@pytest.fixture(scope="module")
def stub_lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("stub") / "libproducts.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wall", "-Wextra", "-I" + os.path.join(ROOT, "cutt_amd", "csrc"),
                           os.path.join(ROOT, "tests", "products_layer_stub.cpp"), os.path.join(ROOT, "cutt_amd", "csrc", "products_api.cpp"), "-o", out])
    return ctypes.CDLL(out)


@pytest.fixture
def stub(cutt, stub_lib, monkeypatch):
    """The binding on the stand-in; `stub.launches()` counts what got through since the last look."""
    for name in dir(cutt):
        if name.startswith(("cuttGrouped", "cuttAttend")):
            f, real = getattr(stub_lib, name), getattr(cutt.lib(), name)
            f.argtypes, f.restype = real.argtypes, real.restype
    monkeypatch.setattr(cutt.api, "_lib", stub_lib)
    numbers = {n: t.in_dll(stub_lib, n) for n, t in (("stubLaunches", ctypes.c_int), ("stubResult", ctypes.c_int), ("stubSpace", ctypes.c_ulonglong))}
    for n in numbers.values():
        n.value = 0

    def launches():
        n, numbers["stubLaunches"].value = numbers["stubLaunches"].value, 0
        return n

    monkeypatch.setattr(cutt, "launches", launches, raising=False)
    monkeypatch.setattr(cutt, "numbers", numbers, raising=False)
    monkeypatch.setattr(cutt, "product", ProductArgs.in_dll(stub_lib, "stubProduct"), raising=False)
    return cutt


def test_accepted(stub):
    assert stub.cuttGroupedProduct(*PRODUCT.values()) == OK and stub.launches() == 1
    assert stub.cuttGroupedProduct(*{**PRODUCT, "transposed": 1, "ws": (384, 16)}.values()) == OK and stub.launches() == 1
    assert stub.cuttGroupedProductWeights(*WEIGHTS.values()) == OK and stub.launches() == 1
    assert stub.cuttAttendPages(*ATTEND.values()) == OK and stub.launches() == 1
    for change in (dict(owners=I), dict(logs=0), dict(qs=(16, 64)), dict(qs=(0, 0)), dict(os=(16, 64)), dict(cs=(512, 16, 256)), dict(cs=(0, 0, 0)), dict(window=5),
                   dict(pages=0, k=0, v=0), dict(requests=0, tables=0), dict(k=D, v=D), dict(scale=-1.0), dict(table=2 ** 20, page=2 ** 20)):
        assert stub.cuttAttendPages(*{**ATTEND, **change}.values()) == OK and stub.launches() == 1, change
    # weights shared by all groups, rows read again and again
    assert stub.cuttGroupedProduct(*{**PRODUCT, "ws": (0, 24), "xs": 0}.values()) == OK and stub.launches() == 1


def test_nothing_to_do_is_no_error(stub):
    assert stub.cuttGroupedProduct(*{**PRODUCT, "rows": 0, "x": 0, "y": 0}.values()) == OK and stub.launches() == 0
    assert stub.cuttAttendPages(*{**ATTEND, "queries": 0, "positions": 0, "q": 0, "out": 0, "logs": 0}.values()) == OK and stub.launches() == 0
    # no rows: the weights' gradients are zeros, which have to be written
    assert stub.cuttGroupedProductWeights(*{**WEIGHTS, "rows": 0, "x": 0, "dy": 0}.values()) == OK and stub.launches() == 1


def test_a_refused_launch_is_an_internal_error(stub):
    stub.numbers["stubResult"].value = 1
    assert stub.cuttGroupedProduct(*PRODUCT.values()) == FAILED
    assert stub.cuttGroupedProductWeights(*WEIGHTS.values()) == FAILED
    assert stub.cuttAttendPages(*ATTEND.values()) == FAILED


def test_workspace_has_to_suffice(stub):
    stub.numbers["stubSpace"].value = 4096
    assert stub.cuttAttendPagesWorkspace(4, 8, 2, 16, 16, 8, 0) == 4096
    assert stub.cuttAttendPages(*{**ATTEND, "space": 4096}.values()) == OK
    for change in (dict(space=4095), dict(work=0), dict(work=H + 2), dict(work=F), dict(work=D + 4), dict(work=G - 4092), dict(work=A - 4)):
        assert stub.cuttAttendPages(*{**ATTEND, **change}.values()) == BAD, change


def test_strides_of_single_entries_are_not_passed_on(stub):
    """The stride of an axis with one entry may be anything; the kernels get 0."""
    odd = 2 ** 61
    assert stub.cuttGroupedProduct(*{**PRODUCT, "rows": 1, "groups": 1, "xs": odd, "ys": odd, "ws": (-odd, 24)}.values()) == OK
    a = stub.product
    assert (a.xStride, a.yStride, a.wGroup, a.wRow) == (0, 0, 0, 24)
    assert stub.cuttGroupedProductWeights(*{**WEIGHTS, "inner": 1, "ws": (24, -odd)}.values()) == OK
    assert (a.xStride, a.yStride, a.wGroup, a.wRow) == (16, 0, 24, 24)
    assert stub.cuttAttendPages(*{**ATTEND, "queries": 1, "qs": (-odd, 16), "os": (-odd, 16)}.values()) == OK


def test_columns_of_one_buffer(stub):
    """x and y side by side in the rows of one buffer are accepted, rows that share a column are not."""
    for apart, answer in ((16, OK), (15, BAD), (40, OK), (41, BAD), (0, BAD)):
        assert stub.cuttGroupedProduct(*{**PRODUCT, "xs": 64, "ys": 64, "y": B + 2 * apart}.values()) == answer, apart


def test_random_arguments(stub):
    """Whatever the numbers are, a call is refused with the one code for it or gets through to the layer."""
    rng = np.random.default_rng(0)
    sizes = [0, 1, 2, 4, 16, 64, 100, 256, 1024, 2 ** 20, 2 ** 31 - 1, -1]
    strides = [0, 1, 16, 64, 4096, 2 ** 40, 2 ** 62, 2 ** 63 - 1, -1, -2 ** 63]

    def size():
        return int(rng.choice(sizes))

    def stride():
        return strides[rng.integers(len(strides))]

    def at():
        return 0 if rng.integers(20) == 0 else int(0x100000000000 * rng.integers(1, 60) + rng.choice([0, 0, 0, 4, 8, 2, 64]))

    through = 0
    for _ in range(20000):
        which = rng.integers(3)
        if which == 0:
            r = stub.cuttGroupedProduct(size(), size(), size(), size(), int(rng.integers(0, 4)), int(rng.integers(2)), 0, at(), at(), stride(), at(),
                                        (stride(), stride()), at(), stride())
        elif which == 1:
            r = stub.cuttGroupedProductWeights(size(), size(), size(), size(), int(rng.integers(0, 4)), 0, at(), at(), stride(), at(), stride(), at(),
                                               (stride(), stride()))
        else:
            heads = size()
            r = stub.cuttAttendPages(size(), size(), heads, rng.choice([heads, 1, 2]), size(), int(rng.integers(0, 4)), size(), size(), size(), size(), 1.0, 0, at(),
                                     at(), at(), at(), (stride(), stride()), at(), at(), (stride(), stride(), stride()), at(), (stride(), stride()), at(), at(), 0)
        n = stub.launches()
        assert r in (OK, BAD) and n <= (r == OK)
        through += n
    assert through > 100


# ---- the oracle -------------------------------------------------------------------
def test_oracle_products_by_hand():
    x = np.arange(8.0).reshape(4, 2)
    w = np.array([[[1.0, 2.0, 3.0], [4.0, 5.0, 6.0]], [[1.0, 0.0, 0.0], [0.0, 1.0, 0.0]]])
    y, size = product_oracle.grouped(x, w, [0, 1, 3], False, np.full((4, 3), 9.0))
    assert y.tolist() == [[4, 5, 6], [2, 3, 0], [4, 5, 0], [9, 9, 9]] and size[0].tolist() == [4, 5, 6]
    turned, _ = product_oracle.grouped(x, w.transpose(0, 2, 1), [0, 1, 3], True, np.full((4, 3), 9.0))
    assert np.array_equal(turned, y)
    dw, _ = product_oracle.weights(x, y, [0, 1, 3], 2)
    assert dw[0].tolist() == [[0, 0, 0], [4, 5, 6]] and dw[1].tolist() == [[2 * 2 + 4 * 4, 2 * 3 + 4 * 5, 0], [3 * 2 + 5 * 4, 3 * 3 + 5 * 5, 0]]
    assert product_oracle.bounds([-3, 2, 1, 9], 4) == [(0, 2), (2, 2), (1, 4)]


def test_oracle_attention_by_hand():
    table = np.array([[1, 0], [-1, 1]])
    assert product_oracle.seen(2, 0, table, 2, 2, 0) == [(1, 0), (1, 1), (0, 0)]
    assert product_oracle.seen(9, 0, table, 2, 2, 8) == [(0, 0), (0, 1)] and product_oracle.seen(3, 1, table, 2, 2, 0) == [(1, 0), (1, 1)]
    for nothing in ((-1, 0), (3, 2), (3, -1), (1, 1)):
        assert product_oracle.seen(*nothing, table, 2, 2, 0) == []
    k = np.zeros((2, 2, 1, 1))
    v = np.arange(4.0).reshape(2, 2, 1, 1)
    out, logs, *_ = product_oracle.attend(np.ones((2, 2, 1)), k, v, table, [0, 1], [2, 0], 0, 1.0)
    assert np.allclose(out[0], (2 + 3 + 0) / 3) and np.allclose(logs[0], np.log(3)) and (out[1] == 0).all() and np.isneginf(logs[1]).all()


def test_oracle_attention_is_the_gradient_of_its_log_sums():
    """d logSums / d (a shift of the score of token t) is the token's weight: with values one at a time, by central differences."""
    rng = np.random.default_rng(1)
    table, owners, positions = np.array([[0, 1]]), [0], [3]
    q, k = rng.standard_normal((1, 1, 3)), rng.standard_normal((2, 2, 1, 3))
    step = 1e-6
    for p, s in itertools.product(range(2), range(2)):
        v = np.zeros_like(k)
        v[p, s] = 1.0
        out = product_oracle.attend(q, k, v, table, owners, positions, 0, 0.7)[0][0, 0, 0]
        ends = []
        for sign in (1, -1):
            moved = k.copy()
            moved[p, s, 0] += sign * step * q[0, 0] / (q[0, 0] @ q[0, 0])
            ends.append(product_oracle.attend(q, moved, v, table, owners, positions, 0, 0.7)[1][0, 0])
        assert abs((ends[0] - ends[1]) / (2 * step * 0.7) - out) < 1e-8
