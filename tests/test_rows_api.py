"""The row operators' boundary without a GPU: exported under their declared names, refusals before any device
access, sizes that need no work, and the oracle of the GPU tests against hand-made values and differences."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import row_oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")
OK, BAD = 0, 2
# Addresses are compared and checked for alignment, never read, on the paths taken here.
A, B, C, D, E, F, G = (0x10000000 * i for i in range(1, 8))


def test_every_declared_function_is_exported_and_bound(cutt):
    text = re.sub(r"/\*.*?\*/", " ", open(os.path.join(INCLUDE, "cutt_rows.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(cutt[A-Z]\w*)\s*\(", text))
    assert len(names) == 10
    lib = ctypes.CDLL(cutt.lib_path())
    for n in names:
        assert hasattr(lib, n) and callable(getattr(cutt, n)), n
    for n, v in (("CUTT_F32", 0), ("CUTT_F16", 1), ("CUTT_BF16", 2), ("CUTT_MAX_EXPERTS", 1024)):
        assert getattr(cutt, n) == v
        assert re.search(r"%s\s*=?\s*%d" % (n, v), text)


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "caller.c"
    src.write_text('#include "cutt_rows.h"\n'
                   "int main(void) { return cuttExpertRows(5, 2, 8, 16) == 130 && cuttExpertSort(0, 0, 0, 0, 1, 0, 4, 0, 0, 0, 0, 0, 0, 0, 0) == "
                   "CUTT_INVALID_PARAMETER ? 0 : 1; }\n")
    exe = str(tmp_path / "caller")
    libdir = os.path.join(ROOT, "cutt_amd")
    subprocess.check_call(["gcc", "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror", "-I", INCLUDE, str(src), "-o", exe, "-L", libdir, "-lcutt",
                           "-Wl,-rpath," + libdir, "-Wl,-rpath-link,/opt/rocm/lib"])
    assert subprocess.run([exe], timeout=120).returncode == 0


def test_rows_bound(cutt):
    assert cutt.cuttExpertRows(0, 1, 1, 64) == 0
    assert cutt.cuttExpertRows(5, 2, 8, 16) == 10 + 8 * 15
    assert cutt.cuttExpertRows(3, 1, 8, 16) == 3 + 3 * 15
    assert cutt.cuttExpertRows(2 ** 31 - 1, 1, 1, 1) == 2 ** 31 - 1
    for bad in ((-1, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1025, 1), (1, 1, 1, 0), (2 ** 30, 2, 1, 1), (2 ** 31 - 1, 1, 2, 2)):
        assert cutt.cuttExpertRows(*bad) == -1
    for ids in ([[0, 1], [1, 2]], [[3, 3], [3, 3]], [[0, 5], [7, 9]]):
        counts, offsets, position, source = row_oracle.sort(ids, 0, 8, 16, 1000)
        assert offsets[-1] <= cutt.cuttExpertRows(2, 2, 8, 16)


SORT = dict(tokens=4, choices=2, first=0, experts=8, align=1, rows=8, id_size=4, stream=0, ids=A, counts=B, offsets=C, position=D, source=E)


@pytest.mark.parametrize("change", [dict(tokens=-1), dict(choices=0), dict(experts=0), dict(experts=1025), dict(align=0), dict(rows=-1),
                                    dict(id_size=2), dict(id_size=0), dict(ids=0), dict(ids=A + 2), dict(id_size=8, ids=A + 4), dict(counts=0),
                                    dict(offsets=0), dict(position=0), dict(source=0), dict(source=E + 1), dict(position=A), dict(counts=C + 32),
                                    dict(source=D + 28), dict(tokens=2 ** 30), dict(align=2 ** 29)])
def test_sort_refuses(cutt, change):
    assert cutt.cuttExpertSort(*{**SORT, **change}.values()) == BAD


def test_sort_refuses_a_short_workspace(cutt):
    need = cutt.cuttExpertSortWorkspace(1 << 20, 8, 256)
    if need:
        big = {**SORT, "tokens": 1 << 20, "choices": 8, "experts": 256, "rows": 0, "source": 0}
        assert cutt.cuttExpertSort(*big.values(), F, need - 1) == BAD
        assert cutt.cuttExpertSort(*big.values(), 0, need) == BAD
        assert cutt.cuttExpertSort(*big.values(), F + 2, need) == BAD
    assert cutt.cuttExpertSortWorkspace(-1, 1, 1) == 0


DISPATCH = dict(tokens=4, choices=2, rows=8, width=16, size=2, stream=0, position=A, source=B, x=C, xs=16, y=D, ys=16)


@pytest.mark.parametrize("change", [dict(tokens=-1), dict(choices=0), dict(rows=-1), dict(width=0), dict(size=3), dict(size=16), dict(size=0),
                                    dict(position=0), dict(source=0), dict(x=0), dict(y=0), dict(x=C + 1), dict(y=D + 1), dict(xs=-1), dict(ys=15),
                                    dict(xs=-16), dict(y=C), dict(y=C + 120), dict(y=A), dict(position=A + 2), dict(xs=2 ** 62), dict(tokens=2 ** 30)])
def test_dispatch_refuses(cutt, change):
    assert cutt.cuttExpertDispatch(*{**DISPATCH, **change}.values()) == BAD


def test_nothing_to_do_is_no_error(cutt):
    assert cutt.cuttExpertDispatch(*{**DISPATCH, "tokens": 0, "rows": 0, "position": 0, "source": 0, "x": 0, "y": 0}.values()) == OK
    assert cutt.cuttExpertDispatchBackward(0, 2, 0, 16, 0, 0, 0, 0, 16, 0, 16) == OK
    assert cutt.cuttExpertCombine(0, 2, 8, 16, 0, 0, 0, 0, A, 16, 0, 16) == OK
    assert cutt.cuttExpertCombineBackward(0, 2, 0, 16, 0, 0, 0, 0, 0, 0, 16, 0, 16, 0, 16, 0) == OK
    assert cutt.cuttPageStore(0, 2, 16, 2, 4, 16, 0, 0, 0, 0, (32, 16), A, 0, (512, 32, 16)) == OK
    # no rows: gradients of rows alone are none
    assert cutt.cuttExpertCombineBackward(*{**BACKWARD, "rows": 0, "dweights": 0}.values()) == OK
    assert cutt.cuttExpertCombineBackward(*{**BACKWARD, "rows": 0, "dy": 0, "source": 0, "dweights": 0}.values()) == OK
    assert cutt.cuttPageStore(4, 2, 16, 2, 0, 16, 0, A, B, 0, (32, 16), 0, 0, (512, 32, 16)) == OK


COMBINE = dict(tokens=4, choices=2, rows=8, width=16, type=2, stream=0, position=A, weights=B, y=C, ys=16, out=D, outs=16)


@pytest.mark.parametrize("change", [dict(tokens=-1), dict(choices=0), dict(rows=-1), dict(width=0), dict(type=3), dict(type=-1), dict(position=0),
                                    dict(weights=0), dict(weights=B + 2), dict(y=0), dict(out=0), dict(out=D + 1), dict(ys=-1), dict(outs=1),
                                    dict(out=C + 8 * 32 - 2), dict(out=B), dict(out=A)])
def test_combine_refuses(cutt, change):
    assert cutt.cuttExpertCombine(*{**COMBINE, **change}.values()) == BAD
    without = {k: v for k, v in {**COMBINE, **change}.items() if k != "weights"}
    if "weights" not in change and change.get("out") != B:
        assert cutt.cuttExpertDispatchBackward(*without.values()) == BAD


BACKWARD = dict(tokens=4, choices=2, rows=8, width=16, type=2, stream=0, position=A, source=B, weights=C, y=D, ys=16, dout=E, douts=16, dy=F, dys=16,
                dweights=G)


@pytest.mark.parametrize("change", [dict(tokens=-1), dict(type=3), dict(width=0), dict(position=0), dict(source=0), dict(weights=0), dict(y=0),
                                    dict(dout=0), dict(dy=0, dweights=0), dict(dy=D), dict(dy=E), dict(dy=G), dict(dweights=G + 1), dict(ys=-1),
                                    dict(douts=-16), dict(dys=1), dict(dweights=C), dict(dy=F + 1)])
def test_combine_backward_refuses(cutt, change):
    assert cutt.cuttExpertCombineBackward(*{**BACKWARD, **change}.values()) == BAD


TABLES = dict(requests=4, page=16, width=8, free_count=8, tokens=32, stream=0, cached=A, added=B, free=C, tables=D, starts=E, used=F, slots=G, positions=0)


@pytest.mark.parametrize("change", [dict(requests=-1), dict(page=0), dict(width=0), dict(free_count=-1), dict(tokens=-1), dict(cached=0), dict(added=0),
                                    dict(free=0), dict(tables=0), dict(starts=0), dict(used=0), dict(slots=0), dict(slots=G + 4), dict(used=E),
                                    dict(tables=A), dict(positions=G), dict(positions=2)])
def test_tables_refuses(cutt, change):
    assert cutt.cuttPageTables(*{**TABLES, **change}.values()) == BAD


PAGES = dict(tokens=4, heads=2, width=16, size=2, pages=4, page=16, stream=0, slots=A, k=B, v=C, rows=(32, 16), kc=D, vc=E, cache=(512, 32, 16))


@pytest.mark.parametrize("change", [dict(tokens=-1), dict(heads=0), dict(width=0), dict(size=3), dict(pages=-1), dict(page=0), dict(slots=0),
                                    dict(slots=A + 4), dict(k=0), dict(v=0), dict(vc=0), dict(kc=0), dict(rows=None), dict(cache=None),
                                    dict(rows=(-32, 16)), dict(cache=(512, 32, -16)), dict(kc=B), dict(kc=C + 64), dict(k=B + 1), dict(vc=E + 1)])
def test_page_moves_refuse(cutt, change):
    args = {**PAGES, **change}
    assert cutt.cuttPageStore(*args.values()) == BAD
    assert cutt.cuttPageLoad(*args.values()) == BAD


def test_page_moves_refuse_rows_on_top_of_each_other(cutt):
    assert cutt.cuttPageStore(*{**PAGES, "cache": (512, 32, 0)}.values()) == BAD
    assert cutt.cuttPageStore(*{**PAGES, "cache": (512, 15, 16)}.values()) == BAD
    assert cutt.cuttPageLoad(*{**PAGES, "rows": (0, 16)}.values()) == BAD
    with pytest.raises(ValueError):
        cutt.cuttPageStore(*{**PAGES, "rows": (32,)}.values())


SANITIZED = ["-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-g", "-O1", "-std=c++17", "-Wall", "-Wextra"]


def test_random_arguments_under_sanitizers(tmp_path):
    """rows_api.cpp on a stand-in for the kernels' layer that looks at what reaches it, with random and extreme arguments."""
    exe = str(tmp_path / "rows_api_stress")
    r = subprocess.run(["g++"] + SANITIZED + ["-I" + INCLUDE, "-I" + os.path.join(ROOT, "cutt_amd", "csrc"), os.path.join(ROOT, "tests", "rows_api_stress.cpp"),
                        os.path.join(ROOT, "cutt_amd", "csrc", "rows_api.cpp"), "-o", exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-3000:]
    assert "rows api ok" in r.stdout


def test_rows_side_by_side_do_not_overlap(cutt):
    """Input and output as columns of one buffer: refused only where they share some (the accepted ones get as far as the launch)."""
    def call(x, y, stride=48):
        return cutt.cuttExpertDispatch(*{**DISPATCH, "x": x, "y": y, "xs": stride, "ys": stride}.values())

    assert call(C, C + 30) == BAD and call(C, C + 66) == BAD and call(C + 64, C) != BAD and call(C, C + 32) != BAD and call(C, C + 96 * 2 + 64) != BAD
    assert call(C + 96 + 32, C) != BAD and call(C + 96 + 30, C) == BAD and call(C + 96 - 30, C) == BAD
    assert cutt.cuttExpertDispatch(*{**DISPATCH, "x": C, "y": C + 32, "xs": 48, "ys": 32}.values()) == BAD


# ---- the oracle ---------------------------------------------------------------
def test_oracle_sort_by_hand():
    counts, offsets, position, source = row_oracle.sort([[2, 0], [0, 9], [2, 2]], 0, 3, 4, 10)
    assert counts.tolist() == [2, 0, 3] and offsets.tolist() == [0, 4, 4, 8]
    assert position.tolist() == [[4, 0], [1, -1], [5, 6]]
    assert source.tolist() == [1, 2, -1, -1, 0, 4, 5, -1, -1, -1]


def test_oracle_tables_by_hand():
    table = np.full((3, 3), -1, dtype=np.int32)
    table[0, 0] = 7
    table, starts, used, slots, positions = row_oracle.tables([3, 0, 0], [2, 0, 5], 4, [5, 6], table, 9)
    assert table.tolist() == [[7, 5, -1], [-1, -1, -1], [6, -1, -1]]
    assert starts.tolist() == [0, 2, 2, 7] and used.tolist() == [3]
    assert slots.tolist() == [31, 20, 24, 25, 26, 27, -1, -1, -1] and positions.tolist() == [3, 4, 0, 1, 2, 3, 4, -1, -1]


def test_oracle_gradients_against_differences():
    """The operators are linear in the rows and in the weights: differences of one step are exact up to rounding in 64 bits."""
    rng = np.random.default_rng(0)
    _, _, position, source = row_oracle.sort(rng.integers(-1, 4, (5, 3)), 0, 4, 4, 40)
    y, dout, w = rng.standard_normal((40, 3)), rng.standard_normal((5, 3)), rng.standard_normal((5, 3))
    dy, dw, _ = row_oracle.combine_backward(y, dout, position, source, w, np.zeros_like(y))
    dx, _ = row_oracle.combine(y, position)

    def loss(y, w):
        return (dout * row_oracle.combine(y, position, w)[0]).sum()

    for grad, of in ((dy, 0), (dw, 1)):
        for at in np.ndindex(grad.shape):
            moved = [y.copy(), w.copy()]
            moved[of][at] += 1.0
            assert abs(loss(*moved) - loss(y, w) - grad[at]) < 1e-12
    x = rng.standard_normal((5, 3))
    for at in np.ndindex(x.shape):
        moved = x.copy()
        moved[at] += 1.0
        zero = np.zeros_like(y)
        step = (y * (row_oracle.dispatch(moved, position, source, zero) - row_oracle.dispatch(x, position, source, zero))).sum()
        assert abs(step - dx[at]) < 1e-12
