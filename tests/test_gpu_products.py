"""The products against the oracle in 64 bits.

Tolerances.  A sum of n products in 32 bits is within (n + 2) * 2^-23 of the sum of the terms' sizes (each addition and each product off by a step at most),
and its result within half a step of its type.  Where all terms are small whole numbers the sums are exact, and results are compared bit by bit: they are the
exact sum rounded once.  Attention: a score is off by d = (width + 4) * 2^-23 times its terms' sizes, an exponential by that relative to itself and a few steps, numerator
and denominator alike; 16-bit types keep an exponential in two parts, each within half a step of what it stands for, or half of the smallest step (2^-25 for half)."""
import itertools

import numpy as np
import pytest
import torch

import cutt_amd as cutt
import product_oracle as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids_of = [str(t).split(".")[1] for t in TYPES]
CODE = {torch.float32: cutt.CUTT_F32, torch.float16: cutt.CUTT_F16, torch.bfloat16: cutt.CUTT_BF16}
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
UNIT = 2.0 ** -23


def stream():
    return torch.cuda.current_stream().cuda_stream


def ok(code):
    assert code == cutt.CUTT_SUCCESS, code


def np64(t):
    return t.double().cpu().numpy()


def made(shape, dtype, whole, g, high=4):
    """Values on the GPU: small whole numbers, or normal ones."""
    if whole:
        return torch.randint(-high, high + 1, shape, generator=g, device="cuda").to(dtype)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def placed(t, pitch, shift):
    """The rows of t [..., width] in a buffer of their own, `pitch` elements apart and `shift` elements off its start; the buffer, and the view."""
    rows = int(np.prod(t.shape[:-1]))
    buffer = torch.full((shift + rows * pitch + 64,), 77.0, dtype=t.dtype, device="cuda")
    strides, step = [], pitch
    for n in reversed(t.shape[:-1]):
        strides.insert(0, step)
        step *= n
    view = buffer.as_strided(t.shape, strides + [1], shift)
    view.copy_(t)
    return buffer, view


def within(got, want, tolerance):
    got = np64(got)
    bad = ~(np.abs(got - want) <= tolerance)
    assert not bad.any(), (int(bad.sum()), got[bad][:5], want[bad][:5], np.broadcast_to(tolerance, want.shape)[bad][:5])


# ---- products -------------------------------------------------------------------
def run_product(x, w, offsets, transposed, y):
    groups, inner = w.shape[0], x.shape[1]
    outer = w.shape[1] if transposed else w.shape[2]
    assert w.stride(2) == 1 and x.stride(1) == 1 and y.stride(1) == 1
    ok(cutt.cuttGroupedProduct(x.shape[0], groups, inner, outer, CODE[x.dtype], transposed, stream(), offsets.data_ptr(), x.data_ptr(), x.stride(0), w.data_ptr(),
                               w.stride()[:2], y.data_ptr(), y.stride(0)))
    return y


def run_weights(x, dy, offsets, dw):
    ok(cutt.cuttGroupedProductWeights(x.shape[0], dw.shape[0], x.shape[1], dy.shape[1], CODE[x.dtype], stream(), offsets.data_ptr(), x.data_ptr(), x.stride(0),
                                      dy.data_ptr(), dy.stride(0), dw.data_ptr(), dw.stride()[:2]))
    return dw


GROUPS = {
    "ragged": [5, 0, 1, 130, 17, 0, 64, 31, 33],
    "one": [300],
    "first": [260, 0, 0, 0],
    "last": [0, 0, 0, 129],
    "singles": [1] * 70,
    "empty": [0, 0, 0],
    "tail": [3, 2],
    "many": [3, 0, 1, 2, 0, 5, 0, 0] * 40,
}
SIZES = [(64, 128), (1, 1), (7, 3), (100, 36), (136, 264), (65, 513), (520, 100), (200, 129), (33, 16), (256, 512)]


def offsets_of(counts, first=0):
    return torch.tensor(np.cumsum([first] + counts), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("groups,size", [(g, s) for i, g in enumerate(GROUPS) for j, s in enumerate(SIZES) if (i + j) % 3 == 0 or g == "ragged"],
                         ids=lambda v: v if isinstance(v, str) else "%dx%d" % v)
def test_product(groups, size, transposed, dtype):
    """Whole numbers, exact sums; a few rows in front of the first group and behind the last one, which stay as they were."""
    counts, (inner, outer) = GROUPS[groups], size
    g, first = generator(1), 2
    rows = first + sum(counts) + 3
    x = made((rows, inner), dtype, True, g)
    w = made((len(counts), outer, inner) if transposed else (len(counts), inner, outer), dtype, True, g, 2)
    y = made((rows, outer), dtype, True, g)
    offsets = offsets_of(counts, first)
    want, _ = oracle.grouped(np64(x), np64(w), offsets.cpu().numpy(), transposed, np64(y))
    run_product(x, w, offsets, transposed, y)
    assert torch.equal(y, torch.tensor(want, device="cuda").to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("groups,size", [(g, s) for i, g in enumerate(GROUPS) for j, s in enumerate(SIZES) if (i + j) % 3 == 0 or g == "ragged"],
                         ids=lambda v: v if isinstance(v, str) else "%dx%d" % v)
def test_weights(groups, size, dtype):
    counts, (inner, outer) = GROUPS[groups], size
    g, first = generator(2), 2
    rows = first + sum(counts) + 3
    x, dy = made((rows, inner), dtype, True, g), made((rows, outer), dtype, True, g)
    dw = made((len(counts), inner, outer), dtype, True, g)
    offsets = offsets_of(counts, first)
    want, _ = oracle.weights(np64(x), np64(dy), offsets.cpu().numpy(), len(counts))
    run_weights(x, dy, offsets, dw)
    assert torch.equal(dw, torch.tensor(want, device="cuda").to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("counts,inner,outer", [([200, 7, 0, 60], 520, 192), ([3, 1, 2, 4], 1000, 130), ([40, 33, 64, 20], 300, 256), ([2] * 5, 77, 333)])
def test_values(counts, inner, outer, transposed, dtype):
    g = generator(3)
    rows, n = sum(counts), len(counts)
    x, dy, offsets = made((rows, inner), dtype, False, g), made((rows, outer), dtype, False, g), offsets_of(counts)
    w = made((n, outer, inner) if transposed else (n, inner, outer), dtype, False, g)
    want, size = oracle.grouped(np64(x), np64(w), offsets.cpu().numpy(), transposed, np.zeros((rows, outer)))
    within(run_product(x, w, offsets, transposed, torch.empty_like(dy)), want, size * (inner + 2) * UNIT + np.abs(want) * HALF[dtype] + LEAST[dtype])
    want, size = oracle.weights(np64(x), np64(dy), offsets.cpu().numpy(), n)
    within(run_weights(x, dy, offsets, torch.empty(n, inner, outer, dtype=dtype, device="cuda")), want,
           size * (max(counts) + 2) * UNIT + np.abs(want) * HALF[dtype] + LEAST[dtype])


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("shift,pad", list(itertools.product([0, 1, 8], [0, 1, 8, 24])))
def test_strides_and_alignment(shift, pad, dtype):
    """Buffers off the 16-byte grid and rows further apart than their width: results as from dense ones, and nothing written between the rows."""
    g, counts, inner, outer = generator(4), [70, 0, 3, 140], 136, 200
    rows, n, offsets = sum(counts), len(counts), offsets_of(counts)
    x, dy = made((rows, inner), dtype, True, g), made((rows, outer), dtype, True, g)
    for transposed in (False, True):
        w = made((n, outer, inner) if transposed else (n, inner, outer), dtype, True, g, 2)
        want = run_product(x, w, offsets, transposed, torch.zeros_like(dy))
        buffer, y = placed(torch.zeros_like(dy), outer + pad, shift)
        clean = buffer.clone()
        run_product(placed(x, inner + pad, shift)[1], placed(w, w.shape[2] + pad, shift)[1], offsets, transposed, y)
        assert torch.equal(y, want)
        y.zero_()
        assert torch.equal(buffer, clean)
    want = run_weights(x, dy, offsets, torch.zeros(n, inner, outer, dtype=dtype, device="cuda"))
    buffer, dw = placed(torch.zeros_like(want), outer + pad, shift)
    clean = buffer.clone()
    run_weights(placed(x, inner + pad, shift)[1], placed(dy, outer + pad, shift)[1], offsets, dw)
    assert torch.equal(dw, want)
    dw.zero_()
    assert torch.equal(buffer, clean)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_neighbours_do_not_leak(dtype):
    """Infinities and NaN in rows of other groups and of none, and beyond the rows' widths, have no part in a group's results."""
    g, counts, inner, outer = generator(5), [9, 40, 150, 1], 72, 136
    for bad in (float("nan"), float("inf")):
        offsets = offsets_of(counts, 4)
        rows, n = 4 + sum(counts) + 5, len(counts)
        x, dy = made((rows, inner), dtype, True, g), made((rows, outer), dtype, True, g)
        w = made((n, inner, outer), dtype, True, g, 2)
        want = run_product(x, w, offsets, False, torch.zeros_like(dy))
        wants = run_weights(x, dy, offsets, torch.zeros(n, inner, outer, dtype=dtype, device="cuda"))
        turned = run_product(x, w.transpose(1, 2).contiguous(), offsets, True, torch.zeros_like(dy))
        assert torch.equal(turned, want)
        for e in range(n):
            lo, hi = offsets[e:e + 2].tolist()
            mine = torch.zeros(rows, 1, dtype=torch.bool, device="cuda")
            mine[lo:hi] = True
            xs, ds = (placed(t.masked_fill(~mine, bad), t.shape[1] + 8, 0) for t in (x, dy))
            for buffer, view in (xs, ds):
                keep = view.clone()
                buffer.fill_(bad)
                view.copy_(keep)
            ws = torch.full((n, inner + 8, outer + 8), bad, dtype=dtype, device="cuda")
            ws[e, :inner, :outer] = w[e]
            assert torch.equal(run_product(xs[1], ws[:, :inner, :outer], offsets, False, torch.zeros_like(dy))[lo:hi], want[lo:hi])
            wt = torch.full((n, outer + 8, inner + 8), bad, dtype=dtype, device="cuda")
            wt[e, :outer, :inner] = w[e].t()
            assert torch.equal(run_product(xs[1], wt[:, :outer, :inner], offsets, True, torch.zeros_like(dy))[lo:hi], want[lo:hi])
            assert torch.equal(run_weights(xs[1], ds[1], offsets, torch.zeros_like(wants))[e], wants[e])


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("counts,inner,outer", [
    ([3, 0, 1, 2], 1000, 64), ([1, 0, 0, 1, 0, 2], 1, 40), ([2, 1], 4103, 30),   # few rows: k's shared by wavefronts, fewer tiles of k's than wavefronts
    ([90, 1, 33], 264, 136), ([300], 640, 200), ([70, 20], 65, 67),
    ([9] * 40, 136, 520), ([2] * 100, 130, 515),                                 # many groups
    ([400, 390, 0, 420, 380], 200, 2056), ([130] * 60, 72, 512)])
def test_shapes(counts, inner, outer, transposed, dtype):
    """Whole numbers, whose sums are exact: few and many rows to a group, few and many tiles."""
    g = generator(10)
    rows, offsets = sum(counts) + 2, offsets_of(counts)
    x, w = made((rows, inner), dtype, True, g, 2), made((len(counts), outer, inner) if transposed else (len(counts), inner, outer), dtype, True, g, 2)
    y = torch.full((rows, outer), 7, dtype=dtype, device="cuda")
    before = np64(y)
    got = np64(run_product(x, w, offsets, transposed, y))
    want, _ = oracle.grouped(np64(x), np64(w), offsets.cpu().numpy(), transposed, before)
    assert np.array_equal(got, np64(torch.from_numpy(want).to(dtype)))


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("counts,inner,outer", [
    ([300, 0, 1100], 136, 200), ([2000], 64, 64), ([513, 64, 65], 65, 131),   # few results of many rows
    ([500] * 16, 264, 1032), ([40, 3] * 8, 500, 777),                            # more
    ([420] * 12, 2048, 4096)])
def test_gradients_of_all_shapes(counts, inner, outer, dtype):
    """Whole numbers, whose sums are exact."""
    g = generator(8)
    rows, offsets = sum(counts) + 5, offsets_of(counts)
    x, dy = made((rows, inner), dtype, True, g, 2), made((rows, outer), dtype, True, g, 2)
    dw = run_weights(x, dy, offsets, torch.full((len(counts), inner, outer), 7, dtype=dtype, device="cuda"))
    at = 0
    for e, n in enumerate(counts):
        want = x[at:at + n].float().t().contiguous() @ dy[at:at + n].float()
        assert torch.equal(dw[e], want.to(dtype))
        at += n


def test_offsets_out_of_range():
    """Offsets beyond the rows count as the nearer end, groups whose end is not above their start are empty; a guard behind y stays."""
    g, rows, inner, outer = generator(6), 200, 40, 72
    x, guard = made((rows, inner), torch.float16, True, g), torch.full((rows + 300, outer), 5.0, dtype=torch.float16, device="cuda")
    for list_of in ([-7, 3, 150, 2 ** 31 - 1], [-2 ** 31, -1, 0, 199], [0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], [10, 10, 9, 9], [200, 200, 300, 400]):
        offsets = torch.tensor(list_of, dtype=torch.int32, device="cuda")
        for transposed in (False, True):
            w = made((3, outer, inner) if transposed else (3, inner, outer), torch.float16, True, g, 2)
            buffer = guard.clone()
            run_product(x, w, offsets, transposed, buffer[:rows])
            want, _ = oracle.grouped(np64(x), np64(w), list_of, transposed, np64(guard[:rows]))
            assert torch.equal(buffer[:rows], torch.tensor(want, device="cuda").half()) and torch.equal(buffer[rows:], guard[rows:])
        dy = made((rows, outer), torch.float16, True, g)
        dw = run_weights(x, dy, offsets, torch.full((3, inner, outer), 9.0, dtype=torch.float16, device="cuda"))
        assert torch.equal(dw, torch.tensor(oracle.weights(np64(x), np64(dy), list_of, 3)[0], device="cuda").half())


def test_offsets_that_descend_stay_inside():
    """Groups that share rows: results are not said, but the rows behind them stay as they were."""
    rows = 5000
    x, w = torch.ones(rows, 64, device="cuda", dtype=torch.bfloat16), torch.ones(1024, 64, 64, device="cuda", dtype=torch.bfloat16)
    offsets = torch.tensor([0, rows] * 512 + [0], dtype=torch.int32, device="cuda")
    y = torch.full((rows + 512, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    run_product(x, w, offsets, False, y[:rows])
    assert bool((y[rows:] == 3).all())
    assert bool(((y[:rows] == 64) | (y[:rows] == 3)).all())


def test_no_rows():
    w = torch.ones(3, 8, 8, device="cuda")
    dw = torch.full((3, 8, 8), 4.0, device="cuda")
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    none = torch.empty(0, 8, device="cuda")
    run_product(none, w, offsets, False, none.clone())
    run_weights(none, none.clone(), offsets, dw)
    assert bool((dw == 0).all())


@pytest.mark.parametrize("outer", [2 ** 28, 2 ** 28 + 1])
def test_more_tiles_than_workgroups(outer):
    """Results of 13 GB, in more tiles than a launch has workgroups; single products, which are exact in 32 bits and rounded once."""
    g = generator(9)
    x, dy = made((3, 8), torch.bfloat16, True, g), made((3, outer), torch.bfloat16, True, g)
    dw = torch.full((3, 8, outer), 7, dtype=torch.bfloat16, device="cuda")
    run_weights(x, dy, offsets_of([1, 1, 1]), dw)
    for e in range(3):
        for i in range(8):
            assert torch.equal(dw[e, i], x[e, i] * dy[e])


def test_small_numbers():
    """Halves below the normal range count in full: products are exact."""
    x = torch.full((3, 64), 2.0 ** -24, dtype=torch.float16, device="cuda")
    w = torch.full((1, 64, 128), 2.0 ** 10, dtype=torch.float16, device="cuda")
    offsets = offsets_of([3])
    assert bool((run_product(x, w, offsets, False, torch.empty(3, 128, dtype=torch.float16, device="cuda")) == 2.0 ** -8).all())
    assert bool((run_product(x, w.transpose(1, 2).contiguous(), offsets, True, torch.empty(3, 128, dtype=torch.float16, device="cuda")) == 2.0 ** -8).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bfloat16", "float32"])
def test_far_offsets(dtype):
    """Groups of weights and rows more than 2^32 elements apart."""
    far, inner, outer = 2 ** 32 + 16, 64, 128
    buffer = torch.empty(far + 70000, dtype=dtype, device="cuda")
    g = generator(7)
    x, w, offsets = made((6, inner), dtype, True, g), made((2, inner, outer), dtype, True, g, 2), offsets_of([4, 2])
    want = run_product(x, w, offsets, False, torch.empty(6, outer, dtype=dtype, device="cuda"))
    ws = buffer.as_strided((2, inner, outer), (far, outer, 1))
    ws.copy_(w)
    assert torch.equal(run_product(x, ws, offsets, False, torch.empty_like(want)), want)
    del ws
    step = far // 5
    xs = buffer.as_strided((6, inner), (step, 1))
    xs.copy_(x)
    assert torch.equal(run_product(xs, w, offsets, False, torch.empty_like(want)), want)
    wants = run_weights(x, want, offsets, torch.empty(2, inner, outer, dtype=dtype, device="cuda"))
    assert torch.equal(run_weights(xs, want, offsets, torch.empty_like(wants)), wants)
    ys = buffer.as_strided((6, outer), (step, 1))
    run_product(x, w, offsets, False, ys)
    assert torch.equal(ys, want)
    dws = buffer.as_strided((2, inner, outer), (far, outer, 1))
    run_weights(x, want, offsets, dws)
    assert torch.equal(dws, wants)


def test_gradients_against_differences():
    """The product is linear in the rows and in the weights: with small whole numbers, differences of one step are exact."""
    g, counts, inner, outer = generator(8), [3, 0, 5], 6, 4
    rows, offsets = sum(counts), offsets_of(counts)
    x, w, dy = made((rows, inner), torch.float32, True, g), made((3, inner, outer), torch.float32, True, g), made((rows, outer), torch.float32, True, g)

    def loss(x, w):
        return float((run_product(x, w, offsets, False, torch.zeros_like(dy)) * dy).sum())

    dx = run_product(dy, w, offsets, True, torch.zeros_like(x))
    dw = run_weights(x, dy, offsets, torch.empty_like(w))
    for grad, of in ((dx, 0), (dw, 1)):
        for at in np.ndindex(*grad.shape):
            moved = [x.clone(), w.clone()]
            moved[of][at] += 1
            assert loss(*moved) - loss(x, w) == float(grad[at])


# ---- attention --------------------------------------------------------------------
class Cache:
    """Pages [pages, page, key heads, width] in either order, some of nobody's; tables with the requests' pages."""

    def __init__(self, lengths, page, key_heads, width, dtype, layout, g, spare=3, wide=1):
        owned = [-(-n // page) for n in lengths]
        self.pages, self.page = sum(owned) + spare, page
        order = torch.randperm(self.pages, generator=g, device="cuda").to(torch.int32)
        self.tables = torch.full((len(lengths), max(owned + [0]) + wide), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(owned):
            self.tables[b, :n] = order[at:at + n]
            at += n
        shape = (self.pages, page, key_heads, width) if layout == "slot" else (self.pages, key_heads, page, width)
        self.k, self.v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
        if layout == "head":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)


def run_attend(q, cache, owners, positions, window, scale, out=None, logs=True, k=None, v=None):
    k, v = cache.k if k is None else k, cache.v if v is None else v
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda") if out is None else out
    logs = torch.empty(q.shape[:2], device="cuda") if logs else None
    queries, heads, width = q.shape
    requests, table = cache.tables.shape
    space = cutt.cuttAttendPagesWorkspace(queries, heads, k.shape[2], width, cache.page, table, window)
    workspace = torch.full((space + 64,), 0xEE, dtype=torch.uint8, device="cuda")
    ok(cutt.cuttAttendPages(queries, requests, heads, k.shape[2], width, CODE[q.dtype], cache.pages, cache.page, table, window, scale, stream(),
                            cache.tables.data_ptr(), 0 if owners is None else owners.data_ptr(), positions.data_ptr(), q.data_ptr(), q.stride()[:2], k.data_ptr(),
                            v.data_ptr(), k.stride()[:3], out.data_ptr(), out.stride()[:2], 0 if logs is None else logs.data_ptr(), workspace.data_ptr(), space))
    assert bool((workspace[space:] == 0xEE).all())
    return out, logs


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check_attend(q, cache, owners, positions, window, scale, out, logs):
    dtype, width = q.dtype, q.shape[2]
    who = np.arange(q.shape[0]) if owners is None else owners.cpu().numpy()
    want, want_logs, size, terms, count, most = oracle.attend(np64(q), np64(cache.k), np64(cache.v), cache.tables.cpu().numpy(), who, positions.cpu().numpy(),
                                                              window, scale)
    score = terms * (width + 4) * UNIT + 8 * UNIT
    n = count[:, None]
    part = {torch.float32: 0.0, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}[dtype]
    least = n[:, :, None] * most * (2.0 ** -25 if dtype == torch.float16 else 0.0)
    tolerance = size * (2 * np.expm1(2 * score) + (2 * n + 40) * UNIT + part)[:, :, None] + least + np.abs(want) * HALF[dtype] * 1.01 + LEAST[dtype]
    within(out, want, tolerance)
    if logs is not None:
        seen = np.isfinite(want_logs)
        got = np64(logs)
        assert np.array_equal(np.isneginf(got), ~seen)
        bad = np.abs(got[seen] - want_logs[seen]) > (2 * score + (n + 10) * UNIT + 4 * np.abs(np.where(seen, want_logs, 0)) * UNIT)[seen]
        assert not bad.any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("lengths,page,heads,key_heads,width,window,layout", [
    ([5, 1, 0, 70], 16, 8, 2, 64, 0, "slot"),
    ([300, 17], 16, 4, 4, 128, 0, "head"),
    ([1], 1, 1, 1, 128, 0, "slot"),
    ([33, 64, 65, 128], 64, 12, 3, 80, 0, "head"),
    ([129, 500], 3, 5, 5, 96, 0, "slot"),
    ([40, 900], 128, 16, 1, 256, 0, "head"),
    ([257, 31], 32, 40, 1, 128, 0, "slot"),      # more heads per key head than one tile of columns holds
    ([200, 64, 63], 16, 34, 2, 64, 50, "slot"),
    ([1000, 20, 100], 100, 6, 2, 192, 77, "head"),
    ([70, 3], 7, 3, 3, 1, 0, "slot"),
    ([70, 30], 16, 6, 3, 7, 0, "head"),
    ([70, 30], 16, 6, 3, 33, 1, "slot"),
    ([150], 16, 4, 2, 100, 0, "head"),
    ([90, 200], 16, 4, 2, 250, 0, "slot"),
    ([2500, 1, 900], 64, 8, 4, 128, 0, "slot"),
    ([6000], 16, 2, 1, 64, 0, "head"),
])
def test_attend(lengths, page, heads, key_heads, width, window, layout, dtype):
    g = generator(11)
    cache = Cache(lengths, page, key_heads, width, dtype, layout, g)
    q = (2 * torch.randn(len(lengths), heads, width, generator=g, device="cuda")).to(dtype)
    positions, scale = ints([n - 1 for n in lengths]), width ** -0.5
    out, logs = run_attend(q, cache, None, positions, window, scale)
    check_attend(q, cache, None, positions, window, scale, out, logs)
    again, _ = run_attend(q, cache, None, positions, window, scale, logs=False)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("requests,drafts,longest,heads,key_heads,width,window,idle", [
    (40, 1, 700, 16, 8, 64, 0, 5),       # ranges that begin and end within queries
    (30, 3, 500, 8, 8, 128, 0, 7),       # drafted tokens, taken together
    (50, 2, 900, 12, 12, 80, 300, 9),
    (256, 1, 4500, 16, 1, 64, 0, 3),     # queries in two pieces of their own
    (700, 3, 4500, 2, 1, 64, 0, 50),     # and drafted ones
    (700, 3, 4500, 2, 1, 64, 2300, 50),
    (300, 4, 200, 8, 8, 64, 0, 4),       # a workgroup for each
])
def test_shares(requests, drafts, longest, heads, key_heads, width, window, idle, dtype):
    """Many queries of long and short requests, every `idle`-th of which has no token."""
    g = generator(18)
    lengths = torch.randint(1, min(longest, 300), (requests,), generator=g, device="cuda").tolist()
    lengths[::idle] = [0] * len(lengths[::idle])
    lengths[1], lengths[requests // 2 | 1], lengths[-1] = longest, longest - 1, longest // 2 + 5
    cache = Cache(lengths, 32, key_heads, width, dtype, "slot", g)
    owners = ints([b for b in range(requests) for _ in range(drafts)])
    positions = ints([n - drafts + i if n else -1 for n in lengths for i in range(drafts)])
    q = (2 * torch.randn(requests * drafts, heads, width, generator=g, device="cuda")).to(dtype)
    out, logs = run_attend(q, cache, owners, positions, window, width ** -0.5)
    check_attend(q, cache, owners, positions, window, width ** -0.5, out, logs)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("window", [0, 10])
def test_owners_and_positions(window, dtype):
    """Several queries of one request, queries of nobody, positions beyond the table, before the first token and far ones."""
    g = generator(12)
    cache = Cache([150, 0, 90], 16, 2, 64, dtype, "slot", g, wide=0)
    owners = ints([0, 0, 0, 2, 2, 1, -1, 3, 2 ** 31 - 1, 2, 0, 0, 2, 0])
    positions = ints([149, 148, 0, 89, 5, 0, 3, 3, 3, -1, 159, 400, 2 ** 31 - 1, -2 ** 31])
    q = torch.randn(14, 6, 64, generator=g, device="cuda").to(dtype)
    out, logs = run_attend(q, cache, owners, positions, window, 0.2)
    check_attend(q, cache, owners, positions, window, 0.2, out, logs)
    for i in (5, 6, 7, 8, 9, 13):
        assert bool((out[i] == 0).all()) and bool((logs[i] == -float("inf")).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("window,layout", [(0, "slot"), (45, "head")])
def test_absent_pages_and_unseen_values(window, layout, dtype):
    """Table entries that are no pages are not seen, and infinities and NaN outside what is seen have no part."""
    g = generator(13)
    cache = Cache([130, 64, 16, 300], 16, 2, 96, dtype, layout, g)
    cache.tables[0, 2], cache.tables[0, 4], cache.tables[1], cache.tables[3, 0], cache.tables[3, 18] = -5, cache.pages, -1, 2 ** 31 - 1, -2 ** 31
    positions = ints([129, 63, 15, 299])
    q = torch.randn(4, 4, 96, generator=g, device="cuda").to(dtype)
    want, logs = run_attend(q, cache, None, positions, window, 0.1)
    check_attend(q, cache, None, positions, window, 0.1, want, logs)
    assert bool((want[1] == 0).all())
    keep = torch.zeros(cache.pages, 16, dtype=torch.bool, device="cuda")
    table = cache.tables.cpu().numpy()
    for i in range(4):
        for p, s in oracle.seen(int(positions[i]), i, table, cache.pages, 16, window):
            keep[p, s] = True
    for bad in (float("nan"), float("inf"), -float("inf")):
        k, v = (t.masked_fill(~keep[:, :, None, None], bad) for t in (cache.k, cache.v))
        k, v = (torch.empty_strided(t.shape, cache.k.stride(), dtype=dtype, device="cuda").copy_(t) for t in (k, v))
        out, again = run_attend(q, cache, None, positions, window, 0.1, k=k, v=v)
        assert torch.equal(out, want) and torch.equal(again, logs)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_extreme_scores(dtype):
    """Scores far apart: one token takes all of the weight, whatever the order; keys of the lowest value; scores of -infinity."""
    g = generator(14)
    cache = Cache([100, 100, 100], 16, 1, 32, dtype, "slot", g)
    table = cache.tables.cpu().numpy()
    low = torch.finfo(dtype).min if dtype != torch.float16 else -60000.0

    def cell(b, t):
        return int(table[b, t // 16]), t % 16

    cache.k.zero_()
    for b, t in ((0, 0), (1, 57), (2, 99)):
        cache.k[cell(b, t)][0, 0] = 100.0
    for b in range(3):
        cache.k[cell(b, 30)][0, 0] = low
    q = torch.zeros(3, 2, 32, dtype=dtype, device="cuda")
    q[:, :, 0] = 4.0
    out, logs = run_attend(q, cache, None, ints([99] * 3), 0, 1.0)
    for b, t in ((0, 0), (1, 57), (2, 99)):
        assert torch.equal(out[b, 0], cache.v[cell(b, t)][0]) and torch.equal(out[b, 1], cache.v[cell(b, t)][0])
    assert float((logs - 400).abs().max()) <= 400 * 2.0 ** -21
    cache.k.zero_()
    cache.k[:, :, :, 0] = -float("inf")
    out, logs = run_attend(q, cache, None, ints([99] * 3), 0, 1.0)
    assert bool((out == 0).all()) and bool((logs == -float("inf")).all())
    cache.k[cell(1, 70)][0, 0] = 1.0
    out, logs = run_attend(q, cache, None, ints([99] * 3), 0, 1.0)
    assert torch.equal(out[1, 1], cache.v[cell(1, 70)][0]) and bool((logs[1] == 4).all()) and bool((out[0] == 0).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("shift,pad", [(1, 0), (0, 8), (1, 1), (3, 5), (8, 8)])
def test_attend_strides_and_alignment(shift, pad, dtype):
    g = generator(15)
    for width in (64, 80, 128):
        cache = Cache([130, 40], 16, 2, width, dtype, "slot", g)
        q = torch.randn(2, 6, width, generator=g, device="cuda").to(dtype)
        want, logs = run_attend(q, cache, None, ints([129, 39]), 0, 0.1)
        k, v, qs = placed(cache.k, width + pad, shift)[1], placed(cache.v, width + pad, shift)[1], placed(q, width + pad, shift)[1]
        buffer, out = placed(torch.zeros_like(q), width + pad, shift)
        clean = buffer.clone()
        _, again = run_attend(qs, cache, None, ints([129, 39]), 0, 0.1, out=out, k=k, v=v)
        assert torch.equal(out, want) and torch.equal(again, logs)
        out.zero_()
        assert torch.equal(buffer, clean)


def test_attend_far_pages():
    """Pages more than 2^32 elements apart."""
    g, far = generator(16), 2 ** 32 + 24
    cache = Cache([40, 20], 32, 2, 64, torch.bfloat16, "slot", g, spare=0)
    assert cache.pages == 3
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    want, _ = run_attend(q, cache, None, ints([39, 19]), 0, 0.125)
    buffer = torch.empty(2 * far + 2 * 32 * 128, dtype=torch.bfloat16, device="cuda")
    k = buffer.as_strided(cache.k.shape, (far, 128, 64, 1))
    v = buffer.as_strided(cache.v.shape, (far, 128, 64, 1), 32 * 128)
    k.copy_(cache.k)
    v.copy_(cache.v)
    assert torch.equal(run_attend(q, cache, None, ints([39, 19]), 0, 0.125, k=k, v=v)[0], want)


def test_no_pages_and_no_requests():
    q = torch.ones(3, 2, 16, device="cuda")
    for requests, pages in ((3, 0), (0, 4)):
        tables, positions = torch.zeros(max(requests, 1), 2, dtype=torch.int32, device="cuda"), ints([5, 0, 31])
        k, out, logs = torch.ones(4, 16, 1, 16, device="cuda"), torch.full_like(q, 9), torch.full((3, 2), 9.0, device="cuda")
        space = cutt.cuttAttendPagesWorkspace(3, 2, 1, 16, 16, 2, 0)
        work = torch.empty(space + 4, dtype=torch.uint8, device="cuda")
        cache = k.data_ptr() if pages else 0
        ok(cutt.cuttAttendPages(3, requests, 2, 1, 16, cutt.CUTT_F32, pages, 16, 2, 0, 1.0, stream(), tables.data_ptr() if requests else 0, 0,
                                positions.data_ptr(), q.data_ptr(), (32, 16), cache, cache, (256, 16, 16), out.data_ptr(), (32, 16), logs.data_ptr(),
                                work.data_ptr(), space))
        assert bool((out == 0).all()) and bool((logs == -float("inf")).all())


def test_results_join_by_their_log_sums():
    """The first tokens of a request and the rest apart, joined, are the whole."""
    g = generator(17)
    cache = Cache([200], 20, 2, 64, torch.float32, "slot", g)
    q = torch.randn(1, 4, 64, generator=g, device="cuda")
    whole, logs = run_attend(q, cache, None, ints([199]), 0, 0.125)
    head, head_logs = run_attend(q, cache, None, ints([79]), 0, 0.125)
    rest, rest_logs = run_attend(q, cache, None, ints([199]), 120, 0.125)
    a, b = torch.exp(head_logs - logs)[..., None], torch.exp(rest_logs - logs)[..., None]
    assert float((a + b - 1).abs().max()) < 1e-5
    assert float((a * head + b * rest - whole).abs().max()) < 1e-5


# ---- as programs call them ---------------------------------------------------------
def step_of(dtype, seed):
    """A decoding step's calls on buffers of its own: (the calls, the results)."""
    g = generator(seed)
    cache = Cache([700, 3, 41, 0, 120], 16, 2, 64, dtype, "slot", g)
    q, positions = torch.randn(5, 8, 64, generator=g, device="cuda").to(dtype), ints([699, 2, 40, -1, 119])
    counts, inner, outer = [3, 0, 9, 1, 0, 70, 2], 128, 192
    rows, offsets = sum(counts), offsets_of(counts)
    x, w = torch.randn(rows, inner, generator=g, device="cuda").to(dtype), torch.randn(len(counts), inner, outer, generator=g, device="cuda").to(dtype)
    y, dx, dw = torch.zeros(rows, outer, dtype=dtype, device="cuda"), torch.zeros_like(x), torch.zeros_like(w)
    out, logs = torch.zeros_like(q), torch.zeros(5, 8, device="cuda")
    space = cutt.cuttAttendPagesWorkspace(5, 8, 2, 64, 16, cache.tables.shape[1], 0)
    workspace = torch.empty(space + 4, dtype=torch.uint8, device="cuda")

    def calls():
        ok(cutt.cuttAttendPages(5, 5, 8, 2, 64, CODE[dtype], cache.pages, 16, cache.tables.shape[1], 0, 0.125, stream(), cache.tables.data_ptr(), 0,
                                positions.data_ptr(), q.data_ptr(), q.stride()[:2], cache.k.data_ptr(), cache.v.data_ptr(), cache.k.stride()[:3], out.data_ptr(),
                                out.stride()[:2], logs.data_ptr(), workspace.data_ptr(), space))
        run_product(x, w, offsets, False, y)
        run_product(y, w, offsets, True, dx)
        run_weights(x, y, offsets, dw)

    return calls, [out, logs, y, dx, dw], [q, x, cache.k]


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_captured_and_replayed(dtype):
    """Two steps in graphs of their own, replayed in turn with new inputs: as the eager calls, bit by bit."""
    steps = [step_of(dtype, s) for s in (21, 22)]
    graphs = []
    for calls, _, _ in steps:
        calls()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            calls()
        graphs.append(graph)
    g = generator(23)
    for _ in range(4):
        for (calls, results, inputs), graph in zip(steps, graphs):
            for t in inputs:
                t.copy_(torch.randn(t.shape, generator=g, device="cuda").to(dtype))
            calls()
            want = [r.clone() for r in results]
            for r in results:
                r.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(results, want):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    """Two steps on streams of their own, with buffers of their own."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    steps = [step_of(torch.bfloat16, s) for s in (31, 32)]
    wants = []
    for calls, results, _ in steps:
        calls()
        wants.append([r.clone() for r in results])
    for _, results, _ in steps:
        for r in results:
            r.fill_(7)
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (calls, _, _) in zip(streams, steps):
            with torch.cuda.stream(s):
                calls()
    torch.cuda.synchronize()
    for (_, results, _), want in zip(steps, wants):
        for a, b in zip(results, want):
            assert torch.equal(a, b)


def test_a_step_of_all():
    """Prompts into empty pages, attention over them, and the rows to their experts, through these and back: captured, and replayed with other lengths and choices.
    Tolerance: a chain of ten operations of up to 512 terms in 32 bits, 10 * 512 * 2^-24 = 3e-4 of the largest value."""
    g = generator(41)
    tokens, requests, heads, key_heads, size, page, table, experts, choices, hidden = 60, 7, 6, 2, 32, 8, 9, 8, 3, 96
    width, kv = heads * size, key_heads * size

    def floats(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def zeros(*shape, dtype=torch.int32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    qkv, up, down = floats(tokens, width + 2 * kv), floats(experts, width, hidden) / width ** 0.5, floats(experts, width, hidden) / hidden ** 0.5
    added, owners, ids, weights = zeros(requests), zeros(tokens), zeros(tokens, choices, dtype=torch.int64), zeros(tokens, choices, dtype=torch.float32)
    pages = requests + tokens // page + 1
    lengths, free, tables = zeros(requests), torch.randperm(pages, generator=g, device="cuda").to(torch.int32), torch.full((requests, table), -1, dtype=torch.int32, device="cuda")
    starts, used, slots, positions = zeros(requests + 1), zeros(1), zeros(tokens, dtype=torch.int64), zeros(tokens)
    k, v = floats(pages, page, key_heads, size), floats(pages, page, key_heads, size)
    mixed, out = zeros(tokens, width, dtype=torch.float32), zeros(tokens, width, dtype=torch.float32)
    rows = cutt.cuttExpertRows(tokens, choices, experts, 4)
    counts, offsets, position, source = zeros(experts), zeros(experts + 1), zeros(tokens, choices), zeros(rows)
    x, inside, y = zeros(rows, width, dtype=torch.float32), zeros(rows, hidden, dtype=torch.float32), zeros(rows, width, dtype=torch.float32)
    sort_space = cutt.cuttExpertSortWorkspace(tokens, choices, experts)
    space = cutt.cuttAttendPagesWorkspace(tokens, heads, key_heads, size, page, table, 0)
    workspace = torch.empty(max(space, sort_space) + 4, dtype=torch.uint8, device="cuda")
    pitch, cache = qkv.stride(0), k.stride()[:3]

    def step():
        ok(cutt.cuttPageTables(requests, page, table, pages, tokens, stream(), lengths.data_ptr(), added.data_ptr(), free.data_ptr(), tables.data_ptr(),
                               starts.data_ptr(), used.data_ptr(), slots.data_ptr(), positions.data_ptr()))
        ok(cutt.cuttPageStore(tokens, key_heads, size, 4, pages, page, stream(), slots.data_ptr(), qkv[:, width:].data_ptr(), qkv[:, width + kv:].data_ptr(), (pitch, size),
                              k.data_ptr(), v.data_ptr(), cache))
        ok(cutt.cuttAttendPages(tokens, requests, heads, key_heads, size, cutt.CUTT_F32, pages, page, table, 0, size ** -0.5, stream(), tables.data_ptr(),
                                owners.data_ptr(), positions.data_ptr(), qkv.data_ptr(), (pitch, size), k.data_ptr(), v.data_ptr(), cache, mixed.data_ptr(),
                                (width, size), 0, workspace.data_ptr(), space))
        ok(cutt.cuttExpertSort(tokens, choices, 0, experts, 4, rows, 8, stream(), ids.data_ptr(), counts.data_ptr(), offsets.data_ptr(), position.data_ptr(),
                               source.data_ptr(), workspace.data_ptr(), sort_space))
        ok(cutt.cuttExpertDispatch(tokens, choices, rows, width, 4, stream(), position.data_ptr(), source.data_ptr(), mixed.data_ptr(), width, x.data_ptr(), width))
        run_product(x, up, offsets, False, inside)
        inside.tanh_()
        run_product(inside, down, offsets, True, y)
        ok(cutt.cuttExpertCombine(tokens, choices, rows, width, cutt.CUTT_F32, stream(), position.data_ptr(), weights.data_ptr(), y.data_ptr(), width, out.data_ptr(),
                                  width))

    def draw():
        cuts = torch.sort(torch.randperm(tokens + 1, generator=g, device="cuda")[:requests - 1])[0].tolist()
        share = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
        added.copy_(ints(share))
        owners.copy_(ints([b for b, n in enumerate(share) for _ in range(n)]))
        qkv.copy_(floats(*qkv.shape))
        ids.copy_(torch.topk(floats(tokens, experts), choices, dim=1)[1])
        weights.copy_(torch.softmax(floats(tokens, choices), dim=1))

    def plain():
        wide = qkv.double()
        q, keys, values = wide[:, :width].view(tokens, heads, size), wide[:, width:width + kv].view(tokens, key_heads, size), wide[:, width + kv:].view(tokens, key_heads, size)
        at = torch.arange(tokens, device="cuda")
        sees = (owners[:, None] == owners[None]) & (at[None] <= at[:, None])
        done = []
        for h in range(heads):
            score = (q[:, h] @ keys[:, h // (heads // key_heads)].t().contiguous() * size ** -0.5).masked_fill(~sees, float("-inf"))
            done.append(torch.softmax(score, dim=1) @ values[:, h // (heads // key_heads)].contiguous())
        one = torch.cat(done, dim=1)
        two = torch.zeros_like(one)
        for c in range(choices):
            for e in range(experts):
                mine = ids[:, c] == e
                two[mine] += weights[mine, c, None].double() * (torch.tanh(one[mine] @ up[e].double()) @ down[e].double().t().contiguous())
        return one, two

    draw()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        draw()
        step()
        eager = [mixed.clone(), out.clone()]
        for got, want in zip(eager, plain()):
            assert float((got - want).abs().max()) <= 3e-4 * float(want.abs().max())
        mixed.fill_(7), out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(mixed, eager[0]) and torch.equal(out, eager[1])
