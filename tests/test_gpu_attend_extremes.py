"""Attention over pages where scores or values are infinite, and where weights are small, against the definition in 64 bits.

Tolerances as for the products' other tests: a score is off by d = (width + 4) * 2^-23 times its terms' sizes, an exponential by that relative to itself and a few steps, numerator
and denominator alike, and the result by half a step of its type.  Terms and sizes are those of the finite tokens: the others have the weight 0, or make their element infinite."""
import numpy as np
import pytest
import torch

import cutt_amd as cutt
import product_oracle as oracle
from test_gpu_products import CODE, HALF, LEAST, TYPES, UNIT, Cache, generator, ids_of, ints, np64, run_attend

pytestmark = pytest.mark.gpu

INF = float("inf")
# What a weight can be off by: 16-bit types keep an exponential in two parts.  Half's smallest step is 2^-24, and the largest exponential is 2^15 at least.
PART = {torch.float32: 0.0, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}
FLOOR = {torch.float32: 0.0, torch.float16: 2.0 ** -40, torch.bfloat16: 0.0}


def tolerance(want, size, terms, count, most, width, dtype):
    """Of out, and of the log sums without what is relative to these."""
    score, n = terms * (width + 4) * UNIT + 8 * UNIT, count[:, None]
    out = size * (2 * np.expm1(2 * score) + (2 * n + 40) * UNIT + PART[dtype])[:, :, None] + n[:, :, None] * most * FLOOR[dtype] + np.abs(want) * HALF[dtype] * 1.01 + LEAST[dtype]
    return out, 2 * score + (n + 10) * UNIT


def check(q, cache, owners, positions, window, scale, out, logs):
    """Keys of infinity or the lowest value count as 1e30, whose scores' exponentials are 0 in 64 bits; a query with no others sees nothing that counts."""
    who = np.arange(q.shape[0]) if owners is None else owners.cpu().numpy()
    rest = (cache.tables.cpu().numpy(), who, positions.cpu().numpy(), window, scale)
    k, v = np64(cache.k), np64(cache.v)
    far = np.abs(k) > 1e30
    with np.errstate(all="ignore"):
        want, want_logs, size, _, count, most = oracle.attend(np64(q), np.where(far, np.sign(k) * 1e30, k), v, *rest)
        terms = oracle.attend(np64(q), np.where(far, 0, k), np.zeros(v.shape), *rest)[3]
        off, off_logs = tolerance(want, size, terms, count, most, q.shape[2], q.dtype)
        out, logs = np64(out), np64(logs)
        none = want_logs < -1e25
        want[none] = 0
        odd = ~np.isfinite(want)
        wrong = np.isfinite(out) == odd
        assert not wrong.any(), (np.argwhere(wrong)[:5], out[wrong][:5], want[wrong][:5])
        assert np.array_equal(out[odd], want[odd], equal_nan=True)
        bad = ~odd & ~(np.abs(out - want) <= off)
        assert not bad.any(), (int(bad.sum()), out[bad][:5], want[bad][:5], off[bad][:5])
        assert np.array_equal(np.isneginf(logs), none)
        bad = ~none & ~(np.abs(logs - want_logs) <= off_logs + 4 * np.abs(np.where(none, 0, want_logs)) * UNIT)
        assert not bad.any(), (logs[bad][:5], want_logs[bad][:5])


def cell(cache, b, t):
    """The page and slot of request b's token t."""
    return int(cache.tables[b, t // cache.page]), t % cache.page


# Requests of one and two tiles and their edges; cut into ranges; drafted tokens whose windows end within tiles.
FORMS = {
    "short": ([1, 16, 33, 100, 256], 1, 0),
    "long": ([6000, 40], 1, 0),
    "drafts": ([90, 300, 31], 3, 50),
}


def form(name, dtype, width, key_heads=2, shared=2, seed=51):
    lengths, drafts, window = FORMS[name]
    g = generator(seed)
    cache = Cache(lengths, 16, key_heads, width, dtype, "slot", g)
    owners = ints([b for b in range(len(lengths)) for _ in range(drafts)])
    positions = ints([n - drafts + i for n in lengths for i in range(drafts)])
    q = torch.randn(len(lengths) * drafts, key_heads * shared, width, generator=g, device="cuda").to(dtype)
    return cache, q, owners, positions, window, lengths, g


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("width,scale", [(32, 32 ** -0.5), (64, 64 ** -0.5), (96, 96 ** -0.5), (128, 128 ** -0.5), (64, 0.1), (64, 0.2), (64, 0.3), (80, 1.0), (256, -0.1),
                                         (40, -0.3)])
def test_scores_of_minus_infinity(width, scale, name, dtype):
    """Tokens with a score of -infinity, every third one, count nothing, whatever the scale's rounding; where there are no others, zeros and -infinity."""
    cache, q, owners, positions, window, lengths, g = form(name, dtype, width)
    q[:, :, 0] = 4.0
    low = -INF if scale > 0 else INF
    for b, n in enumerate(lengths):
        for t in range(0, n, 3):
            cache.k[cell(cache, b, t)][:, 0] = low
    out, logs = run_attend(q, cache, owners, positions, window, scale)
    check(q, cache, owners, positions, window, scale, out, logs)
    cache.k[..., 0] = low
    out, logs = run_attend(q, cache, owners, positions, window, scale)
    assert bool((out == 0).all()) and bool((logs == -INF).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [128 ** -0.5, 0.1, 0.3])
def test_keys_of_the_lowest_value(scale, dtype):
    """Their scores leave the range of 32 bits."""
    cache, q, owners, positions, window, lengths, g = form("short", dtype, 128)
    q[:, :, 0] = 4.0
    for b, n in enumerate(lengths):
        for t in range(0, n - 1, 2):
            cache.k[cell(cache, b, t)][:, 0] = torch.finfo(dtype).min
    out, logs = run_attend(q, cache, owners, positions, window, scale)
    check(q, cache, owners, positions, window, scale, out, logs)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("scale", [3.4e38, -3.4e38, 2.5e38])
def test_largest_scales(scale, dtype):
    """Scales whose product with log2 e leaves the range of 32 bits: scores of 0 stay 0, and one that is higher takes all of the weight."""
    cache, q, owners, positions, window, lengths, g = form("short", dtype, 64)
    q.zero_()
    out, logs = run_attend(q, cache, owners, positions, window, scale)
    check(q, cache, owners, positions, window, scale, out, logs)
    q[:, :, 0] = 2.0 ** -24
    cache.k.zero_()
    for b, n in enumerate(lengths):
        cache.k[cell(cache, b, n // 2)][:, 0] = -2.0 ** -20 if scale < 0 else 2.0 ** -20
    out, logs = run_attend(q, cache, owners, positions, window, scale)
    assert float((logs / (abs(scale) * 2.0 ** -44) - 1).abs().max()) <= 2.0 ** -20
    for i, b in enumerate(owners.tolist()):
        v = cache.v[cell(cache, b, lengths[b] // 2)]
        for h in range(4):
            assert torch.equal(out[i, h], v[h // 2])


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("name", FORMS)
def test_scores_of_plus_infinity(name, dtype):
    """A score of +infinity: the log sum is +infinity, and out, infinity over infinity, is no number; other heads are as without it.  A score that is no number: neither."""
    cache, q, owners, positions, window, lengths, g = form(name, dtype, 64)
    want, want_logs = run_attend(q, cache, owners, positions, window, 0.125)
    for bad in (INF, float("nan")):
        other = Cache.__new__(Cache)
        other.__dict__.update(cache.__dict__, k=cache.k.clone())
        other.k[cell(cache, 0, lengths[0] - 1 if len(owners) == len(lengths) else lengths[0] - 3)][1, 5] = bad
        out, logs = run_attend(q, other, owners, positions, window, 0.125)
        for i, b in enumerate(owners.tolist()):
            for h in range(4):
                score = float(q[i, h, 5]) * bad
                if b or h < 2:
                    assert torch.equal(out[i, h], want[i, h]) and torch.equal(logs[i, h], want_logs[i, h])
                elif score != -INF:
                    assert bool(out[i, h].isnan().all())
                    assert float(logs[i, h]) == INF if score == INF else bool(logs[i, h].isnan())


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("width,key_heads", [(64, 2), (128, 2), (200, 1), (77, 2)])
@pytest.mark.parametrize("name", FORMS)
def test_infinite_values(name, width, key_heads, dtype):
    """Infinities in values that are seen make their element infinite, one of either sign or NaN make it no number; all other elements are as they were."""
    cache, q, owners, positions, window, lengths, g = form(name, dtype, width, key_heads)
    for b, n in enumerate(lengths):
        for d, (t, x) in enumerate([(0, INF), (n // 2, -INF), (n - 1, INF), (n // 3, float("nan")), (n // 2, INF), (min(n - 1, 20), -INF), (max(n - 40, 0), INF)]):
            cache.v[cell(cache, b, t)][:, 3 * d + 1] = x
        for t, x in ((n // 3, INF), (n - 1, -INF)):
            cache.v[cell(cache, b, t)][:, 40 + (n == 1)] = x
    out, logs = run_attend(q, cache, owners, positions, window, 0.125)
    check(q, cache, owners, positions, window, 0.125, out, logs)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("queries", [1, 2, 5])
def test_infinite_values_at_the_end_of_cut_queries(queries, dtype):
    """Where the last part of a query's tokens, and of every other part too, holds infinities: as many parts as there are, none of them counts twice or as nothing."""
    for longest in (1000, 2100, 2900, 5000):
        g = generator(61)
        cache = Cache([longest - 100 * i for i in range(queries)], 16, 1, 64, dtype, "slot", g)
        q = torch.randn(queries, 2, 64, generator=g, device="cuda").to(dtype)
        positions = ints([longest - 100 * i - 1 for i in range(queries)])
        for b in range(queries):
            n = longest - 100 * b
            for d in range(8):
                cache.v[cell(cache, b, (n - 1) * d // 7)][0, d] = INF
            cache.v[cell(cache, b, n - 1)][0, 9] = -INF
        out, logs = run_attend(q, cache, None, positions, 0, 0.125)
        check(q, cache, None, positions, 0, 0.125, out, logs)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("below", [15.0, 30.0, 60.0, 80.0])
def test_infinite_values_of_small_weights(below, dtype):
    """As long as a weight is a number of 32 bits above 0, an infinity times it is one, whatever 16 bits would make of the weight."""
    cache, q, owners, positions, window, lengths, g = form("short", dtype, 64, 1)
    cache.k.zero_()
    q.zero_()
    q[:, :, 0] = 1.0
    for b, n in enumerate(lengths):
        cache.k[cell(cache, b, n // 2)][:, 0] = below
        for t in range(0, n, 7):
            cache.v[cell(cache, b, t)][:, t % 60] = INF if t % 2 else -INF
    out, logs = run_attend(q, cache, owners, positions, window, 1.0)
    check(q, cache, owners, positions, window, 1.0, out, logs)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("key_heads,requests", [(1, 1), (4, 3), (2, 140)])
@pytest.mark.parametrize("below", [6.0, 10.0, 14.0, 18.0, 20.0])
def test_long_tails_of_small_weights(below, key_heads, requests, dtype):
    """One token of value 0 that outweighs each of 4095 others by e^below: these are all there is in the result."""
    g, n = generator(71), 4096 if requests < 100 else 700
    cache = Cache([n] * requests, 64, key_heads, 64, dtype, "slot", g)
    cache.k.zero_()
    cache.v.uniform_(20000, 60000, generator=g)
    q = torch.zeros(requests, 2 * key_heads, 64, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    for b in range(requests):
        at = cell(cache, b, (b * 997 + 5) % n)
        cache.k[at][:, 0] = below
        cache.v[at] = 0
    positions = ints([n - 1] * requests)
    out, logs = run_attend(q, cache, None, positions, 0, 1.0)
    check(q, cache, None, positions, 0, 1.0, out, logs)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("name", FORMS)
def test_results_beside_queries(name, dtype):
    """Queries and results in the columns of one buffer, as a fused projection leaves them: results as into a buffer of their own, everything else as it was."""
    cache, q, owners, positions, window, lengths, g = form(name, dtype, 64)
    queries, heads, width = q.shape
    want, want_logs = run_attend(q, cache, owners, positions, window, 0.125)
    rows = torch.full((queries, 3 * heads, width), 5.0, dtype=dtype, device="cuda")
    rows[:, :heads] = q
    out, logs = run_attend(rows[:, :heads], cache, owners, positions, window, 0.125, out=rows[:, heads:2 * heads])
    assert torch.equal(out, want) and torch.equal(logs, want_logs)
    assert torch.equal(rows[:, :heads], q) and bool((rows[:, 2 * heads:] == 5).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("requests,longest,heads,key_heads,width", [(256, 4500, 16, 1, 64), (2, 55000, 16, 16, 32)])
def test_infinite_values_of_long_parts(requests, longest, heads, key_heads, width, dtype):
    """Workgroups whose parts have more tokens than they work out addresses for at a time, one of them without an infinity; others take many queries one after the other."""
    g = generator(81)
    lengths = [5] * requests
    lengths[0], lengths[requests // 2] = longest, longest // 2 + 77
    cache = Cache(lengths, 32, key_heads, width, dtype, "head", g)
    q = torch.randn(requests, heads, width, generator=g, device="cuda").to(dtype)
    for b, n in ((0, longest), (requests - 1, lengths[-1])):
        for d, t in enumerate((0, 1200, n // 2, n - 1, n - 1030)):
            if 0 <= t < n:
                cache.v[cell(cache, b, t)][:, 2 * d] = INF if d % 2 else -INF
    positions = ints([n - 1 for n in lengths])
    out, logs = run_attend(q, cache, None, positions, 0, width ** -0.5)
    check(q, cache, None, positions, 0, width ** -0.5, out, logs)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=ids_of[1:])
def test_queries_without_numbers(dtype):
    """A query of NaN gets NaN, whatever infinities its tokens have; the others of its request are as without it."""
    cache, q, owners, positions, window, lengths, g = form("drafts", dtype, 64)
    cache.v[cell(cache, 0, lengths[0] - 3)][:, 7] = INF
    want, want_logs = run_attend(q, cache, owners, positions, window, 0.125)
    assert bool((want[:3, :, 7] == INF).all())
    q[1] = float("nan")
    out, logs = run_attend(q, cache, owners, positions, window, 0.125)
    assert bool(out[1].isnan().all()) and bool(logs[1].isnan().all())
    others = [i for i in range(len(owners)) if i != 1]
    assert torch.equal(out[others], want[others]) and torch.equal(logs[others], want_logs[others])


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_infinities_that_come_and_go_between_replays(dtype):
    """A captured call whose cache gets infinite values and loses them: every replay as the eager call, bit by bit."""
    cache, q, owners, positions, window, lengths, g = form("long", dtype, 64)
    out, logs = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    queries, heads, width = q.shape
    space = cutt.cuttAttendPagesWorkspace(queries, heads, 2, width, cache.page, cache.tables.shape[1], window)
    work = torch.empty(space, dtype=torch.uint8, device="cuda")

    def call():
        assert cutt.cuttAttendPages(queries, len(lengths), heads, 2, width, CODE[dtype], cache.pages, cache.page, cache.tables.shape[1], window, 0.125,
                                    torch.cuda.current_stream().cuda_stream, cache.tables.data_ptr(), owners.data_ptr(), positions.data_ptr(), q.data_ptr(),
                                    q.stride()[:2], cache.k.data_ptr(), cache.v.data_ptr(), cache.k.stride()[:3], out.data_ptr(), out.stride()[:2], logs.data_ptr(),
                                    work.data_ptr(), space) == cutt.CUTT_SUCCESS

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    clean = cache.v.clone()
    for turn in range(5):
        cache.v.copy_(clean)
        if turn % 2:
            cache.v[cell(cache, 0, 1000 * turn)][:, 11] = INF
            cache.v[cell(cache, 1, 39)][:, 12] = -INF
        call()
        want, want_logs = out.clone(), logs.clone()
        out.fill_(7), logs.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(9), want.nan_to_num(9)) and torch.equal(logs, want_logs)
        assert bool((out[0, :, 11] == INF).all()) == bool(turn % 2) and not bool(out.isnan().any())
