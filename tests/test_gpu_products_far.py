"""Products and gradients of more tiles than a launch has workgroups, where a workgroup makes a second tile in the same LDS, and of operands beyond 1 GiB.  Small whole
numbers, whose sums are exact."""
import pytest
import torch

from test_gpu_products import generator, made, offsets_of, run_product, run_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("outer", [2 ** 25, 2 ** 25 + 1])
def test_second_tiles_of_a_product(outer):
    """20 groups of a row, 2^18 and more strips of columns each; the weights are one group's, which all share."""
    g, groups, inner = generator(1), 20, 8
    x, w = made((groups, inner), torch.bfloat16, True, g), torch.empty(inner, outer, dtype=torch.bfloat16, device="cuda")
    for line in w:
        line.copy_(made((outer,), torch.bfloat16, True, g))
    y = torch.full((groups, outer), 77, dtype=torch.bfloat16, device="cuda")
    run_product(x, w[None].expand(groups, inner, outer), offsets_of([1] * groups), False, y)
    for e in range(groups):
        want = torch.zeros(outer, device="cuda")
        for i in range(inner):
            want += x[e, i].float() * w[i].float()
        assert torch.equal(y[e], want.bfloat16()), e


@pytest.mark.parametrize("transposed", [False, True])
def test_second_tiles_by_rows(transposed):
    """Ten rows to a group in the mean, some groups in two tiles, 4096 strips; the same weights for all."""
    g, groups, inner, outer = generator(2), 1024, 8, 2 ** 19
    counts = [70 if i % 40 == 39 else 9 for i in range(groups)]
    x = made((sum(counts), inner), torch.float16, True, g)
    w = made((outer, inner) if transposed else (inner, outer), torch.float16, True, g)
    y = torch.full((sum(counts), outer), 77, dtype=torch.float16, device="cuda")
    run_product(x, w[None].expand(groups, *w.shape), offsets_of(counts), transposed, y)
    m = (w.t() if transposed else w).float().contiguous()
    for at in range(0, sum(counts), 1024):
        assert torch.equal(y[at:at + 1024], (x[at:at + 1024].float() @ m).half()), at


@pytest.mark.parametrize("outer", [2 ** 19 + 128, 2 ** 19 + 129])
def test_second_tiles_of_a_gradient(outer):
    """1024 groups of three rows and fewer, 4097 strips each."""
    g, groups, inner = generator(3), 1024, 8
    counts = [e % 4 for e in range(groups)]
    x, dy = made((sum(counts), inner), torch.bfloat16, True, g), made((sum(counts), outer), torch.bfloat16, True, g)
    dw = torch.full((groups, inner, outer), 77, dtype=torch.bfloat16, device="cuda")
    run_weights(x, dy, offsets_of(counts), dw)
    at = 0
    for e, n in enumerate(counts):
        want = torch.zeros(inner, outer, device="cuda")
        for r in range(at, at + n):
            want += x[r].float()[:, None] * dy[r].float()[None]
        at += n
        assert torch.equal(dw[e], want.bfloat16()), e


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bfloat16", "float32"])
def test_gradient_of_rows_around_a_gigabyte(dtype):
    """An operand's rows from just below 2^30 bytes on to just above them: the same results."""
    g, counts, inner, outer = generator(4), [300, 0, 613, 111], 72, 136
    rows, offsets = sum(counts), offsets_of(counts)
    x, dy = made((rows, inner), dtype, True, g), made((rows, outer), dtype, True, g)
    want = run_weights(x, dy, offsets, torch.empty(len(counts), inner, outer, dtype=dtype, device="cuda"))
    at = 0
    for e, n in enumerate(counts):
        assert torch.equal(want[e], (x[at:at + n].float().t().contiguous() @ dy[at:at + n].float()).to(dtype))
        at += n
    size = torch.finfo(dtype).bits // 8
    even = 2 ** 30 // size // rows // 8 * 8
    buffer = torch.full(((even + 64) * rows,), float("nan"), dtype=dtype, device="cuda")
    for pitch in (even - 8, even, even + 8, even + 64):
        far = buffer.as_strided((rows, inner), (pitch, 1))
        far.copy_(x)
        assert torch.equal(run_weights(far, dy, offsets, torch.empty_like(want)), want)
        far = buffer.as_strided((rows, outer), (pitch, 1))
        far.copy_(dy)
        assert torch.equal(run_weights(x, far, offsets, torch.empty_like(want)), want)
