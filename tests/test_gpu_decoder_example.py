"""The decoder layer of examples/decoder_layer.py: what the row operators compute together is what plain torch operations do.

Tolerances: 32-bit products and softmax in another order of summation; a chain of about ten operations of up to 512 terms each
stays within 10 * 512 * 2^-24 = 3e-4 of the largest value.  Gradients in norm: the same chain, 3e-4; in bfloat16, a few roundings of 2^-8 per value that
are independent, below 2^-5."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import decoder_layer  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompts,page", [((37, 1, 64, 0, 5), 16), ((3,), 4), ((0, 0, 17), 1), ((20, 33), 64)])
def test_serving(prompts, page):
    worst, biggest = decoder_layer.serve(prompts=prompts, page=page)
    assert worst <= 3e-4 * biggest


@pytest.mark.parametrize("experts,choices,tokens", [(8, 3, 100), (1, 1, 5), (16, 16, 33), (4, 2, 1)])
def test_gradients(experts, choices, tokens):
    assert decoder_layer.train(experts=experts, choices=choices, tokens=tokens) <= 3e-4


def test_gradients_in_bfloat16():
    assert decoder_layer.train(dtype=torch.bfloat16) <= 2.0 ** -5


@pytest.mark.parametrize("experts,choices,tokens", [(8, 3, 100), (1, 1, 5), (16, 16, 33), (4, 2, 1)])
def test_second_derivatives(experts, choices, tokens):
    """Through the gradients once more: twice the chain."""
    assert decoder_layer.train(experts=experts, choices=choices, tokens=tokens, second=True) <= 6e-4


@pytest.mark.parametrize("of_rows,of_weights", [(True, False), (False, True), (True, True)])
def test_one_gradient_of_combine(of_rows, of_weights):
    """Rows and weights that are not contiguous, one of them or both with a gradient; small whole numbers, so that every sum is exact."""
    g = torch.Generator(device="cuda")
    g.manual_seed(2)

    def whole(*shape):
        return torch.randint(-4, 5, shape, generator=g, device="cuda").float()

    routing = decoder_layer.Routing(torch.randint(0, 4, (9, 2), generator=g, device="cuda"), 4, 4)
    rows, weights, dout = whole(16, routing.rows).requires_grad_(of_rows), whole(2, 9).requires_grad_(of_weights), whole(9, 16)
    leaves = [t for t in (rows, weights) if t.requires_grad]
    at = routing.position.long()
    assert int(at.min()) >= 0
    got = torch.autograd.grad((decoder_layer.Combine.apply(rows.t(), weights.t(), routing) * dout).sum(), leaves)
    want = torch.autograd.grad(((rows.t()[at] * weights.t()[:, :, None]).sum(1) * dout).sum(), leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
