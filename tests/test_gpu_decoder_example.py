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
