"""Calls of the vocabulary operators that their documentation allows and that are out of the ordinary: empty operands, operands that start or
end oddly, values changed between the passes, switches of the process."""

import math

import pytest
import torch

from lm_engine import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _healthy():
    yield
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab,tokens,hidden", [(0, 0, 16), (0, 0, 3), (5, 0, 16), (5, 3, 0), (0, 0, 0)])
def test_embedding_of_nothing(dtype, vocab, tokens, hidden):
    w = torch.zeros(vocab, hidden, device="cuda", dtype=dtype, requires_grad=True)
    out = ops.embedding(w, torch.zeros(tokens, device="cuda", dtype=torch.long), sorted_gradient=True)
    (grad,) = torch.autograd.grad(out.sum(), w)
    assert out.shape == (tokens, hidden) and grad.shape == w.shape and (grad == 0).all()
    w.main_grad = torch.ones(vocab, hidden, device="cuda")
    ops.embedding(w, torch.zeros(tokens, device="cuda", dtype=torch.long), sorted_gradient=True).sum().backward()
    assert (w.main_grad == 1).all()
