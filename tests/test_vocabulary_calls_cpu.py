"""Calls of the vocabulary operators that their documentation allows and that are out of the ordinary, where no GPU is needed."""

import math

import pytest
import torch

from lm_engine import ops


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_ignored_rows_are_in_no_product_of_the_fused_linear_log_probs(dtype):
    gen = torch.Generator().manual_seed(0)
    x, w = (torch.randn(n, 12, generator=gen).to(dtype) for n in (6, 40))
    labels = torch.tensor([3, -100, 39, 40, 0, -1])
    ignored = (labels < 0) | (labels >= 40)
    results = []
    for junk in (0.0, math.nan, math.inf):
        x[ignored] = junk
        a, b = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
        outs = ops.fused_linear_token_log_probs(a, b, labels, return_entropy=True)
        results.append((*outs, *torch.autograd.grad(outs[0].sum() + outs[1].sum(), (a, b))))
    for result in results:
        for got, want in zip(result, results[0]):
            assert torch.isfinite(got).all() and torch.equal(got, want)
    assert (results[0][2][ignored] == 0).all() and results[0][3].abs().max() > 0
