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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hidden", [12, 64])
def test_fused_linear_log_probs_off_the_kernels_form_their_logits_in_32_bits(dtype, hidden):
    gen = torch.Generator().manual_seed(hidden)
    x, w = (torch.randn(n, hidden, generator=gen).to(dtype) for n in (20, 300))
    labels = torch.randint(0, 300, (20,), generator=gen)
    labels[5] = -100
    x.requires_grad_(True), w.requires_grad_(True)
    lp, entropy = ops.fused_linear_token_log_probs(x, w, labels, return_entropy=True)
    dx, dw = torch.autograd.grad(lp.sum(), (x, w))
    x64, w64 = x.detach().double(), w.detach().double()
    logp = (x64 @ w64.t()).log_softmax(-1)
    want = torch.where(labels < 0, 0.0, logp.gather(1, labels.clamp_min(0)[:, None])[:, 0])
    # `hidden` products and additions and at most 300 terms of the softmax, each rounded to fp32, of logits below 64
    bound = (hidden + 300 + 16) * 2.0**-24 * (1 + (x64.abs() @ w64.abs().t()).max())
    assert lp.dtype == torch.float32 and ((lp.double() - want).abs() <= bound).all() and torch.isfinite(entropy).all()
    dz = -logp.exp()
    dz[torch.arange(20), labels.clamp_min(0)] += 1
    dz[labels < 0] = 0
    half = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[dtype]
    for got, exact, size in ((dx, dz @ w64, dz.abs() @ w64.abs()), (dw, dz.t() @ x64, dz.abs().t() @ x64.abs())):
        assert got.dtype == dtype and ((got.double() - exact).abs() <= half * exact.abs() + 4 * bound * size + 2.0**-24).all()
    assert (dx[5] == 0).all()


def test_followers_of_the_timeline_are_told_of_its_switches(monkeypatch):
    from lm_engine.ops import timeline

    monkeypatch.setattr(timeline, "_FOLLOWERS", [])
    monkeypatch.setattr(timeline, "_TIMING", False)
    monkeypatch.setattr(timeline, "_NVTX", False)
    told = []
    timeline.follow(told.append)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    timeline.enable_timing()
    timeline.enable_nvtx()
    timeline.enable_timing(False)
    timeline.enable_nvtx(False)
    assert told == [None, timeline.site, timeline.site, timeline.site, None]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    timeline.enable_timing()  # nothing to time here
    assert told[-1] is None
