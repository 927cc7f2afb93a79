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


@pytest.mark.parametrize("packed", [True, False])
def test_masks_are_shifted_like_the_log_probs_of_a_model(packed):
    """The documented use: position t holds token t + 1, so a mask of answer tokens moves one position to the left and is off at last positions."""
    from lm_engine.hf_models import get_token_log_probs

    gen = torch.Generator().manual_seed(0)
    lengths, vocab = [5, 5, 5, 5], 11
    logits = torch.randn(20, vocab, generator=gen, dtype=torch.float64)
    tokens = torch.randint(0, vocab, (20,), generator=gen)
    answer_tokens = torch.tensor([0, 0, 1, 1, 1] + [0, 1, 1, 0, 0] + [1, 0, 0, 1, 1] + [0, 0, 0, 0, 1]).bool()
    cu = torch.tensor([0, 5, 10, 15, 20])
    if packed:
        lp = get_token_log_probs(logits, tokens, cu_seqlens=cu, use_padding_free_transformer=True)
        mask = answer_tokens.roll(-1)
        mask[cu[1:].long() - 1] = False
    else:
        logits, tokens, answer_tokens, cu = logits.view(4, 5, vocab), tokens.view(4, 5), answer_tokens.view(4, 5), None
        lp = get_token_log_probs(logits, tokens)
        mask = answer_tokens.roll(-1, 1)
        mask[:, -1] = False
    old, reference = lp - 0.1 * torch.randn(lp.shape, generator=gen), lp + 0.1 * torch.randn(lp.shape, generator=gen)
    advantages = torch.tensor([1.0, -0.5, 2.0, -1.5], dtype=torch.float64)

    logp = logits.reshape(4, 5, vocab).log_softmax(-1)
    old4, ref4, answer4, token4 = old.view(4, 5), reference.view(4, 5), answer_tokens.view(4, 5), tokens.view(4, 5)
    values, sums = [], []
    for i in range(4):
        # a token is predicted one position earlier; the first token of a document is predicted by nothing
        own = [(logp[i, t - 1, token4[i, t]], old4[i, t - 1], ref4[i, t - 1]) for t in range(1, 5) if answer4[i, t]]
        values.append([max(-advantages[i] * (a - b).exp(), -advantages[i] * (a - b).exp().clamp(0.8, 1.2)).item() for a, b, _ in own])
        sums.append(sum((a - r).item() for a, _, r in own) / len(own))
    token_mean = sum(map(sum, values)) / sum(map(len, values))
    sequence_mean = sum(sum(v) / len(v) for v in values) / 4
    for reduction, want in (("token_mean", token_mean), ("sequence_mean", sequence_mean)):
        got = ops.policy_loss(lp, old, advantages, cu_seqlens=cu, mask=mask, reduction=reduction).loss.item()
        assert got == pytest.approx(want, rel=1e-12)
        unshifted = ops.policy_loss(lp, old, advantages, cu_seqlens=cu, mask=answer_tokens, reduction=reduction).loss.item()
        assert abs(unshifted - want) > 1e-3
    got = ops.preference_loss(lp, reference, cu, beta=0.5, average_log_probs=True, mask=mask).loss.item()
    assert got == pytest.approx(sum(math.log1p(math.exp(-0.5 * (sums[i] - sums[i + 2]))) for i in range(2)) / 2, rel=1e-12)
