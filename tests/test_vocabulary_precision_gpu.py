"""Values of the vocabulary operators where a rounding could be lost: labels at the type's lowest value, rows far from zero, tokens that
are all but certain, long sums. Each bound counts the roundings of the definition (half a step of the type each)."""

import math

import pytest
import torch

from lm_engine import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _healthy():
    yield
    ops.check_status()


# ----------------------------------------------------------------------------- labels of the lowest value
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1.0, 0.75])
def test_a_label_of_the_types_lowest_value_keeps_a_finite_log_probability(dtype, scale):
    lowest = torch.finfo(dtype).min
    logits = torch.randn(5, 1000, generator=torch.Generator("cuda").manual_seed(0), device="cuda").to(dtype)
    labels = torch.tensor([3, 999, 0, 500, -100], device="cuda")
    logits[torch.arange(3), labels[:3]] = lowest
    logits.requires_grad_(True)
    lp, entropy = ops.token_log_probs(logits, labels, logit_scale=scale, return_entropy=True)
    want = (scale * logits.detach().double()).log_softmax(-1)
    # x - m and the scaled difference are rounded once each; the log-sum-exp is nothing next to 1e4
    assert ((lp[:3].double() - want[torch.arange(3), labels[:3]]).abs() <= 2 * 2.0**-24 * scale * abs(lowest) + 1e-5).all() and torch.isfinite(lp).all()
    assert torch.isfinite(entropy).all()
    # two passes that score the token alike have a ratio of 1, in both losses
    advantages = torch.ones(1, device="cuda")
    assert ops.policy_loss(lp[None], lp.detach()[None], advantages).loss.item() == -1.0
    pair = torch.stack([lp[:2], lp[1:3]])
    assert ops.preference_loss(pair, pair.detach()).loss.item() == pytest.approx(math.log(2), rel=2.0**-23)
    (grad,) = torch.autograd.grad(lp.sum() + entropy.sum(), logits)
    assert torch.isfinite(grad).all()


@pytest.mark.parametrize("keep", [None, True, False])
def test_a_label_of_the_lowest_value_from_hidden_states(keep):
    lowest = torch.finfo(torch.bfloat16).min
    x = torch.zeros(2, 8, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1.0
    w = torch.zeros(300, 8, device="cuda", dtype=torch.bfloat16)
    w[7, 0], w[290, 0] = lowest, lowest
    labels = torch.tensor([7, 290], device="cuda")
    if keep is not None:
        x.requires_grad_(True)
    lp = ops.fused_linear_token_log_probs(x, w, labels, keep_logits=keep)
    assert (lp.double() == lowest).all()  # log 298 is nothing next to it
    if keep is not None:
        (dx,) = torch.autograd.grad(lp.sum(), x)
        assert torch.isfinite(dx[:, 1:]).all()
