"""Vocabulary operators on the CPU: the PyTorch restatements against the definitions, gradients against differences, and refusals."""

import math

import pytest
import torch

from lm_engine import ops


def _definition(z, labels, ignore_index=-100):
    """Log-probabilities and entropies row by row in 64 bits, from the definition."""
    lps, ents = [], []
    for row, y in zip(z.double(), labels.tolist()):
        if y == ignore_index or not 0 <= y < z.shape[-1]:
            lps.append(0.0)
            ents.append(0.0)
            continue
        p = torch.exp(row - row.max())
        p = p / p.sum()
        lps.append(math.log(p[y]) if p[y] > 0 else -math.inf)
        ents.append(-sum(q * math.log(q) for q in p.tolist() if q > 0))
    return torch.tensor(lps, dtype=torch.float64), torch.tensor(ents, dtype=torch.float64)


@pytest.mark.parametrize("vocab", [1, 2, 33])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_log_probs_follow_the_definition(vocab, dtype):
    gen = torch.Generator().manual_seed(vocab)
    logits = (3 * torch.randn(9, vocab, generator=gen)).to(dtype)
    labels = torch.randint(0, vocab, (9,), generator=gen)
    labels[2], labels[5], labels[6] = -100, vocab, -1
    lp, ent = ops.token_log_probs(logits, labels, logit_scale=0.5, return_entropy=True)
    want_lp, want_ent = _definition(0.5 * logits.float(), labels)
    assert lp.dtype == ent.dtype == torch.float32 and lp.shape == labels.shape
    # fp32 softmax of at most 33 terms of size below 8: a few dozen roundings of 2^-24 relative to 8
    assert (lp - want_lp).abs().max() < 64 * 8 * 2.0**-24 and (ent - want_ent).abs().max() < 64 * 8 * 2.0**-24


def test_token_log_probs_gradients_and_masked_rows():
    gen = torch.Generator().manual_seed(0)
    logits = torch.randn(2, 4, 11, dtype=torch.float64, generator=gen, requires_grad=True)
    labels = torch.randint(0, 11, (2, 4), generator=gen)
    labels[0, 1] = 7
    fn = lambda z: ops.token_log_probs(z, labels, logit_scale=1.3, ignore_index=7, return_entropy=True)
    assert torch.autograd.gradcheck(fn, (logits,))
    # a row that is ignored may hold anything, and -inf logits are tokens of probability 0
    z = torch.randn(3, 5, generator=gen)
    z[0] = math.nan
    z[1, 3] = -math.inf
    z.requires_grad_(True)
    lp, ent = ops.token_log_probs(z, torch.tensor([-100, 1, 2]), return_entropy=True)
    (lp.sum() + ent.sum()).backward()
    assert torch.isfinite(lp).all() and torch.isfinite(ent).all() and torch.isfinite(z.grad).all()
    assert z.grad[0].abs().max() == 0 and z.grad[1, 3] == 0


def test_fused_linear_token_log_probs_equal_the_two_steps():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 5, 12, dtype=torch.float64, generator=gen, requires_grad=True)
    w = torch.randn(19, 12, dtype=torch.float64, generator=gen, requires_grad=True)
    labels = torch.randint(0, 19, (2, 5), generator=gen)
    labels[1, 2] = -100
    got = ops.fused_linear_token_log_probs(x, w, labels, logit_scale=0.7, return_entropy=True)
    want = ops.token_log_probs(x @ w.t(), labels, logit_scale=0.7, return_entropy=True)
    assert torch.allclose(got[0], want[0]) and torch.allclose(got[1], want[1])
    assert torch.autograd.gradcheck(lambda a, b: ops.fused_linear_token_log_probs(a, b, labels), (x, w))


@pytest.mark.parametrize("loss_type,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("average", [False, True])
def test_preference_loss_follows_the_formula(loss_type, smoothing, average):
    gen = torch.Generator().manual_seed(3)
    cu = torch.tensor([1, 4, 4, 9, 12])  # two pairs; the second chosen answer is empty, token 0 and 12 belong to no answer
    lp = (-torch.rand(13, dtype=torch.float64, generator=gen)).requires_grad_(True)
    ref = -torch.rand(13, dtype=torch.float64, generator=gen)
    mask = torch.ones(13, dtype=torch.bool)
    mask[5] = False
    call = lambda a, reduction: ops.preference_loss(a, ref, cu, beta=0.3, loss_type=loss_type, label_smoothing=smoothing, average_log_probs=average, mask=mask, reduction=reduction)
    spans = [[1, 2, 3], [], [4, 6, 7, 8], [9, 10, 11]]
    s = [sum((lp[t] - ref[t]).item() for t in span) / (max(len(span), 1) if average else 1) for span in spans]
    want = []
    for c, r in ((s[0], s[2]), (s[1], s[3])):
        d = c - r
        if loss_type == "sigmoid":
            want.append(-(1 - smoothing) * math.log(1 / (1 + math.exp(-0.3 * d))) - smoothing * math.log(1 / (1 + math.exp(0.3 * d))))
        else:
            want.append(max(0.0, 1 - 0.3 * d) if loss_type == "hinge" else (d - 1 / 0.6) ** 2)
    out = call(lp, "none")
    assert torch.allclose(out.loss, torch.tensor(want, dtype=torch.float64), rtol=1e-12)
    assert torch.allclose(out.chosen_rewards, 0.3 * torch.tensor([s[0], s[1]], dtype=torch.float64), rtol=1e-12, atol=1e-15)
    assert torch.allclose(out.rejected_rewards, 0.3 * torch.tensor([s[2], s[3]], dtype=torch.float64), rtol=1e-12)
    assert not out.chosen_rewards.requires_grad
    assert torch.allclose(call(lp, "mean").loss, sum(want) / 2 * torch.ones((), dtype=torch.float64))
    assert torch.allclose(call(lp, "sum").loss, sum(want) * torch.ones((), dtype=torch.float64))
    assert torch.autograd.gradcheck(lambda a: call(a, "none").loss, (lp,))
    (grad,) = torch.autograd.grad(call(lp, "mean").loss, lp)
    assert (grad[[0, 5, 12]] == 0).all()


@pytest.mark.parametrize("reduction", ["sum", "token_mean", "sequence_mean"])
@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("dual_clip", [None, 1.5])
def test_policy_loss_follows_the_formula(reduction, per_token, dual_clip):
    gen = torch.Generator().manual_seed(4)
    lp = (-torch.rand(3, 6, dtype=torch.float64, generator=gen)).requires_grad_(True)
    old, ref = lp.detach() + 0.4 * torch.randn(3, 6, dtype=torch.float64, generator=gen), -torch.rand(3, 6, dtype=torch.float64, generator=gen)
    adv = torch.randn((3, 6) if per_token else (3,), dtype=torch.float64, generator=gen)
    mask = torch.rand(3, 6, generator=gen) < 0.7
    mask[1] = False  # an answer without tokens
    with torch.no_grad():
        old[1, 0], ref[1, 1] = math.nan, math.inf  # never looked at
    call = lambda a: ops.policy_loss(a, old, adv, reference_log_probs=ref, mask=mask, clip_low=0.2, clip_high=0.3, dual_clip=dual_clip, kl_coef=0.1, reduction=reduction)
    total, kls, clips, per_answer = 0.0, [], 0, []
    for i in range(3):
        values = []
        for t in range(6):
            if not mask[i, t]:
                continue
            a = (adv[i, t] if per_token else adv[i]).item()
            r = math.exp(lp[i, t].item() - old[i, t].item())
            value = max(-a * r, -a * min(max(r, 0.8), 1.3))
            clip = (a > 0 and r > 1.3) or (a < 0 and r < 0.8)
            if dual_clip and a < 0 and value > -dual_clip * a:
                value, clip = -dual_clip * a, True
            k = ref[i, t].item() - lp[i, t].item()
            kls.append(math.expm1(k) - k)
            values.append(value + 0.1 * kls[-1])
            clips += clip
        if values:
            per_answer.append(sum(values) / len(values))
            total += sum(values)
    want = total if reduction == "sum" else total / len(kls) if reduction == "token_mean" else sum(per_answer) / len(per_answer)
    out = call(lp)
    assert out.loss.item() == pytest.approx(want, rel=1e-12)
    assert out.kl.item() == pytest.approx(sum(kls) / len(kls), rel=1e-12) and out.clip_fraction.item() == pytest.approx(clips / len(kls), rel=1e-12)
    assert torch.autograd.gradcheck(lambda a: call(a).loss, (lp,))
    (grad,) = torch.autograd.grad(out.loss, lp)
    assert (grad[~mask] == 0).all() and torch.isfinite(grad).all()


def test_policy_loss_with_nothing_kept_is_zero():
    lp = torch.full((2, 3), -1.0, requires_grad=True)
    for reduction in ("sum", "token_mean", "sequence_mean"):
        out = ops.policy_loss(lp, lp.detach(), torch.ones(2), mask=torch.zeros(2, 3, dtype=torch.bool), reduction=reduction)
        assert out.loss.item() == 0 and out.kl.item() == 0 and out.clip_fraction.item() == 0
        (grad,) = torch.autograd.grad(out.loss, lp)
        assert (grad == 0).all()


def test_sorted_embedding_on_the_cpu_is_the_plain_one():
    w = torch.randn(7, 3, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[0, 6], [6, 2]])
    assert torch.equal(ops.embedding(w, ids, 2.0, sorted_gradient=True), 2.0 * w.detach()[ids])
    assert torch.autograd.gradcheck(lambda a: ops.embedding(a, ids, 2.0, sorted_gradient=True), (w,))


def test_token_log_probs_of_a_model_shift_like_the_language_modelling_loss():
    """Summed log-probabilities are minus the summed loss, padded and packed, from logits and from hidden states, and drive both losses."""
    from lm_engine.hf_models import get_autoregressive_language_modeling_loss, get_token_log_probs

    gen = torch.Generator().manual_seed(5)
    hidden, weight = torch.randn(2, 6, 8, generator=gen), torch.randn(13, 8, generator=gen)
    labels = torch.randint(0, 13, (2, 6), generator=gen)
    labels[0, :3] = -100
    logits = hidden @ weight.t()
    want = get_autoregressive_language_modeling_loss(logits, labels, reduction="sum", logit_scale=0.5)
    lp = get_token_log_probs(logits, labels, logit_scale=0.5)
    assert lp.shape == labels.shape and torch.allclose(lp.sum(), -want, rtol=1e-5) and (lp[:, -1] == 0).all() and (lp[0, :2] == 0).all()
    assert torch.allclose(get_token_log_probs(None, labels, hidden, weight, logit_scale=0.5), lp, atol=1e-5)
    unshifted = get_token_log_probs(logits, labels, logit_scale=0.5, shift_logits_and_labels=False)
    assert torch.allclose(unshifted.sum(), -get_autoregressive_language_modeling_loss(logits, labels, reduction="sum", logit_scale=0.5, shift_logits_and_labels=False), rtol=1e-5)
    cu = torch.tensor([0, 4, 4, 9, 12], dtype=torch.int32)
    flat, packed = logits.reshape(12, 13), labels.reshape(12)
    want = get_autoregressive_language_modeling_loss(flat, packed.clone(), cu_seqlens=cu, use_padding_free_transformer=True, reduction="sum")
    lp, entropy = get_token_log_probs(flat, packed, cu_seqlens=cu, use_padding_free_transformer=True, return_entropy=True)
    assert torch.allclose(lp.sum(), -want, rtol=1e-5) and (lp[[3, 8, 11]] == 0).all() and (entropy >= 0).all()
    leaf = lp.detach().requires_grad_(True)
    (grad,) = torch.autograd.grad(ops.preference_loss(leaf, lp.detach() - 0.1, cu).loss, leaf)
    assert torch.isfinite(grad).all() and grad.abs().max() > 0
    with pytest.raises(ValueError):
        get_token_log_probs(logits, labels, tensor_parallel_enabled=True)
    with pytest.raises(ValueError):
        get_token_log_probs(flat, packed, use_padding_free_transformer=True)


def test_embedding_layer_follows_the_deterministic_switch(monkeypatch):
    from lm_engine.hf_models.layers.basic import ParameterizedEmbedding

    layer = ParameterizedEmbedding(5, 4, std=0.1)
    ids = torch.tensor([1, 4, 1])
    called = []
    monkeypatch.setattr(ops, "embedding_sorted", lambda w, i, s: called.append(s) or torch.nn.functional.embedding(i, w))
    plain = layer(ids)
    assert not called
    torch.use_deterministic_algorithms(True)
    try:
        assert torch.equal(layer(ids), plain) and called == [1.0]
        assert torch.equal(ops.embedding(layer.weight, ids, sorted_gradient=False), plain) and called == [1.0]
    finally:
        torch.use_deterministic_algorithms(False)


LP = torch.zeros(4, 3)
CU = torch.tensor([0, 3, 6, 9, 12])


@pytest.mark.parametrize("call", [
    lambda: ops.token_log_probs(torch.zeros(3, 5), torch.zeros(3)),                                      # labels not integer
    lambda: ops.token_log_probs(torch.zeros(3, 5), torch.zeros(4, dtype=torch.long)),                    # shape
    lambda: ops.token_log_probs(torch.zeros(3, 0), torch.zeros(3, dtype=torch.long)),                    # no vocabulary
    lambda: ops.token_log_probs(torch.zeros(3, 5, dtype=torch.long), torch.zeros(3, dtype=torch.long)),  # logits not floating point
    lambda: ops.token_log_probs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.long), logit_scale=0.0),
    lambda: ops.token_log_probs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.long), logit_scale=-1.0),
    lambda: ops.token_log_probs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.long), logit_scale=math.inf),
    lambda: ops.fused_linear_token_log_probs(torch.zeros(3, 8), torch.zeros(5, 9), torch.zeros(3, dtype=torch.long)),
    lambda: ops.fused_linear_token_log_probs(torch.zeros(3, 8), torch.zeros(5, 8).bfloat16(), torch.zeros(3, dtype=torch.long)),
    lambda: ops.fused_linear_token_log_probs(torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(2, dtype=torch.long)),
    lambda: ops.fused_linear_token_log_probs(torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.long), logit_scale=math.nan),
    lambda: ops.preference_loss(torch.zeros(3, 3), None),                                                # odd number of answers
    lambda: ops.preference_loss(torch.zeros(0, 3), None),
    lambda: ops.preference_loss(torch.zeros(12), None),                                                  # packed without cu_seqlens
    lambda: ops.preference_loss(LP, None, CU),                                                           # padded with cu_seqlens
    lambda: ops.preference_loss(LP.flatten(), None, CU.float()),
    lambda: ops.preference_loss(LP, torch.zeros(4, 4)),
    lambda: ops.preference_loss(LP, torch.zeros(4, 3, requires_grad=True)),
    lambda: ops.preference_loss(LP, None, beta=0.0),
    lambda: ops.preference_loss(LP, None, beta=math.nan),
    lambda: ops.preference_loss(LP, None, loss_type="log"),
    lambda: ops.preference_loss(LP, None, reduction="batch"),
    lambda: ops.preference_loss(LP, None, label_smoothing=0.5),
    lambda: ops.preference_loss(LP, None, label_smoothing=0.1, loss_type="ipo"),
    lambda: ops.preference_loss(LP, None, mask=torch.ones(4, 3)),
    lambda: ops.preference_loss(LP, None, mask=torch.ones(4, 2, dtype=torch.bool)),
    lambda: ops.preference_loss(torch.zeros(4, 3, dtype=torch.long), None),
    lambda: ops.policy_loss(LP, torch.zeros(4, 2), torch.zeros(4)),
    lambda: ops.policy_loss(LP, torch.zeros(4, 3, requires_grad=True), torch.zeros(4)),
    lambda: ops.policy_loss(LP, LP, torch.zeros(3)),
    lambda: ops.policy_loss(LP, LP, torch.zeros(4, requires_grad=True)),
    lambda: ops.policy_loss(LP, LP, torch.zeros(4), clip_low=1.5),
    lambda: ops.policy_loss(LP, LP, torch.zeros(4), clip_high=-0.1),
    lambda: ops.policy_loss(LP, LP, torch.zeros(4), dual_clip=1.0),
    lambda: ops.policy_loss(LP, LP, torch.zeros(4), kl_coef=0.1),                                        # no reference
    lambda: ops.policy_loss(LP, LP, torch.zeros(4), reference_log_probs=LP, kl_coef=-0.1),
    lambda: ops.policy_loss(LP, LP, torch.zeros(4), reduction="mean"),
    lambda: ops.embedding(torch.zeros(5, 4), torch.zeros(3), sorted_gradient=True),
    lambda: ops.embedding(torch.zeros(5), torch.zeros(3, dtype=torch.long), sorted_gradient=True),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()


F32, I64 = (lambda *s: torch.zeros(*s)), (lambda *s: torch.zeros(*s, dtype=torch.long))
LOSS = dict(zip(("kind", "beta", "smoothing", "average", "reduction"), (0, 0.1, 0.0, False, 2)))
POLICY = (0.2, 0.2, 0.0, 0.0, 1)


@pytest.mark.parametrize("call", [
    lambda C: C.token_log_probs(F32(3, 5), F32(3), 1.0, -100, False),
    lambda C: C.token_log_probs(F32(3, 5), I64(4), 1.0, -100, False),
    lambda C: C.token_log_probs(F32(3, 0), I64(3), 1.0, -100, False),
    lambda C: C.token_log_probs(F32(3, 5), I64(3), -0.5, -100, False),
    lambda C: C.linear_token_log_probs(F32(3, 8), F32(5, 9), I64(3), 1.0, -100, False, 256, 0, F32(1)),
    lambda C: C.linear_token_log_probs(F32(3, 8), F32(5, 8).half(), I64(3), 1.0, -100, False, 256, 0, F32(1)),
    lambda C: C.linear_token_log_probs(F32(3, 8), F32(5, 8), I64(3), math.inf, -100, False, 256, 0, F32(1)),
    lambda C: C.preference_loss(F32(3, 3), None, None, None, *LOSS.values()),
    lambda C: C.preference_loss(F32(12), None, None, None, *LOSS.values()),
    lambda C: C.preference_loss(F32(12), None, F32(5), None, *LOSS.values()),
    lambda C: C.preference_loss(F32(4, 3), F32(4, 4), None, None, *LOSS.values()),
    lambda C: C.preference_loss(F32(4, 3), None, None, F32(4, 3), *LOSS.values()),
    lambda C: C.preference_loss(F32(4, 3), None, None, None, *(LOSS | dict(beta=0.0)).values()),
    lambda C: C.preference_loss(F32(4, 3), None, None, None, *(LOSS | dict(kind=2, smoothing=0.1)).values()),
    lambda C: C.policy_loss(F32(4, 3), F32(4, 3), F32(3), None, None, None, *POLICY),
    lambda C: C.policy_loss(F32(4, 3), F32(4, 3).requires_grad_(True), F32(4), None, None, None, *POLICY),
    lambda C: C.policy_loss(F32(4, 3), F32(4, 3), F32(4), None, None, None, 1.2, *POLICY[1:]),
    lambda C: C.policy_loss(F32(4, 3), F32(4, 3), F32(4), None, None, None, 0.2, 0.2, 0.0, 0.1, 1),
    lambda C: C.policy_loss(F32(4, 3), F32(4, 3), F32(4), None, None, None, 0.2, 0.2, 0.5, 0.0, 1),
    lambda C: C.embedding_sorted(F32(5, 4), F32(3), 1.0, F32(1)),
    lambda C: C.embedding_sorted(F32(5), I64(3), 1.0, F32(1)),
])
def test_the_extension_refuses_the_same_calls(call):
    """Its checks come before anything that needs a device, so their errors (numbers in them included) are raised here as they are on a GPU."""
    with pytest.raises(ValueError):
        call(ops.native())


def test_an_ignored_label_beyond_32_bits_is_no_int32_label():
    z = torch.randn(4, 5, generator=torch.Generator().manual_seed(0))
    labels = torch.tensor([0, 1, 2, 0])
    got = ops.token_log_probs(z, labels.int(), ignore_index=-(1 << 40))
    assert torch.equal(got, ops.token_log_probs(z, labels))
