"""Vocabulary operators on the GPU against their definitions in 64 bits.

Tolerances. A rounding to type t is off by at most eps(t) / 2 relative to the value. Scores are formed as fp32 (x - m) c with
c = fl(logit_scale log2 e): relative error 2^-23 of |x - m| c from c and roundings of 2^-24 of the difference and the result; the base-2 exponential is good to 2^-22; a row's
sum adds at most V / 512 + 32 terms in sequence (512 threads, then trees). That bounds the error of a log-sum-exp by
LSE_ERR = (4 max|z| + V / 512 + 64) 2^-23, and the relative error of a probability by the same.
"""

import math

import pytest
import torch

from lm_engine import ops

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


@pytest.fixture(autouse=True)
def _healthy():
    yield
    ops.check_status()


def _lse_err(z64, extra=0.0):
    finite = z64[torch.isfinite(z64)]
    top = finite.abs().max().item() if finite.numel() else 0.0
    return (4 * top + z64.shape[-1] / 512 + 64) * 2.0**-23 + extra


def _score(z, labels, ignore_index, g, h):
    """Log-probability, entropy, score gradient (rows of 64-bit scores z) and the probabilities."""
    kept = (labels != ignore_index) & (labels >= 0) & (labels < z.shape[-1])
    y = torch.where(kept, labels.long(), 0)[:, None]
    z = torch.where(kept[:, None], z, 0.0)
    logp = z.log_softmax(-1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    ent = -plogp.sum(-1)
    grad = -g[:, None] * p
    grad.scatter_add_(1, y, g[:, None].clone())
    grad -= h[:, None] * (plogp + p * ent[:, None])
    keep = kept.double()
    return logp.gather(1, y)[:, 0] * keep, ent * keep, grad * keep[:, None], p * keep[:, None], logp, kept


def _check_log_probs(z, labels, ignore_index, g, h, lp, ent, grad=None, scale=1.0, dtype=torch.float32, extra=0.0):
    want_lp, want_ent, want_grad, p, logp, kept = _score(z, labels, ignore_index, g, h)
    err = _lse_err(z, extra)
    assert (lp.double() - want_lp).abs().max() <= err + 2.0**-24 * want_lp.abs().max()
    if ent is not None:
        # H = sum of -p log p: relative error of p on each term, plus the log-sum-exp's
        assert (ent.double() - want_ent).abs().max() <= err * (2 + want_ent.abs().max())
    if grad is not None:
        # factors of p: g + |h| (|log p| + H), of which every one is off by err relative to p; the label's own g is exact to a rounding
        size = p * (g.abs()[:, None] + h.abs()[:, None] * (torch.where(p > 0, logp.abs(), 0.0) + want_ent[:, None] + 1))
        bound = scale * (4 * err * size + 2.0**-23 * g.abs()[:, None]) + HALF[dtype] * scale * want_grad.abs() + 2.0**-25 * (dtype == torch.float16)
        off = (grad.double() - scale * want_grad).abs()
        assert (off <= bound).all(), (off - bound).max()
        assert (grad[~kept] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,vocab", [(1, 1), (3, 7), (5, 8), (2, 1003), (300, 1000), (17, 50001)])
@pytest.mark.parametrize("entropy", [False, True])
def test_token_log_probs(dtype, tokens, vocab, entropy):
    gen = torch.Generator("cuda").manual_seed(tokens * vocab)
    logits = (3 * torch.randn(tokens, vocab, generator=gen, device="cuda")).to(dtype).requires_grad_(True)
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    if tokens > 2:
        labels[1], labels[2] = -100, vocab
    g, h = torch.randn(tokens, generator=gen, device="cuda"), torch.randn(tokens, generator=gen, device="cuda")
    out = ops.token_log_probs(logits, labels, logit_scale=0.75, return_entropy=entropy)
    outs = out if entropy else (out,)
    (grad,) = torch.autograd.grad(outs, logits, [g, h][: len(outs)])
    assert grad.dtype == dtype and grad.shape == logits.shape
    h64 = h.double() if entropy else torch.zeros(tokens, device="cuda", dtype=torch.float64)
    _check_log_probs(0.75 * logits.detach().double(), labels, -100, g.double(), h64, outs[0], outs[1] if entropy else None, grad, 0.75, dtype)
    with torch.no_grad():
        again = ops.token_log_probs(logits, labels.int(), logit_scale=0.75, return_entropy=entropy)
    assert torch.equal(again[0] if entropy else again, outs[0])


@pytest.mark.parametrize("offset,pitch", [(0, 1008), (1, 1008), (3, 1001), (5, 1003)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_log_probs_strided_rows_read_nothing_else(offset, pitch, dtype):
    vocab, tokens = 997, 9
    gen = torch.Generator("cuda").manual_seed(offset)
    buffer = torch.full((tokens * pitch + 64,), math.nan, device="cuda", dtype=dtype)
    logits = buffer[offset : offset + tokens * pitch].view(tokens, pitch)[:, :vocab]
    logits.copy_(torch.randn(tokens, vocab, generator=gen, device="cuda"))
    logits.requires_grad_(True)
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    lp, ent = ops.token_log_probs(logits, labels, return_entropy=True)
    g, h = torch.randn(tokens, generator=gen, device="cuda"), torch.randn(tokens, generator=gen, device="cuda")
    (grad,) = torch.autograd.grad((lp, ent), logits, (g, h))
    _check_log_probs(logits.detach().double(), labels, -100, g.double(), h.double(), lp, ent, grad, 1.0, dtype)


def test_token_log_probs_of_a_shifted_batch():
    gen = torch.Generator("cuda").manual_seed(0)
    logits = torch.randn(3, 7, 130, generator=gen, device="cuda").bfloat16().requires_grad_(True)
    tokens = torch.randint(0, 130, (3, 7), generator=gen, device="cuda")
    lp = ops.token_log_probs(logits[:, :-1], tokens[:, 1:])
    assert lp.shape == (3, 6)
    lp.sum().backward()  # broadcast upstream gradient
    z = logits.detach()[:, :-1].reshape(-1, 130).double()
    one, zero = torch.ones(18, device="cuda", dtype=torch.float64), torch.zeros(18, device="cuda", dtype=torch.float64)
    _check_log_probs(z, tokens[:, 1:].reshape(-1), -100, one, zero, lp.reshape(-1), None, logits.grad[:, :-1].reshape(-1, 130), 1.0, torch.bfloat16)
    assert (logits.grad[:, -1] == 0).all()


def test_token_log_probs_where_masks_and_infinities_are():
    vocab = 2050
    logits = torch.randn(6, vocab, device="cuda")
    logits[0] = math.nan                      # ignored row
    logits[1, 5:] = -math.inf                 # nearly everything is banned
    logits[2] = torch.finfo(torch.float32).min  # a mask of the type's lowest value everywhere: uniform
    logits[3] = -math.inf                     # nothing is left
    logits[4, ::2] = torch.finfo(torch.float32).min
    logits[5, 7] = math.nan
    labels = torch.tensor([-100, 3, 0, 1, 1, 2], device="cuda")
    logits.requires_grad_(True)
    lp, ent = ops.token_log_probs(logits, labels, return_entropy=True)
    lp.sum().add(ent.sum()).backward()
    want_lp, want_ent = [torch.zeros(6, dtype=torch.float64) for _ in range(2)]
    for r in (1, 4):
        d = logits.detach()[r].double().cpu().log_softmax(-1)
        want_lp[r], want_ent[r] = d[labels[r]], -(d.exp() * d.clamp_min(-1e300)).sum()
    want_lp[2], want_ent[2] = -math.log(vocab), math.log(vocab)
    good = [0, 1, 2, 4]
    # the row of -3.4e38 cancels exactly: x - m is 0 for every token
    err = _lse_err(torch.randn(1, vocab)) + 32 * 2.0**-23
    assert (lp.cpu().double() - want_lp)[good].abs().max() <= err and (ent.cpu().double() - want_ent)[good].abs().max() <= 10 * err
    assert torch.isfinite(logits.grad[good]).all() and (logits.grad[0] == 0).all() and (logits.grad[1, 5:] == 0).all()
    assert lp[3].isnan() and lp[5].isnan() and logits.grad[3].isnan().all() and logits.grad[5].isnan().all()


def test_token_log_probs_of_nothing():
    logits = torch.zeros(0, 40, device="cuda", requires_grad=True)
    lp = ops.token_log_probs(logits, torch.zeros(0, dtype=torch.long, device="cuda"))
    lp.sum().backward()
    assert lp.shape == (0,) and logits.grad.shape == (0, 40)


# ----------------------------------------------------------------------------- from hidden states
def _linear_case(tokens, hidden, vocab, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").bfloat16()
    w = (2 / math.sqrt(hidden) * torch.randn(vocab, hidden, generator=gen, device="cuda")).bfloat16()
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    g, h = torch.randn(tokens, generator=gen, device="cuda"), 0.3 * torch.randn(tokens, generator=gen, device="cuda")
    return x, w, labels, g, h


def _check_linear(x, w, labels, g, h, lp, ent, dx, dw, scale=1.0, ignore_index=-100):
    """An fp32 accumulator of H products is off by at most (H / 16 + 16) 2^-24 of their absolute sum (16 products per step); d(logits) is stored in bf16,
    so the products that follow are off by at most 2^-8 of their absolute sums, plus the output's own rounding."""
    x64, w64 = x.detach().double(), w.detach().double()
    logit_err = scale * ((x64.shape[1] / 16 + 16) * 2.0**-24 * (x64.abs() @ w64.abs().t())).max().item()
    z = scale * (x64 @ w64.t())
    h64 = h.double() if ent is not None else torch.zeros_like(g, dtype=torch.float64)
    _check_log_probs(z, labels, ignore_index, g.double(), h64, lp, ent, extra=2 * logit_err)
    if dx is None:
        return
    want_lp, want_ent, dz, p, logp, kept = _score(z, labels, ignore_index, g.double(), h64)
    dz = scale * dz
    rel = 2.0**-8 + 8 * _lse_err(z, 2 * logit_err)
    slack = rel * (dz.abs() + 2.0**-8 * scale * p * (g.abs() + h64.abs() * (want_ent + 8))[:, None])
    for got, want, bound in ((dx, dz @ w64, slack @ w64.abs()), (dw, dz.t() @ x64, slack.t() @ x64.abs())):
        off = (got.double() - want).abs()
        limit = bound + HALF.get(got.dtype, 0.0) * want.abs() + (dz.shape[0] + dz.shape[1]) * 2.0**-24 * bound / rel
        assert (off <= limit).all(), (off - limit).max()


@pytest.mark.parametrize("tokens,hidden,vocab", [(1, 8, 1), (3, 64, 40), (130, 72, 257), (256, 128, 1024), (300, 256, 1003), (777, 512, 5000)])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("keep", [0, 4 << 30])
def test_fused_linear_token_log_probs(tokens, hidden, vocab, entropy, keep, monkeypatch):
    import lm_engine.ops.vocabulary as vocabulary

    monkeypatch.setattr(vocabulary, "_KEEP_LOGITS_BYTES", keep)
    x, w, labels, g, h = _linear_case(tokens, hidden, vocab, tokens)
    if tokens > 2:
        labels[0], labels[2] = -100, -7
    x.requires_grad_(True)
    w.requires_grad_(True)
    out = ops.fused_linear_token_log_probs(x, w, labels, logit_scale=0.8, return_entropy=entropy)
    outs = out if entropy else (out,)
    dx, dw = torch.autograd.grad(outs, (x, w), [g, h][: len(outs)])
    assert dx.dtype == dw.dtype == torch.bfloat16
    _check_linear(x, w, labels, g, h, outs[0], outs[1] if entropy else None, dx, dw, 0.8)
    with torch.no_grad():
        again = ops.fused_linear_token_log_probs(x, w, labels, logit_scale=0.8, return_entropy=entropy)
    assert torch.equal(again[0] if entropy else again, outs[0])  # the same bits on every run


def test_fused_linear_token_log_probs_in_chunks_and_into_main_grad(monkeypatch):
    import lm_engine.ops.vocabulary as vocabulary

    x, w, labels, g, h = _linear_case(700, 64, 600, 5)
    x.requires_grad_(True)
    w.requires_grad_(True)
    whole = torch.autograd.grad(ops.fused_linear_token_log_probs(x, w, labels), (x, w), g)
    monkeypatch.setattr(vocabulary, "_flce_chunk_rows", lambda T, V: 256)
    chunks = torch.autograd.grad(ops.fused_linear_token_log_probs(x, w, labels), (x, w), g)
    assert torch.equal(whole[0], chunks[0])
    zero = torch.zeros_like(h)
    lp = ops.fused_linear_token_log_probs(x, w, labels)
    _check_linear(x, w, labels, g, zero, lp.detach(), None, *chunks)
    # an engine-owned fp32 buffer is added to and autograd sees no gradient of the weight
    w.main_grad = torch.full((600, 64), 2.0, device="cuda")
    (lp * g).sum().backward()
    assert w.grad is None
    _check_linear(x, w, labels, g, zero, lp.detach(), None, x.grad, w.main_grad - 2.0)


@pytest.mark.parametrize("tokens,hidden,vocab", [(1, 8, 1), (130, 72, 257), (300, 256, 1003), (1000, 64, 5000)])
@pytest.mark.parametrize("entropy", [False, True])
def test_fused_linear_token_log_probs_kept_or_formed_twice_are_the_same(tokens, hidden, vocab, entropy):
    x, w, labels, g, h = _linear_case(tokens, hidden, vocab, tokens)
    labels[::3] = -100
    x.requires_grad_(True)
    w.requires_grad_(True)
    results = []
    for keep in (False, True):
        out = ops.fused_linear_token_log_probs(x, w, labels, logit_scale=1.25, return_entropy=entropy, keep_logits=keep)
        outs = out if entropy else (out,)
        results.append((*outs, *torch.autograd.grad(outs, (x, w), [g, h][: len(outs)])))
    for i, (a, b) in enumerate(zip(*results)):
        if i < len(outs):
            assert torch.equal(a, b)
        else:  # the exponents' last rounding differs: (x - m) c - log2 s against x c - (m c + log2 s)
            assert (a.float() - b.float()).norm() <= 2.0**-10 * b.float().norm()


@pytest.mark.parametrize("keep", [0, 4 << 30])
@pytest.mark.parametrize("kept", [0.0, 0.01, 0.5])
@pytest.mark.parametrize("chunk,tokens", [(128, 1000), (384, 1000), (4096, 1000), (4096, 100), (4096, 3)])
def test_fused_linear_token_log_probs_leaves_ignored_rows_out(kept, chunk, tokens, keep, monkeypatch):
    import lm_engine.ops.vocabulary as vocabulary

    monkeypatch.setattr(vocabulary, "_KEEP_LOGITS_BYTES", keep)
    monkeypatch.setattr(vocabulary, "_flce_chunk_rows", lambda T, V: min(T, chunk))
    x, w, labels, g, h = _linear_case(tokens, 64, 333, 8)
    labels[torch.rand(tokens, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) >= kept] = -100
    x[labels == -100] = math.nan  # not looked at
    junk = torch.full((64 << 20,), math.nan, device="cuda")  # what the allocator hands out next holds NaN
    del junk
    x.requires_grad_(True)
    w.requires_grad_(True)
    lp, ent = ops.fused_linear_token_log_probs(x, w, labels, return_entropy=True)
    dx, dw = torch.autograd.grad((lp, ent), (x, w), (g, h))
    assert (lp[labels == -100] == 0).all() and (ent[labels == -100] == 0).all() and (dx[labels == -100] == 0).all()
    with torch.no_grad():
        x[labels == -100] = 0
    _check_linear(x, w, labels, g, h, lp, ent, dx, dw)


def test_fused_linear_token_log_probs_strided_operands_and_shapes():
    x, w, labels, g, h = _linear_case(24, 64, 300, 6)
    wide = torch.zeros(24, 96, device="cuda", dtype=torch.bfloat16)
    wide[:, 16:80] = x
    odd = torch.zeros(300, 67, device="cuda", dtype=torch.bfloat16)
    odd[:, 1:65] = w  # rows that no tensor map can describe: copied
    lp = ops.fused_linear_token_log_probs(wide[:, 16:80].unflatten(0, (2, 12)), odd[:, 1:65], labels.view(2, 12).int(), ignore_index=int(labels[3]))
    want = ops.fused_linear_token_log_probs(x, w, labels, ignore_index=int(labels[3]))
    assert torch.equal(lp.flatten(), want) and want[3] == 0
    empty = ops.fused_linear_token_log_probs(x[:0].requires_grad_(True), w.requires_grad_(True), labels[:0])
    (dw,) = torch.autograd.grad(empty.sum(), w)
    assert empty.shape == (0,) and (dw == 0).all()


# ----------------------------------------------------------------------------- losses
def _cu(lengths, start=0):
    return torch.tensor([start] + [start + sum(lengths[: i + 1]) for i in range(len(lengths))], dtype=torch.int32, device="cuda")


LENGTHS = [[1, 1], [0, 3, 5, 0], [300, 7, 256, 512, 1, 255], [70000, 3, 2500, 1]]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("kind", ["sigmoid", "smoothed", "hinge", "ipo"])
@pytest.mark.parametrize("average", [False, True])
def test_preference_loss(lengths, kind, average):
    gen = torch.Generator("cuda").manual_seed(len(lengths))
    cu, total = _cu(lengths, 2), sum(lengths) + 5
    ref = -2 * torch.rand(total, generator=gen, device="cuda")
    lp = (ref + 0.05 * torch.randn(total, generator=gen, device="cuda")).requires_grad_(True)
    mask = torch.rand(total, generator=gen, device="cuda") < 0.7
    with torch.no_grad():
        ref[~mask] = math.nan
    kw = dict(beta=0.2, loss_type="sigmoid" if kind == "smoothed" else kind, label_smoothing=0.1 if kind == "smoothed" else 0.0, average_log_probs=average, mask=mask)
    lp64 = lp.detach().cpu().double().requires_grad_(True)
    for reduction in ("mean", "sum", "none"):
        got = ops.preference_loss(lp, ref, cu, reduction=reduction, **kw)
        want = ops.preference_loss(lp64, ref.cpu().double(), cu.cpu(), reduction=reduction, **(kw | dict(mask=mask.cpu())))
        up = torch.randn(got.loss.shape, generator=gen, device="cuda")
        (grad,) = torch.autograd.grad(got.loss, lp, up)
        (want_grad,) = torch.autograd.grad(want.loss, lp64, up.cpu().double())
        # sums and losses are formed in 64 bits from exact fp32 differences, beta and the smoothing are fp32 (2^-24 each, amplified
        # by at most 1 / (1 - 2 e) and, in the square of ipo, by twice its factor 1 / (2 beta) = 2.5 next to sums of a few units): 16 roundings
        for a, b in ((got.loss, want.loss), (got.chosen_rewards, want.chosen_rewards), (got.rejected_rewards, want.rejected_rewards), (grad, want_grad)):
            assert (a.detach().cpu().double() - b.detach()).abs().max() <= 16 * 2.0**-24 * max(1.0, b.abs().max().item())
        assert (grad[~mask] == 0).all() and (grad[:2] == 0).all() and (grad[-3:] == 0).all()


def test_preference_loss_padded_other_types_and_no_reference():
    gen = torch.Generator("cuda").manual_seed(1)
    lp = (-torch.rand(6, 33, generator=gen, device="cuda")).bfloat16().requires_grad_(True)
    mask = (torch.rand(6, 33, generator=gen, device="cuda") < 0.5).long()
    out = ops.preference_loss(lp, None, mask=mask)
    (grad,) = torch.autograd.grad(out.loss, lp)
    lp64 = lp.detach().cpu().double().requires_grad_(True)
    want = ops.preference_loss(lp64, None, mask=mask.cpu())
    (want_grad,) = torch.autograd.grad(want.loss, lp64)
    assert abs(out.loss.item() - want.loss.item()) <= 16 * 2.0**-24 and grad.dtype == torch.bfloat16
    assert ((grad.cpu().double() - want_grad).abs() <= 1.01 * 2.0**-8 * want_grad.abs()).all()
    packed = ops.preference_loss(lp.detach().flatten(), None, torch.arange(0, 199, 33, device="cuda"), mask=mask.flatten())
    assert torch.equal(packed.loss, out.loss)  # int64 cu_seqlens, the same sums in the same order


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("reduction", ["sum", "token_mean", "sequence_mean"])
@pytest.mark.parametrize("per_token,kl,dual", [(False, 0.0, None), (True, 0.1, None), (False, 0.1, 1.4)])
def test_policy_loss(lengths, reduction, per_token, kl, dual):
    gen = torch.Generator("cuda").manual_seed(len(lengths))
    cu, total = _cu(lengths, 1), sum(lengths) + 3
    old = -2 * torch.rand(total, generator=gen, device="cuda")
    lp = (old + 0.3 * torch.randn(total, generator=gen, device="cuda")).requires_grad_(True)
    ref = old + 0.3 * torch.randn(total, generator=gen, device="cuda")
    ref[::7] = lp.detach()[::7] * (1 + 2.0**-12)  # KL terms of nearly equal values
    adv = torch.randn(total if per_token else len(lengths), generator=gen, device="cuda")
    adv[0] = 0.0
    mask = torch.rand(total, generator=gen, device="cuda") < 0.7
    with torch.no_grad():
        old[~mask], ref[~mask] = math.nan, -math.inf
    kw = dict(clip_low=0.2, clip_high=0.3, dual_clip=dual, kl_coef=kl, reduction=reduction)
    got = ops.policy_loss(lp, old, adv, reference_log_probs=ref, cu_seqlens=cu, mask=mask, **kw)
    lp64 = lp.detach().cpu().double().requires_grad_(True)
    want = ops.policy_loss(lp64, old.cpu().double(), adv.cpu().double(), reference_log_probs=ref.cpu().double(), cu_seqlens=cu.cpu(), mask=mask.cpu(), **kw)
    (grad,) = torch.autograd.grad(got.loss, lp, torch.tensor(0.5, device="cuda"))
    (want_grad,) = torch.autograd.grad(want.loss, lp64, torch.tensor(0.5, dtype=torch.float64))
    # a token: differences, exponentials and products, 8 roundings of 2^-24 of terms |A| r + kl (1 + e^k); a warp adds 256 tokens (8 in
    # sequence, then a tree of 5): 16 more; the rest is 64 bits. Relative to the sum of the absolute terms.
    size = (3.0 * adv.abs().max().item() + 1) * (sum(lengths) if reduction == "sum" else 1)
    assert abs(got.loss.item() - want.loss.item()) <= 24 * 2.0**-24 * size
    assert abs(got.kl.item() - want.kl.item()) <= 24 * 2.0**-24 * max(want.kl.item(), 1e-6) and got.clip_fraction.item() == pytest.approx(want.clip_fraction.item(), abs=2.0**-23)
    off = (grad.cpu().double() - want_grad).abs()
    assert (off <= 16 * 2.0**-24 * (want_grad.abs() + size * want_grad.abs().max().clamp_max(1.0))).all()
    assert (grad[~mask] == 0).all() and (grad[:1] == 0).all() and (grad[-2:] == 0).all()
    with torch.no_grad():
        again = ops.policy_loss(lp, old, adv, reference_log_probs=ref, cu_seqlens=cu, mask=mask, **kw)
    assert torch.equal(again.loss, got.loss)


def test_policy_loss_edges():
    lp = torch.tensor([[0.0, -1.0, -2.0], [-200.0, 0.0, -1.0]], device="cuda", requires_grad=True)
    old = torch.tensor([[-200.0, -1.0, -2.0], [0.0, -200.0, -1.0]], device="cuda")
    adv = torch.tensor([0.0, 1.0], device="cuda")
    out = ops.policy_loss(lp, old, adv, reduction="sum")  # an infinite ratio without advantage counts nothing, one with a positive one is clipped
    (grad,) = torch.autograd.grad(out.loss, lp)
    assert out.loss.item() == pytest.approx(-(1.2 + 1.0), rel=4 * 2.0**-24)
    assert torch.equal(grad, torch.tensor([[0.0, 0.0, 0.0], [0.0, 0.0, -1.0]], device="cuda"))
    none = ops.policy_loss(lp, old, adv, mask=torch.zeros(2, 3, dtype=torch.bool, device="cuda"), reduction="sequence_mean")
    (grad,) = torch.autograd.grad(none.loss, lp)
    assert none.loss.item() == 0 and none.kl.item() == 0 and none.clip_fraction.item() == 0 and (grad == 0).all()
    empty = ops.policy_loss(torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"), cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert empty.loss.item() == 0


# ----------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hidden,vocab,repeat", [(1, 8, 1, 0), (5, 3, 4, 0), (64, 64, 1000, 0), (2048, 40, 300, 0.5), (2049, 24, 5, 0), (5000, 129, 70000, 0.9), (40000, 16, 100, 0)])
def test_embedding_with_sorted_gradient(dtype, tokens, hidden, vocab, repeat):
    gen = torch.Generator("cuda").manual_seed(tokens)
    w = torch.randn(vocab, hidden, generator=gen, device="cuda").to(dtype).requires_grad_(True)
    ids = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    ids[torch.rand(tokens, generator=gen, device="cuda") < repeat] = vocab - 1
    dout = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype)
    out = ops.embedding(w, ids, 1.5, sorted_gradient=True)
    assert torch.equal(out, (w.detach()[ids].float() * 1.5).to(dtype))
    (grad,) = torch.autograd.grad(out, w, dout)
    exact = torch.zeros(vocab, hidden, device="cuda", dtype=torch.float64).index_add_(0, ids, 1.5 * dout.double())
    total = torch.zeros(vocab, hidden, device="cuda", dtype=torch.float64).index_add_(0, ids, 1.5 * dout.double().abs())
    # additions in sequence: 32 in a block, then the partial sums of at most tokens / 32 blocks on 8 lanes
    limit = (32 + tokens / 256 + 12) * 2.0**-24 * total + HALF[dtype] * exact.abs() + 2.0**-24 * (dtype == torch.float16)
    assert ((grad.double() - exact).abs() <= limit).all()
    (again,) = torch.autograd.grad(ops.embedding(w, ids.int(), 1.5, sorted_gradient=True), w, dout)
    assert torch.equal(grad, again)
    # into the engine's fp32 buffer: added to what is there
    w.main_grad = torch.full((vocab, hidden), 3.0, device="cuda")
    ops.embedding(w, ids.view(-1, 1), 1.5, sorted_gradient=True).backward(dout.view(tokens, 1, hidden))
    assert w.grad is None
    assert ((w.main_grad.double() - 3.0 - exact).abs() <= (44 + tokens / 256) * 2.0**-24 * (total + 3.0)).all()


def test_embedding_with_sorted_gradient_ids_outside_of_the_table():
    w = torch.randn(10, 16, device="cuda").bfloat16().requires_grad_(True)
    ids = torch.tensor([3, -1, 9, 10, 3, 2**33], device="cuda")
    out = ops.embedding(w, ids, sorted_gradient=True)
    assert (out[[1, 3, 5]] == 0).all() and torch.equal(out[[0, 2, 4]], w.detach()[[3, 9, 3]])
    with pytest.raises(RuntimeError, match="token id outside"):
        ops.check_status()
    (grad,) = torch.autograd.grad(out, w, torch.ones_like(out))
    want = torch.zeros(10, 16, device="cuda")
    want[3], want[9] = 2, 1
    assert torch.equal(grad.float(), want)
    empty = ops.embedding(w, ids[:0], sorted_gradient=True)
    (grad,) = torch.autograd.grad(empty.sum(), w)
    assert empty.shape == (0, 16) and (grad == 0).all()


# ----------------------------------------------------------------------------- together
def _tuning_step(kind, weight, embed, head, ids, labels, cu, reference, advantages):
    """Embedding (tied to nothing) -> one product -> log-probabilities -> loss -> gradients of all three weights."""
    x = ops.embedding(embed, ids, 2.0, sorted_gradient=True)
    x = ops.linear(x, weight)
    lp = ops.fused_linear_token_log_probs(x, head, labels)
    mask = labels != -100
    if kind == "preference":
        loss = ops.preference_loss(lp, reference, cu, mask=mask).loss
    else:
        loss = ops.policy_loss(lp, reference, advantages, reference_log_probs=reference, cu_seqlens=cu, mask=mask, kl_coef=0.1, reduction="sequence_mean").loss
    # no graph outlives the step: gradient accumulators of a live eager graph belong to its stream, which a capture cannot join
    grads = torch.autograd.grad(loss, (embed, weight, head))
    return (loss.detach(), *grads)


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_a_tuning_step_matches_plain_torch_and_replays_from_a_graph(kind):
    gen = torch.Generator("cuda").manual_seed(2)
    vocab, hidden, lengths = 500, 64, [40, 70, 33, 129]
    total = sum(lengths)
    embed, head = [(0.5 * torch.randn(vocab, hidden, generator=gen, device="cuda")).bfloat16().requires_grad_(True) for _ in range(2)]
    weight = (torch.randn(hidden, hidden, generator=gen, device="cuda") / 8).bfloat16().requires_grad_(True)
    ids = torch.randint(0, vocab, (total,), generator=gen, device="cuda")
    labels = torch.roll(ids, -1)
    labels[torch.rand(total, generator=gen, device="cuda") < 0.3] = -100
    cu, reference, advantages = _cu(lengths), -6.2 + torch.randn(total, generator=gen, device="cuda"), torch.randn(4, generator=gen, device="cuda")
    args = (weight, embed, head, ids, labels, cu, reference, advantages)
    got = _tuning_step(kind, *args)

    leaves = [t.detach().float().requires_grad_(True) for t in (embed, weight, head)]
    x = (leaves[0][ids] * 2.0) @ leaves[1].t()
    logp = (x @ leaves[2].t()).log_softmax(-1)
    mask = labels != -100
    lp = torch.where(mask, logp.gather(1, labels.clamp_min(0)[:, None])[:, 0], 0.0).cpu()
    kw = dict(mask=mask.cpu())
    if kind == "preference":
        loss = ops.preference_loss(lp, reference.cpu(), cu.cpu(), **kw).loss
    else:
        loss = ops.policy_loss(lp, reference.cpu(), advantages.cpu(), reference_log_probs=reference.cpu(), cu_seqlens=cu.cpu(), kl_coef=0.1, reduction="sequence_mean", **kw).loss
    want = torch.autograd.grad(loss, leaves)
    # three bf16 roundings (2^-8 each at most, independent) lie between the weights and the loss and three more on the way back
    for a, b in zip(got[1:], want):
        assert ((a.float() - b).norm() / b.norm()).item() < 6 * 2.0**-8

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _tuning_step(kind, *args)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _tuning_step(kind, *args)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, got):
        assert torch.equal(a, b)
    with torch.no_grad():
        ids.copy_(torch.randint(0, vocab, (total,), generator=gen, device="cuda"))
    graph.replay()
    again = _tuning_step(kind, *args)
    torch.cuda.synchronize()
    for a, b in zip(captured, again):
        assert torch.equal(a, b)


def test_a_second_backward_pass_gives_the_same_gradients():
    logits = torch.randn(4, 100, device="cuda", requires_grad=True)
    labels = torch.tensor([1, 2, -100, 4], device="cuda")
    lp = ops.token_log_probs(logits, labels)
    loss = ops.policy_loss(lp[None], lp.detach()[None], torch.ones(1, device="cuda")).loss
    first = torch.autograd.grad(loss, logits, retain_graph=True)[0].clone()
    assert torch.equal(torch.autograd.grad(loss, logits)[0], first) and first.abs().max() > 0


@pytest.mark.parametrize("call", [
    lambda f, i: ops.token_log_probs(f(3, 5), f(3)),
    lambda f, i: ops.token_log_probs(f(3, 5), i(4)),
    lambda f, i: ops.token_log_probs(f(3, 5), i(3).cpu()),
    lambda f, i: ops.token_log_probs(f(3, 0), i(3)),
    lambda f, i: ops.token_log_probs(f(3, 5), i(3), logit_scale=0.0),
    lambda f, i: ops.token_log_probs(f(3, 5), i(3), logit_scale=math.nan),
    lambda f, i: ops.fused_linear_token_log_probs(f(3, 8).bfloat16(), f(5, 16).bfloat16(), i(3)),
    lambda f, i: ops.fused_linear_token_log_probs(f(3, 8).bfloat16(), f(5, 8), i(3)),
    lambda f, i: ops.fused_linear_token_log_probs(f(3, 8).bfloat16(), f(5, 8).bfloat16(), i(2)),
    lambda f, i: ops.preference_loss(f(3, 3), None),
    lambda f, i: ops.preference_loss(f(0, 3), None),
    lambda f, i: ops.preference_loss(f(12), None),
    lambda f, i: ops.preference_loss(f(4, 3), None, i(5)),
    lambda f, i: ops.preference_loss(f(12), None, f(5)),
    lambda f, i: ops.preference_loss(f(12), None, i(5).cpu()),
    lambda f, i: ops.preference_loss(f(4, 3), f(4, 4)),
    lambda f, i: ops.preference_loss(f(4, 3), f(4, 3).cpu()),
    lambda f, i: ops.preference_loss(f(4, 3), f(4, 3).requires_grad_(True)),
    lambda f, i: ops.preference_loss(f(4, 3), None, beta=0.0),
    lambda f, i: ops.preference_loss(f(4, 3), None, loss_type="log"),
    lambda f, i: ops.preference_loss(f(4, 3), None, reduction="batch"),
    lambda f, i: ops.preference_loss(f(4, 3), None, label_smoothing=0.5),
    lambda f, i: ops.preference_loss(f(4, 3), None, label_smoothing=0.1, loss_type="ipo"),
    lambda f, i: ops.preference_loss(f(4, 3), None, mask=f(4, 3)),
    lambda f, i: ops.preference_loss(f(4, 3), None, mask=i(4, 2)),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 2), f(4)),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3).requires_grad_(True), f(4)),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3), f(3)),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3), f(4).requires_grad_(True)),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3), f(4), clip_low=1.5),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3), f(4), clip_high=-0.1),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3), f(4), dual_clip=1.0),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3), f(4), kl_coef=0.1),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3), f(4), reference_log_probs=f(4, 3), kl_coef=-0.1),
    lambda f, i: ops.policy_loss(f(4, 3), f(4, 3), f(4), reduction="mean"),
    lambda f, i: ops.embedding(f(5, 4), f(3), sorted_gradient=True),
    lambda f, i: ops.embedding(f(5, 4), i(3).cpu(), sorted_gradient=True),
    lambda f, i: ops.embedding(f(5), i(3), sorted_gradient=True),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call(lambda *s: torch.zeros(*s, device="cuda"), lambda *s: torch.zeros(*s, dtype=torch.long, device="cuda"))


def test_outputs_may_be_changed_in_place_and_second_derivatives_are_refused():
    logits = torch.randn(4, 50, device="cuda", requires_grad=True)
    labels = torch.tensor([1, 2, -100, 4], device="cuda")
    lp = ops.token_log_probs(logits, labels)
    lp *= 2.0
    out = ops.policy_loss(lp[None], lp.detach()[None], torch.ones(1, device="cuda"))
    loss = out.loss
    loss /= 4
    out.kl.add_(1)
    (grad,) = torch.autograd.grad(loss, logits, create_graph=True)
    (want,) = torch.autograd.grad(-2.0 / 16 * torch.log_softmax(logits, -1)[[0, 1, 3], [1, 2, 4]].sum() * (4 / 4), logits)
    assert (grad.detach() - want).abs().max() < 1e-6
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        grad.sum().backward()
    pair = ops.preference_loss(torch.zeros(2, 3, device="cuda", requires_grad=True), None, reduction="none")
    pair.loss.mul_(3.0)
    pair.chosen_rewards.add_(1.0)
    assert pair.loss.item() == pytest.approx(3 * math.log(2), rel=1e-6)


def test_offsets_past_32_bits():
    """2.6e9 logits and a table of 2.2e9 values: the last rows are those of a small call."""
    tokens, vocab = 20011, 128256
    logits = torch.zeros(tokens, vocab, device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator("cuda").manual_seed(0)
    logits[-3:] = torch.randn(3, vocab, generator=gen, device="cuda")
    labels = torch.full((tokens,), -100, device="cuda")
    labels[-3:] = torch.tensor([0, vocab - 1, 77], device="cuda")
    logits.requires_grad_(True)
    lp = ops.token_log_probs(logits, labels)
    (grad,) = torch.autograd.grad(lp.sum(), logits)
    one = torch.ones(3, device="cuda", dtype=torch.float64)
    _check_log_probs(logits.detach()[-3:].double(), labels[-3:], -100, one, 0 * one, lp[-3:], None, grad[-3:], 1.0, torch.bfloat16)
    assert (lp[:-3] == 0).all() and grad[:-3].abs().max() == 0
    del logits, grad
    w = torch.zeros(550_000, 4096, device="cuda", dtype=torch.bfloat16)
    w[-1] = torch.randn(4096, generator=gen, device="cuda")
    w.requires_grad_(True)
    ids = torch.tensor([549_999, 3, 549_999], device="cuda", dtype=torch.int32)
    out = ops.embedding(w, ids, sorted_gradient=True)
    assert torch.equal(out[0], w.detach()[-1]) and torch.equal(out[2], out[0]) and (out[1] == 0).all()
    (grad,) = torch.autograd.grad(out, w, torch.ones_like(out))
    assert (grad[-1] == 2).all() and (grad[3] == 1).all() and grad.sum(dtype=torch.float64).item() == 3 * 4096


def test_on_a_stream_of_its_own_and_twice_at_once():
    """Two streams run the same step on their own inputs at the same time; both give what the default stream gives."""
    def step(seed):
        x, w, labels, g, h = _linear_case(400, 128, 3000, seed)
        labels[::5] = -100
        x.requires_grad_(True)
        w.requires_grad_(True)
        ids = labels.clamp_min(0)
        lp = ops.fused_linear_token_log_probs(x, w, labels)
        cu = torch.tensor([0, 100, 150, 350, 400], device="cuda", dtype=torch.int32)
        pref = ops.preference_loss(lp, lp.detach() - 0.1 * g, cu)
        pol = ops.policy_loss(lp, lp.detach() + 0.3 * h, g, cu_seqlens=cu)
        emb = ops.embedding(w, ids, 0.5, sorted_gradient=True)
        grads = torch.autograd.grad(pref.loss + pol.loss + (emb * x.detach()).sum(), (x, w))
        return [t.detach() for t in (lp, pref.loss, pol.loss, emb, *grads)]

    want = [step(s) for s in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = step(i + 1)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


def test_training_after_inference_mode_and_after_a_raised_status(monkeypatch):
    """The status word is made by the first call, here one under inference mode, and is cleared between a forward pass and its backward pass."""
    monkeypatch.setattr(ops, "_STATUS", {})
    gen = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(5, 64, device="cuda", generator=gen, dtype=torch.bfloat16)
    w = torch.randn(100, 64, device="cuda", generator=gen, dtype=torch.bfloat16)
    labels = torch.tensor([1, 99, -100, 4, 0], device="cuda")
    with torch.inference_mode():
        scored = ops.fused_linear_token_log_probs(x, w, labels)
    x.requires_grad_(True)
    w.requires_grad_(True)
    lp = ops.fused_linear_token_log_probs(x, w, labels)
    assert torch.equal(lp.detach(), scored)
    rows = ops.embedding_sorted(w, labels)  # -100 is not in the table
    with pytest.raises(RuntimeError, match="outside of its table"):
        ops.check_status()
    (lp.sum() + rows.sum()).backward()
    again = torch.autograd.grad(ops.fused_linear_token_log_probs(x, w, labels).sum(), x)[0]
    assert torch.equal(x.grad, again)


def test_main_grad_of_a_recomputed_block_and_a_table_changed_in_place():
    from torch.utils.checkpoint import checkpoint

    gen = torch.Generator("cuda").manual_seed(0)
    ids = torch.randint(0, 100, (7,), device="cuda", generator=gen)

    def block(w):
        return ops.fused_linear_token_log_probs(ops.embedding_sorted(w, ids), w, ids)

    grads = []
    for recompute in (False, True):
        gen.manual_seed(1)
        w = torch.randn(100, 64, device="cuda", generator=gen, dtype=torch.bfloat16).requires_grad_(True)
        w.main_grad = torch.zeros(100, 64, device="cuda")
        lp = checkpoint(block, w, use_reentrant=False) if recompute else block(w)
        lp.sum().backward()
        assert w.grad is None
        grads.append(w.main_grad)
    assert grads[0].abs().sum() > 0 and torch.equal(*grads)

    # the gradient of a lookup does not depend on the table's values
    table = torch.zeros(100, 64, device="cuda", requires_grad=True)
    rows = ops.embedding_sorted(table, ids)
    with torch.no_grad():
        table.add_(1.0)
    rows.sum().backward()
    assert torch.equal(table.grad, torch.bincount(ids, minlength=100).float()[:, None].expand(100, 64))


def test_operands_without_dimensions_are_refused():
    one = torch.tensor(1.0, device="cuda", dtype=torch.bfloat16)
    rows = torch.zeros(3, 8, device="cuda", dtype=torch.bfloat16)
    label = torch.tensor(1, device="cuda")
    for x, w, labels in ((one, rows, label), (rows, one, label.expand(3))):
        with pytest.raises(ValueError):
            ops.fused_linear_token_log_probs(x, w, labels)
