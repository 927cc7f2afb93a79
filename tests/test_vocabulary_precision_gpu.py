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

# ----------------------------------------------------------------------------- rows far from zero, tokens all but certain
def _grid(tokens, vocab, seed):
    """Scores on a grid of 1/16 below 4 in size: exact in every type, and next to a shift too where it is a multiple of 32 below 2^17 (fp32)."""
    gen = torch.Generator("cuda").manual_seed(seed)
    base = torch.randint(-63, 64, (tokens, vocab), generator=gen, device="cuda") / 16
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    g, h = torch.randn(tokens, generator=gen, device="cuda"), torch.randn(tokens, generator=gen, device="cuda")
    return base, labels, g, h


@pytest.mark.parametrize("dtype,shift", [(torch.float32, 96.0), (torch.float32, 1024.0), (torch.float32, -10240.0), (torch.float16, 64.0)])
@pytest.mark.parametrize("tokens,vocab", [(5, 1003), (40, 50000)])
@pytest.mark.parametrize("scale", [1.0, 0.7])
def test_log_probs_do_not_depend_on_where_a_row_lies(dtype, shift, tokens, vocab, scale):
    """A softmax depends on differences alone. Those are exact here, so every later value has to be the same, bit for bit."""
    base, labels, g, h = _grid(tokens, vocab, vocab)
    results = []
    for z in (base, base + shift):
        z = z.to(dtype).requires_grad_(True)
        outs = ops.token_log_probs(z, labels, logit_scale=scale, return_entropy=True)
        results.append((*outs, *torch.autograd.grad(outs, z, (g, h)), *torch.autograd.grad(ops.token_log_probs(z, labels, logit_scale=scale), z, g)))
    for a, b in zip(*results):
        assert torch.equal(a, b), (a.double() - b.double()).abs().max().item()


@pytest.mark.parametrize("shift", [96.0, 1024.0, -10240.0])
@pytest.mark.parametrize("keep", [True, False])
def test_fused_linear_log_probs_do_not_depend_on_where_a_row_lies(shift, keep):
    """Logits on the grid: row t of x takes column 1 + t of the weight, and column 0 adds the shift to all of them. All products and their sums are exact."""
    tokens, hidden, vocab = 63, 64, 5003
    base, labels, g, h = _grid(tokens, vocab, 3)
    x = torch.zeros(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1.0
    x[torch.arange(tokens), 1 + torch.arange(tokens)] = 1.0
    results = []
    for s in (0.0, shift):
        w = torch.zeros(vocab, hidden, device="cuda", dtype=torch.bfloat16)
        w[:, 0], w[:, 1:] = s, base.t()
        x.requires_grad_(True), w.requires_grad_(True)
        outs = ops.fused_linear_token_log_probs(x, w, labels, return_entropy=True, keep_logits=keep)
        dx, dw = torch.autograd.grad(outs, (x, w), (g, h))
        results.append((*outs, dx[:, 1:], dw))
    for a, b in zip(*results):
        assert torch.equal(a, b), (a.double() - b.double()).abs().max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top", [20.0, 40.0, 100.0])
def test_no_log_probability_is_above_zero(dtype, top):
    gen = torch.Generator("cuda").manual_seed(int(top))
    tokens, vocab = 600, 4001
    logits = (2.5 * torch.randn(tokens, vocab, generator=gen, device="cuda")).to(dtype)
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    logits[torch.arange(tokens), labels] += top
    lp, entropy = ops.token_log_probs(logits, labels, return_entropy=True)
    want = logits.double().log_softmax(-1).gather(1, labels[:, None])[:, 0]
    assert (lp <= 0).all() and (entropy >= 0).all()
    # the sum is 1 + r with r < 1 in all but a few rows: its additions and the logarithm round by half a step of it (2^-24) in each of the
    # (at most 4001 / 256 / 4 + 24 additions and 24 merges) steps that still move it; terms of r are good to 2^-20
    assert ((lp.double() - want).abs() <= 52 * 2.0**-24 + 2.0**-20 * want.abs()).all()
    if top >= 40:
        assert lp.abs().max() <= 2.0**-23  # what is left of the sum next to 1


@pytest.mark.parametrize("top", [24.0, 40.0, 96.0])
def test_no_log_probability_from_hidden_states_is_above_zero(top):
    tokens, hidden, vocab = 63, 64, 4001
    base, labels, _, _ = _grid(tokens, vocab, 5)
    x = torch.zeros(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    x[torch.arange(tokens), 1 + torch.arange(tokens)] = 1.0
    base[torch.arange(tokens), labels] = top
    w = torch.zeros(vocab, hidden, device="cuda", dtype=torch.bfloat16)
    w[:, 1:] = base.t()
    lp, entropy = ops.fused_linear_token_log_probs(x, w, labels, return_entropy=True)
    want = base.double().log_softmax(-1).gather(1, labels[:, None])[:, 0]
    assert (lp <= 0).all() and (entropy >= 0).all()
    assert ((lp.double() - want).abs() <= 52 * 2.0**-24 + 2.0**-20 * want.abs()).all()

# ----------------------------------------------------------------------------- long sums of the embedding's gradient
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hidden", [(100, 64), (1000, 64), (200001, 16), (30000, 3)])
@pytest.mark.parametrize("into_buffer", [False, True])
def test_the_gradient_of_a_frequent_token_is_a_sum_of_few_roundings(dtype, tokens, hidden, into_buffer):
    gen = torch.Generator("cuda").manual_seed(tokens)
    w = torch.zeros(7, hidden, device="cuda", dtype=dtype, requires_grad=True)
    ids = torch.full((tokens,), 3, device="cuda")
    ids[::97] = 5
    dout = (1 + torch.rand(tokens, hidden, generator=gen, device="cuda")).to(dtype) / 64
    exact = torch.zeros(7, hidden, device="cuda", dtype=torch.float64).index_add_(0, ids, dout.double())
    if into_buffer:
        w.main_grad = torch.zeros(7, hidden, device="cuda")
    out = ops.embedding(w, ids, sorted_gradient=True)
    if into_buffer:
        out.backward(dout)
        grad = w.main_grad
    else:
        (grad,) = torch.autograd.grad(out, w, dout)
    # fp32 rows: a chunk's sum is rounded once, their total once, all values have one sign. 16-bit rows hold at most 11 bits, and sums of
    # up to 128 of them in one binade below 2^18 steps are exact.
    half = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-24 if into_buffer else 2.0**-8, torch.float16: 2.0**-24 if into_buffer else 2.0**-11}[dtype]
    assert ((grad.double() - exact).abs() <= (half + 2.0**-24) * (1 + 2.0**-20) * exact).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,hidden", [(8192, 1024), (4099, 64)])
def test_the_order_of_the_embeddings_sums_does_not_depend_on_addresses(dtype, tokens, hidden):
    """Upstream gradients and buffers that start at an odd element are read and written narrowly, and give the same bits."""
    gen = torch.Generator("cuda").manual_seed(hidden)
    ids = torch.randint(0, 30, (tokens,), generator=gen, device="cuda")
    dout = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype)
    shifted = torch.empty(tokens * hidden + 1, device="cuda", dtype=dtype)[1:].view(tokens, hidden).copy_(dout)
    buffer = torch.zeros(30 * hidden + 1, device="cuda")[1:].view(30, hidden)
    grads = []
    for up, main_grad in ((dout, torch.zeros(30, hidden, device="cuda")), (shifted, torch.zeros(30, hidden, device="cuda")), (dout, buffer)):
        w = torch.zeros(30, hidden, device="cuda", dtype=dtype, requires_grad=True)
        out = ops.embedding(w, ids, 0.3, sorted_gradient=True)
        (grad,) = torch.autograd.grad(out, w, up)
        w.main_grad = main_grad
        ops.embedding(w, ids, 0.3, sorted_gradient=True).backward(up)
        grads.append((grad, main_grad))
    for grad, main_grad in grads[1:]:
        assert torch.equal(grad, grads[0][0]) and torch.equal(main_grad, grads[0][1])
