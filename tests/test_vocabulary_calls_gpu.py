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


# ----------------------------------------------------------------------------- operands that no tensor map can describe
def _operands(tokens, hidden=64, vocab=300):
    gen = torch.Generator("cuda").manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").bfloat16()
    w = (torch.randn(vocab, hidden, generator=gen, device="cuda") / 8).bfloat16()
    return x, w, torch.randint(0, vocab, (tokens,), generator=gen, device="cuda"), torch.randn(tokens, generator=gen, device="cuda")


def _at_an_odd_address(t):
    return torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)[1:].view(t.shape).copy_(t)


def _in_odd_rows(t):
    return torch.zeros(t.shape[0], t.shape[1] + 3, device=t.device, dtype=t.dtype)[:, : t.shape[1]].copy_(t)


def _of_one_column_stride(t):
    return t.t().contiguous().t()


@pytest.mark.parametrize("place", [_at_an_odd_address, _in_odd_rows, _of_one_column_stride])
@pytest.mark.parametrize("tokens,vocab", [(1, 300), (1, 1), (20, 300)])
@pytest.mark.parametrize("into_buffer", [False, True])
def test_fused_linear_log_probs_of_operands_that_lie_oddly(place, tokens, vocab, into_buffer):
    x, w, labels, g = _operands(tokens, vocab=vocab)
    results = []
    for a, b in ((x, w), (place(x), w), (x, place(w)), (place(x), place(w))):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        if into_buffer:
            b.main_grad = torch.zeros(vocab, 64, device="cuda")
        lp = ops.fused_linear_token_log_probs(a, b, labels)
        lp.backward(g)
        assert (b.grad is None) == into_buffer
        with torch.no_grad():
            assert torch.equal(ops.fused_linear_token_log_probs(a, b, labels), lp)
        results.append((lp.detach(), a.grad, b.main_grad if into_buffer else b.grad))
    for result in results[1:]:
        for got, want in zip(result, results[0]):
            assert torch.equal(got, want)


@pytest.mark.parametrize("place", [_at_an_odd_address, _in_odd_rows, _of_one_column_stride])
def test_a_table_that_lies_oddly_finds_its_main_grad(place):
    _, w, ids, _ = _operands(20)
    dout = torch.randn(20, 64, device="cuda").bfloat16()
    buffers = []
    for table in (w, place(w)):
        table = table.detach().requires_grad_(True)
        table.main_grad = torch.zeros(300, 64, device="cuda")
        out = ops.embedding(table, ids, sorted_gradient=True)
        assert torch.equal(out, w[ids])
        out.backward(dout)
        assert table.grad is None
        buffers.append(table.main_grad)
    assert buffers[0].abs().max() > 0 and torch.equal(*buffers)


# ----------------------------------------------------------------------------- the deterministic switch
@pytest.fixture
def deterministic():
    torch.use_deterministic_algorithms(True)
    yield
    torch.use_deterministic_algorithms(False)


def test_fp32_tables_keep_their_embedding_under_deterministic_algorithms(deterministic, monkeypatch):
    w = torch.randn(50, 8, device="cuda", requires_grad=True)
    ids = torch.randint(0, 50, (40,), device="cuda")

    def never():
        raise AssertionError("the extension is not needed here")

    monkeypatch.setattr(ops, "native", never)
    out = ops.embedding(w, ids, 2.0)
    (grad,) = torch.autograd.grad(out.square().sum(), w, create_graph=True)
    (second,) = torch.autograd.grad(grad.sum(), w)  # out^2 = 4 w[ids]^2, twice differentiated: 8 for each time an id appears
    assert torch.equal(second, 8.0 * torch.bincount(ids, minlength=50).float()[:, None].expand(50, 8))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        assert (torch.autograd.forward_ad.unpack_dual(ops.embedding(dual, ids, 2.0)).tangent == 2).all()


@pytest.mark.parametrize("kind", [torch.int16, torch.uint8, torch.int32])
def test_bf16_tables_take_any_integer_ids_under_deterministic_algorithms(deterministic, kind):
    w = torch.randn(50, 16, device="cuda").bfloat16().requires_grad_(True)
    ids = torch.randint(0, 50, (3, 40), device="cuda")
    (want,) = torch.autograd.grad(ops.embedding(w, ids, sorted_gradient=True).sum(), w)
    out = ops.embedding(w, ids.to(kind))
    assert torch.equal(out, w[ids]) and torch.equal(torch.autograd.grad(out.sum(), w)[0], want)


# ----------------------------------------------------------------------------- values changed between the passes
@pytest.mark.parametrize("padded", [False, True])
def test_log_probs_may_be_changed_between_the_passes_of_the_losses(padded):
    """Neither loss needs them again: what their gradients take is formed in the forward pass."""
    shape = (4, 25) if padded else (100,)
    cu = None if padded else torch.tensor([0, 10, 10, 70, 100], device="cuda", dtype=torch.int32)
    values, old = torch.randn(shape, device="cuda") / 10, torch.randn(shape, device="cuda") / 10
    for loss in (lambda lp: ops.preference_loss(lp, old, cu).loss, lambda lp: ops.policy_loss(lp, old, torch.ones(4, device="cuda"), cu_seqlens=cu).loss):
        grads = []
        for change in (False, True):
            lp = values.clone().requires_grad_(True)
            out = loss(lp)
            if change:
                with torch.no_grad():
                    lp.zero_()
            grads.append(torch.autograd.grad(out, lp)[0])
        assert grads[0].abs().max() > 0 and torch.equal(*grads)


# ----------------------------------------------------------------------------- launch sites
def test_backward_passes_open_their_sites():
    from lm_engine.ops import timeline

    x, w, labels, g = _operands(40)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    cu = torch.tensor([0, 10, 20, 30, 40], device="cuda", dtype=torch.int32)

    def step():
        rows = ops.embedding(w, labels, sorted_gradient=True)
        lp = ops.fused_linear_token_log_probs(rows + x, w, labels, keep_logits=False)
        lp = lp + ops.token_log_probs(x @ w.t(), labels)
        loss = ops.preference_loss(lp, None, cu).loss + ops.policy_loss(lp, lp.detach(), torch.ones(4, device="cuda"), cu_seqlens=cu).loss
        return torch.autograd.grad(loss, (x, w))

    plain = step()
    both = {"token_log_probs": ["token_log_probs.bwd"], "preference_loss": ["preference_loss.bwd"], "policy_loss": ["policy_loss.bwd"],
            "embedding": ["embedding.bwd"], "loss.lm_head.log_probs": ["loss.lm_head.dlogits", "loss.lm_head.dgrad", "loss.lm_head.wgrad"]}
    timeline.enable_timing()
    try:
        timed = step()
        sites = timeline.report()
    finally:
        timeline.enable_timing(False)
    for forward, backward in both.items():
        for name in (forward, *backward):
            assert sites[name]["calls"] == 1 and sites[name]["ms"] > 0, name
    step()
    assert timeline.report().keys() == sites.keys() and all(timeline.report()[n]["calls"] == sites[n]["calls"] for n in sites)
    for a, b in zip(plain, timed):
        assert torch.equal(a, b)


def test_an_error_of_a_site_reaches_the_caller():
    _, w, ids, _ = _operands(5)
    w.requires_grad_(True)
    out = ops.embedding(w, ids, sorted_gradient=True).sum()

    def refuse(name):
        raise KeyError(name)

    ops.native().set_site(refuse)
    try:
        with pytest.raises(RuntimeError, match="launch site embedding.bwd: KeyError"):
            out.backward(retain_graph=True)
    finally:
        ops.native().set_site(None)
    out.backward()
    assert w.grad.abs().max() == torch.bincount(ids).max()
