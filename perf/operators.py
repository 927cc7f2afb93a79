"""Operators over the vocabulary in a preference or reward tuning step, and the cases they are measured at.

Five operators: the log-probabilities (and entropies) of given tokens under a row of logits; the same from hidden
states and the output projection's weight, without keeping the logits; the preference loss over pairs of answers; the
clipped policy loss with a KL term; and the embedding lookup whose gradient is summed in sorted token order. ``run``
holds each in its plain form (elementary torch operations in 32 bits, rounded once) and as the call a user makes.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # scoring a handful of answers during generation: the smallest call, latency counts
        dict(name="logp-score-32x49152-bf16", op="logp", tokens=32, vocab=49152, pitch=49152, dtype="bf16", entropy=False, train=False),
        # one micro-batch of a tuning step on materialised logits (tensor of the model's forward pass), both directions
        dict(name="logp-train-4096x128256-bf16", op="logp", tokens=4096, vocab=128256, pitch=128256, dtype="bf16", entropy=False, train=True),
        # fp32 logits whose vocabulary was padded to a multiple of 64 and sliced back: odd width, strided rows, entropy bonus
        dict(name="logp-train-1531x50001of50304-fp32-entropy", op="logp", tokens=1531, vocab=50001, pitch=50304, dtype="fp32", entropy=True, train=True),
        # reference model's pass over a ragged batch: no gradient, the logits never exist
        dict(name="linear-score-777x2048x49152", op="linear", tokens=777, hidden=2048, vocab=49152, entropy=True, train=False),
        # the policy's pass of the 8B configuration: gradients of hidden states and of the output weight
        dict(name="linear-train-4096x4096x128256", op="linear", tokens=4096, hidden=4096, vocab=128256, entropy=False, train=True),
        # preference loss of a small micro-batch (4 pairs) and of a large gathered batch of long answers
        dict(name="preference-4x300", op="preference", pairs=4, length=300, loss_type="sigmoid", smoothing=0.0, average=False, train=True),
        dict(name="preference-256x4096-smoothed", op="preference", pairs=256, length=4096, loss_type="sigmoid", smoothing=0.1, average=False, train=True),
        # policy loss of one micro-batch with one advantage per answer, and of a whole rollout with one per token
        dict(name="policy-16x256-sequence", op="policy", sequences=16, length=256, per_token=False, kl=True, reduction="sequence_mean", train=True),
        dict(name="policy-1024x2048-token", op="policy", sequences=1024, length=2048, per_token=True, kl=True, reduction="token_mean", train=True),
        # embedding of a short packed batch, of a long one of the 8B configuration, and of one that is mostly one padding token
        dict(name="embedding-512x768of50304-bf16", op="embedding", tokens=512, hidden=768, vocab=50304, dtype="bf16", scale=1.0, repeat=0.0),
        dict(name="embedding-32768x4096of128256-bf16", op="embedding", tokens=32768, hidden=4096, vocab=128256, dtype="bf16", scale=12.0, repeat=0.0),
        dict(name="embedding-10001x1536of49152-fp32-padded", op="embedding", tokens=10001, hidden=1536, vocab=49152, dtype="fp32", scale=0.5, repeat=0.4),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logp", "linear", "preference", "policy", "embedding"])
    if op == "logp":
        vocab = _log_int(rng, 1000, 128256)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        pitch = vocab + rng.choice([0, 0, rng.randrange(1, 64)])
        tokens = _log_int(rng, 1, max(2, min(8192, 4096 * 128256 * 2 // (pitch * DTYPES[dtype].itemsize))))
        return dict(op=op, tokens=tokens, vocab=vocab, pitch=pitch, dtype=dtype, entropy=rng.random() < 0.4, train=rng.random() < 0.7)
    if op == "linear":
        hidden = 8 * _log_int(rng, 64, 512)
        vocab = _log_int(rng, 1000, 128256)
        return dict(op=op, tokens=_log_int(rng, 1, 4096), hidden=hidden, vocab=vocab, entropy=rng.random() < 0.4, train=rng.random() < 0.6)
    if op == "preference":
        pairs = _log_int(rng, 1, 256)
        return dict(op=op, pairs=pairs, length=_log_int(rng, 1, 4096), loss_type=rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"]),
                    smoothing=rng.choice([0.0, 0.1]), average=rng.random() < 0.3, train=rng.random() < 0.8)
    if op == "policy":
        sequences = _log_int(rng, 1, 1024)
        return dict(op=op, sequences=sequences, length=_log_int(rng, 1, 2048), per_token=rng.random() < 0.5, kl=rng.random() < 0.7,
                    reduction=rng.choice(["token_mean", "sequence_mean", "sum"]), train=rng.random() < 0.8)
    return dict(op="embedding", tokens=_log_int(rng, 1, 32768), hidden=8 * _log_int(rng, 8, 512), vocab=_log_int(rng, 300, 128256),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), scale=rng.choice([1.0, 0.5, 12.0]), repeat=rng.choice([0.0, 0.0, 0.4, 0.9]))


# ---------------------------------------------------------------------------------------------------- inputs
IGNORE = -100
BETA = 0.1
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.05


def _labels(tokens, vocab, gen):
    """Token labels of which one in eight (prompt tokens) is ignored."""
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    ignored = torch.randperm(tokens, generator=gen, device="cuda")[: tokens // 8]
    labels[ignored] = IGNORE
    return labels


def _lengths(count, length):
    """``count`` ragged lengths between half of ``length`` and ``length`` (a case's shape, the same for every seed)."""
    return [length - (7919 * (i + 1)) % (length // 2 + 1) for i in range(count)]


def _cu_seqlens(count, length):
    """Their running sum as the packed models take it (int32, on the device)."""
    n = torch.tensor([0] + _lengths(count, length), device="cuda")
    return n.cumsum(0).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    state = dict(case=case)
    if case["op"] == "logp":
        dtype = DTYPES[case["dtype"]]
        tokens, vocab = case["tokens"], case["vocab"]
        buffer = torch.randn(tokens, case["pitch"], generator=gen, device="cuda", dtype=torch.float32).mul_(2.5).to(dtype)
        logits = buffer[:, :vocab]
        labels = _labels(tokens, vocab, gen)
        # trained models put much of the mass on the label in about half of the rows
        sure = torch.rand(tokens, generator=gen, device="cuda") < 0.5
        rows = torch.nonzero(sure & (labels != IGNORE)).flatten()
        buffer[rows, labels[rows]] += 12.0
        state.update(logits=logits.detach(), labels=labels, dlogp=randn(tokens) / tokens, dentropy=randn(tokens) / tokens)
        if case["train"]:
            state["logits"].requires_grad_(True)
    elif case["op"] == "linear":
        tokens, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
        x = randn(tokens, hidden).to(torch.bfloat16)
        weight = torch.randn(vocab, hidden, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(2.0 / math.sqrt(hidden))
        labels = _labels(tokens, vocab, gen)
        state.update(x=x, weight=weight, labels=labels, dlogp=randn(tokens), dentropy=0.1 * randn(tokens))
        if case["train"]:
            x.requires_grad_(True)
            weight.requires_grad_(True)
    elif case["op"] == "preference":
        cu = _cu_seqlens(2 * case["pairs"], case["length"])
        total = int(cu[-1])
        reference = -2.0 * torch.rand(total, generator=gen, device="cuda").square()
        log_probs = reference + 0.1 * randn(total)
        keep = torch.rand(total, generator=gen, device="cuda") < 0.75
        state.update(log_probs=log_probs, reference=reference, cu=cu, keep=keep)
        if case["train"]:
            log_probs.requires_grad_(True)
    elif case["op"] == "policy":
        cu = _cu_seqlens(case["sequences"], case["length"])
        total = int(cu[-1])
        old = -2.0 * torch.rand(total, generator=gen, device="cuda").square()
        log_probs = old + 0.15 * randn(total)
        reference = old + 0.2 * randn(total)
        keep = torch.rand(total, generator=gen, device="cuda") < 0.75
        advantages = randn(total if case["per_token"] else case["sequences"])
        state.update(log_probs=log_probs, old=old, reference=reference if case["kl"] else None, advantages=advantages, cu=cu, keep=keep)
        if case["train"]:
            log_probs.requires_grad_(True)
    else:
        dtype = DTYPES[case["dtype"]]
        tokens, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
        weight = torch.randn(vocab, hidden, generator=gen, device="cuda", dtype=torch.float32).mul_(0.02).to(dtype)
        # token frequencies fall off like 1 / rank; `repeat` of the tokens are one padding id
        u = torch.rand(tokens, generator=gen, device="cuda")
        ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
        ids[torch.rand(tokens, generator=gen, device="cuda") < case["repeat"]] = vocab // 2
        state.update(weight=weight.requires_grad_(True), ids=ids, dout=randn(tokens, hidden).to(dtype))
    return state


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _RUN_OWN[state["case"]["op"]](state, state["case"])
    return _RUN_PLAIN[state["case"]["op"]](state, state["case"])


def _own_logp(s, case):
    from lm_engine import ops

    out = ops.token_log_probs(s["logits"], s["labels"], return_entropy=case["entropy"])
    outs = out if case["entropy"] else (out,)
    if not case["train"]:
        return outs
    (grad,) = torch.autograd.grad(outs, [s["logits"]], [s["dlogp"], s["dentropy"]][: len(outs)])
    return (*(o.detach() for o in outs), grad)


def _own_linear(s, case):
    from lm_engine import ops

    out = ops.fused_linear_token_log_probs(s["x"], s["weight"], s["labels"], return_entropy=case["entropy"])
    outs = out if case["entropy"] else (out,)
    if not case["train"]:
        return outs
    grads = torch.autograd.grad(outs, [s["x"], s["weight"]], [s["dlogp"], s["dentropy"]][: len(outs)])
    return (*(o.detach() for o in outs), *grads)


def _own_preference(s, case):
    from lm_engine import ops

    loss, chosen, rejected = ops.preference_loss(
        s["log_probs"], s["reference"], s["cu"], beta=BETA, loss_type=case["loss_type"], label_smoothing=_smoothing(case),
        average_log_probs=case["average"], mask=s["keep"])
    if not case["train"]:
        return loss, chosen, rejected
    (grad,) = torch.autograd.grad(loss, [s["log_probs"]])
    return loss.detach(), chosen, rejected, grad


def _own_policy(s, case):
    from lm_engine import ops

    loss, kl, clipped = ops.policy_loss(
        s["log_probs"], s["old"], s["advantages"], reference_log_probs=s["reference"], cu_seqlens=s["cu"], mask=s["keep"],
        clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF if case["kl"] else 0.0, reduction=case["reduction"])
    if not case["train"]:
        return loss, kl, clipped
    (grad,) = torch.autograd.grad(loss, [s["log_probs"]])
    return loss.detach(), kl, clipped, grad


def _own_embedding(s, case):
    from lm_engine import ops

    out = ops.embedding(s["weight"], s["ids"], case["scale"], sorted_gradient=True)
    (grad,) = torch.autograd.grad(out, [s["weight"]], s["dout"])
    return out.detach(), grad


def _smoothing(case):
    return case["smoothing"] if case["loss_type"] == "sigmoid" else 0.0


def _log_softmax_parts(z, labels):
    """Row maximum shifted log-softmax pieces of fp32 scores: (log-probability of the label, entropy, probabilities, log-probabilities)."""
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    logp = z - torch.log(total)
    p = e / total
    kept = labels != IGNORE
    picked = logp.gather(1, labels.clamp_min(0)[:, None])[:, 0]
    entropy = -(p * logp).sum(-1)
    return torch.where(kept, picked, 0.0), torch.where(kept, entropy, 0.0), p, logp, kept


def _score_gradient(p, logp, entropy, labels, kept, dlogp, dentropy):
    """d(score) = g (onehot - p) - h p (log p + H), zero in ignored rows."""
    g = torch.where(kept, dlogp, 0.0)[:, None]
    dz = -p * g
    dz.scatter_add_(1, labels.clamp_min(0)[:, None], g)
    if dentropy is not None:
        h = torch.where(kept, dentropy, 0.0)[:, None]
        dz -= h * p * (logp + entropy[:, None])
    return dz


def _plain_logp(s, case):
    logits = s["logits"].detach()
    picked, entropy, p, logp, kept = _log_softmax_parts(logits.float(), s["labels"])
    outs = (picked, entropy) if case["entropy"] else (picked,)
    if not case["train"]:
        return outs
    dz = _score_gradient(p, logp, entropy, s["labels"], kept, s["dlogp"], s["dentropy"] if case["entropy"] else None)
    return (*outs, dz.to(logits.dtype))


def _plain_linear(s, case):
    x, weight = s["x"].detach().float(), s["weight"].detach().float()
    picked, entropy, p, logp, kept = _log_softmax_parts(x @ weight.t(), s["labels"])
    outs = (picked, entropy) if case["entropy"] else (picked,)
    if not case["train"]:
        return outs
    dz = _score_gradient(p, logp, entropy, s["labels"], kept, s["dlogp"], s["dentropy"] if case["entropy"] else None)
    return (*outs, (dz @ weight).to(torch.bfloat16), (dz.t() @ x).to(torch.bfloat16))


def _sequence_of_token(cu, total):
    """Index of the sequence that each packed token belongs to."""
    return torch.searchsorted(cu[1:].contiguous(), torch.arange(total, device=cu.device, dtype=cu.dtype), right=True)


def _plain_preference(s, case):
    log_probs, cu, keep = s["log_probs"].detach(), s["cu"], s["keep"]
    count = 2 * case["pairs"]
    seq = _sequence_of_token(cu, log_probs.numel())
    # long sums of small differences: added in 64 bits
    d = torch.where(keep, log_probs.double() - s["reference"].double(), 0.0)
    sums = torch.zeros(count, device=d.device, dtype=torch.float64).index_add_(0, seq, d)
    tokens = torch.zeros(count, device=d.device, dtype=torch.float64).index_add_(0, seq, keep.double())
    if case["average"]:
        sums = sums / tokens.clamp_min(1.0)
    chosen, rejected = sums[: case["pairs"]], sums[case["pairs"] :]
    margin = BETA * (chosen - rejected)
    eps = _smoothing(case)
    if case["loss_type"] == "sigmoid":
        losses = (1 - eps) * torch.logaddexp(torch.zeros_like(margin), -margin) + eps * torch.logaddexp(torch.zeros_like(margin), margin)
        slope = -BETA * ((1 - eps) * torch.sigmoid(-margin) - eps * torch.sigmoid(margin))
    elif case["loss_type"] == "hinge":
        losses = (1 - margin).clamp_min(0.0)
        slope = torch.where(margin < 1, -BETA, 0.0).to(margin.dtype)
    else:
        losses = (chosen - rejected - 1 / (2 * BETA)).square()
        slope = 2 * (chosen - rejected - 1 / (2 * BETA))
    outs = (losses.mean().float(), (BETA * chosen).float(), (BETA * rejected).float())
    if not case["train"]:
        return outs
    per_sequence = torch.cat([slope, -slope]) / case["pairs"]
    if case["average"]:
        per_sequence = per_sequence / tokens.clamp_min(1.0)
    return (*outs, torch.where(keep, per_sequence[seq], 0.0).float())


def _plain_policy(s, case):
    log_probs, old, cu, keep = s["log_probs"].detach(), s["old"], s["cu"], s["keep"]
    total, count = log_probs.numel(), case["sequences"]
    seq = _sequence_of_token(cu, total)
    a = s["advantages"] if case["per_token"] else s["advantages"][seq]
    # a ratio next to a clipping border decides whether its token has a gradient: formed and compared in 64 bits
    ratio = torch.exp(log_probs.double() - old.double())
    clipped_ratio = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    active = a * clipped_ratio < a * ratio
    ratio, clipped_ratio = ratio.float(), clipped_ratio.float()
    surrogate = torch.where(active, -a * clipped_ratio, -a * ratio)
    slope = torch.where(active, 0.0, -a * ratio)
    kl = torch.zeros_like(surrogate)
    if case["kl"]:
        d = (s["reference"] - log_probs).double()  # exp(d) - 1 - d cancels for small d: 64 bits
        kl = (torch.expm1(d) - d).float()
        slope = slope - KL_COEF * torch.expm1(d).float()
    values = torch.where(keep, surrogate + KL_COEF * kl, 0.0).double()
    kept = keep.double()
    tokens = kept.sum()
    if case["reduction"] == "sequence_mean":
        per_sequence = torch.zeros(count, device=kept.device, dtype=torch.float64).index_add_(0, seq, kept)
        used = (per_sequence > 0).double().sum().clamp_min(1.0)
        weight = 1.0 / (per_sequence.clamp_min(1.0)[seq] * used)
    elif case["reduction"] == "token_mean":
        weight = torch.full_like(kept, 1.0) / tokens.clamp_min(1.0)
    else:
        weight = torch.full_like(kept, 1.0)
    outs = ((values * weight).sum().float(), ((kl.double() * kept).sum() / tokens.clamp_min(1.0)).float(),
            ((active.double() * kept).sum() / tokens.clamp_min(1.0)).float())
    if not case["train"]:
        return outs
    return (*outs, torch.where(keep, slope.double() * weight, 0.0).float())


def _plain_embedding(s, case):
    weight, ids, dout = s["weight"].detach(), s["ids"], s["dout"]
    out = (weight[ids].float() * case["scale"]).to(weight.dtype)
    # thousands of rows meet in a frequent token's sum: 64 bits where the result keeps more than 16
    wide = torch.float64 if weight.dtype == torch.float32 else torch.float32
    grad = torch.zeros(weight.shape, device=weight.device, dtype=wide)
    grad.index_add_(0, ids, dout.to(wide) * case["scale"])
    return out, grad.to(weight.dtype)


_RUN_OWN = dict(logp=_own_logp, linear=_own_linear, preference=_own_preference, policy=_own_policy, embedding=_own_embedding)
_RUN_PLAIN = dict(logp=_plain_logp, linear=_plain_linear, preference=_plain_preference, policy=_plain_policy, embedding=_plain_embedding)


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "logp":
        kept = case["tokens"] - case["tokens"] // 8
        size = DTYPES[case["dtype"]].itemsize
        one = case["tokens"] * case["vocab"]
        read = kept * case["vocab"] * size + case["tokens"] * 8
        out = case["tokens"] * 4 * (2 if case["entropy"] else 1)
        flops = 4 * kept * case["vocab"]
        if case["train"]:
            return dict(bytes=read + 2 * out + one * size, flops=2 * flops)
        return dict(bytes=read + out, flops=flops)
    if case["op"] == "linear":
        kept = case["tokens"] - case["tokens"] // 8
        product = 2 * kept * case["hidden"] * case["vocab"]
        matrices = 2 * (case["tokens"] + case["vocab"]) * case["hidden"]
        rows = case["tokens"] * (8 + 4 * (2 if case["entropy"] else 1))
        if case["train"]:
            return dict(bytes=2 * matrices + 2 * rows, flops=3 * product)
        return dict(bytes=matrices + rows, flops=product)
    if case["op"] == "preference":
        tokens = sum(_lengths(2 * case["pairs"], case["length"]))
        return dict(bytes=tokens * (4 + 4 + 1 + (4 if case["train"] else 0)) + case["pairs"] * 24, flops=4 * tokens)
    if case["op"] == "policy":
        tokens = sum(_lengths(case["sequences"], case["length"]))
        per_token = 4 + 4 + 1 + (4 if case["per_token"] else 0) + (4 if case["kl"] else 0) + (4 if case["train"] else 0)
        return dict(bytes=tokens * per_token + case["sequences"] * 8, flops=20 * tokens)
    size = DTYPES[case["dtype"]].itemsize
    values = case["tokens"] * case["hidden"]
    # table rows read once for each distinct token (expected number under 1 / rank frequencies), output, upstream
    # gradient and the whole weight gradient
    drawn, norm = case["tokens"] * (1 - case["repeat"]), math.log(case["vocab"] + 1.0)
    distinct = sum(-math.expm1(-drawn * math.log1p(1.0 / (k + 1)) / norm) for k in range(case["vocab"]))
    return dict(bytes=int(size * (distinct * case["hidden"] + 2 * values + case["vocab"] * case["hidden"]) + 8 * case["tokens"]), flops=2 * values)


# ---------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_linear_rows(z, labels, dlogp, dentropy):
    """Log-probability, entropy and score gradient of rows of 64-bit scores (`z` is overwritten by the gradient)."""
    lse = torch.logsumexp(z, dim=1)
    z -= lse[:, None]
    valid = (labels != IGNORE).double()
    index = labels.clamp_min(0)
    at_label = z[torch.arange(z.shape[0], device=z.device), index] * valid
    p = z.exp()
    h = -torch.einsum("tv,tv->t", p, z)
    if dlogp is None:
        return at_label, h * valid, None
    z += h[:, None]
    z *= (dentropy.double() * valid)[:, None]
    z += (dlogp.double() * valid)[:, None]
    z *= -p
    z[torch.arange(z.shape[0], device=z.device), index] += dlogp.double() * valid
    return at_label, h * valid, z


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("logp", "linear"):
        train = case["train"]
        dlogp = s["dlogp"] if train else None
        dentropy = (s["dentropy"] if case["entropy"] else torch.zeros_like(s["dlogp"])) if train else None
        if case["op"] == "logp":
            z = s["logits"].detach().double()
        else:
            x, w = s["x"].detach().double(), s["weight"].detach().double()
            z = torch.mm(x, w.T)
        logp, h, dz = _exact_linear_rows(z, s["labels"], dlogp, dentropy)
        outs = (logp, h) if case["entropy"] else (logp,)
        if not train:
            return outs
        if case["op"] == "logp":
            return (*outs, dz)
        return (*outs, torch.mm(dz, w), torch.mm(dz.T, x))
    if case["op"] == "preference":
        lp = s["log_probs"].detach().double().requires_grad_(True)
        lengths = (s["cu"][1:] - s["cu"][:-1]).long()
        seq = torch.repeat_interleave(torch.arange(lengths.numel(), device="cuda"), lengths)
        m = s["keep"].double()
        ratio = torch.zeros(lengths.numel(), device="cuda", dtype=torch.float64).scatter_add(0, seq, (lp - s["reference"].double()) * m)
        if case["average"]:
            n = torch.zeros_like(ratio).detach().scatter_add(0, seq, m)
            ratio = ratio / torch.where(n == 0, 1.0, n)
        w, l = ratio.chunk(2)
        if case["loss_type"] == "sigmoid":
            e = _smoothing(case)
            per_pair = -(1 - e) * torch.nn.functional.logsigmoid(BETA * (w - l)) - e * torch.nn.functional.logsigmoid(BETA * (l - w))
        elif case["loss_type"] == "hinge":
            per_pair = torch.relu(1 - BETA * (w - l))
        else:
            per_pair = (w - l - 0.5 / BETA) ** 2
        loss = per_pair.sum() / per_pair.numel()
        outs = (loss.detach(), BETA * w.detach(), BETA * l.detach())
        return (*outs, *torch.autograd.grad(loss, lp)) if case["train"] else outs
    if case["op"] == "policy":
        lp = s["log_probs"].detach().double().requires_grad_(True)
        lengths = (s["cu"][1:] - s["cu"][:-1]).long()
        seq = torch.repeat_interleave(torch.arange(lengths.numel(), device="cuda"), lengths)
        a = s["advantages"].double()
        a = a if case["per_token"] else torch.repeat_interleave(a, lengths)
        r = (lp - s["old"].double()).exp()
        bounded = r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
        objective = torch.minimum(a * r, a * bounded)
        m = s["keep"].double()
        n = m.sum().clamp_min(1.0)
        kl = torch.zeros_like(objective)
        if case["kl"]:
            kl = (s["reference"].double() - lp).expm1() - (s["reference"].double() - lp)
        term = (KL_COEF * kl - objective) * m
        if case["reduction"] == "token_mean":
            loss = term.sum() / n
        elif case["reduction"] == "sum":
            loss = term.sum()
        else:
            length = torch.zeros(lengths.numel(), device="cuda", dtype=torch.float64).scatter_add(0, seq, m)
            means = torch.zeros_like(length).scatter_add(0, seq, term) / torch.where(length == 0, 1.0, length)
            loss = means.sum() / (length > 0).sum().clamp_min(1)
        fraction = ((a * bounded < a * r).double() * m).sum() / n
        outs = (loss.detach(), ((kl * m).sum() / n).detach(), fraction.detach())
        return (*outs, *torch.autograd.grad(loss, lp)) if case["train"] else outs
    w, d, ids = s["weight"].detach().double(), s["dout"].double(), s["ids"]
    grad = torch.zeros_like(w).index_put_((ids,), d * case["scale"], accumulate=True)
    return torch.index_select(w, 0, ids) * case["scale"], grad
