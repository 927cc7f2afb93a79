"""Operators over the vocabulary for preference and reward tuning.

* :func:`token_log_probs`: log-probabilities (and entropies) of given tokens under rows of logits
* :func:`fused_linear_token_log_probs`: the same from hidden states and the output weight
* :func:`preference_loss`: loss over pairs of answers from their summed log-probability ratios
* :func:`policy_loss`: clipped policy-gradient loss with a KL term
* :func:`embedding_sorted`: embedding whose gradient is summed in sorted token order (``ops.embedding(sorted_gradient=True)``)

Each runs the sm_100a kernels of ``csrc/ops`` and ``csrc/gemm`` on CUDA tensors and a plain PyTorch restatement elsewhere.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import _flce_chunk_rows, native, note_fallback, status_word
from .timeline import site

_LOGIT_TYPES = (torch.bfloat16, torch.float16, torch.float32)


# CUDA tensors of the kernels' types go straight to the extension, which makes the same checks (as ValueErrors) as the Python
# code makes for the other path: one call of the smallest cases costs a few microseconds there, tens of them here. `native()`
# raises where the extension cannot be loaded.


def _check_labels(labels: torch.Tensor, rows: torch.Size, device: torch.device, name: str = "labels") -> None:
    if labels.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} must be int64 or int32, got {labels.dtype}")
    if labels.shape != rows:
        raise ValueError(f"{name} must have the shape {tuple(rows)}, got {tuple(labels.shape)}")
    if labels.device != device:
        raise ValueError(f"{name} must be on {device}, got {labels.device}")


def _check_logit_scale(logit_scale: float) -> float:
    logit_scale = float(logit_scale)
    if not (math.isfinite(logit_scale) and logit_scale > 0):
        raise ValueError(f"logit_scale must be positive and finite, got {logit_scale}")
    return logit_scale


# Fused linear form: fp32 logits up to this size are kept between the passes instead of being formed twice.
# 4096 x 4096 x 128256 (2.1 GB) both directions: 10.2 ms kept, 12.5 ms formed twice.
_KEEP_LOGITS_BYTES = 4 << 30


# ----------------------------------------------------------------------------- token log-probabilities
def _kept(labels: torch.Tensor, ignore_index: int, vocab: int) -> torch.Tensor:
    return (labels != ignore_index) & (labels >= 0) & (labels < vocab)


def _token_log_probs_torch(logits: torch.Tensor, labels: torch.Tensor, logit_scale: float, ignore_index: int, return_entropy: bool):
    vocab, labels = logits.shape[-1], labels.long()  # an ignore_index beyond 32 bits would wrap around next to int32 labels
    kept = _kept(labels, ignore_index, vocab)
    z = logits if logits.dtype == torch.float64 else logits.float()
    z = torch.where(kept[..., None], z, 0.0) * logit_scale  # whatever an ignored row holds, it has no part and no gradient
    logp = z.log_softmax(-1)
    picked = logp.gather(-1, torch.where(kept, labels, 0)[..., None]).squeeze(-1)
    picked = torch.where(kept, picked, 0.0)
    if not return_entropy:
        return picked
    # a token of probability 0 contributes 0, also where its log-probability is -inf
    entropy = -(logp.exp() * logp.clamp_min(torch.finfo(logp.dtype).min)).sum(-1)
    return picked, torch.where(kept, entropy, 0.0)


def token_log_probs(logits: torch.Tensor, labels: torch.Tensor, *, logit_scale: float = 1.0, ignore_index: int = -100,
                    return_entropy: bool = False):
    """Log-probability of ``labels[...]`` under ``softmax(logit_scale * logits[..., :])``, fp32, shaped like ``labels``; with
    ``return_entropy`` also the entropy of each row's distribution (nats).

    Rows whose label is ``ignore_index`` (or lies outside of the vocabulary) give 0 and no gradient, whatever they hold. Logits of
    ``-inf`` are tokens of probability 0; a row of nothing but ``-inf`` has no distribution and gives NaN. ``logit_scale`` (1 /
    temperature, 1 / ``m_width``) must be positive. bf16, fp16 and fp32 logits of any row stride run on the kernels."""
    if logits.is_cuda and logits.dtype in _LOGIT_TYPES:
        with site("token_log_probs"):
            out = native().token_log_probs(logits, labels, logit_scale, ignore_index, return_entropy)
        return tuple(out) if return_entropy else out[0]
    logit_scale = _check_logit_scale(logit_scale)
    if logits.dim() < 1 or logits.shape[-1] == 0 or not logits.is_floating_point():
        raise ValueError(f"logits must be floating point with a last dimension of at least 1, got {logits.dtype} {tuple(logits.shape)}")
    _check_labels(labels, logits.shape[:-1], logits.device)
    return _token_log_probs_torch(logits, labels, logit_scale, ignore_index, return_entropy)


# ----------------------------------------------------------------------------- from hidden states
def fused_linear_token_log_probs(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, logit_scale: float = 1.0,
                                 ignore_index: int = -100, return_entropy: bool = False, keep_logits: bool | None = None):
    """:func:`token_log_probs` of ``logits = x @ weight.T`` from the operands: ``x [..., H]``, ``weight [V, H]``, ``labels [...]``.

    The logits are formed in fp32 on the tensor cores and reduced where they are. Without gradients they never reach memory;
    with gradients they are kept in fp32 until the backward pass (``keep_logits``; by default where that takes at most 4 GiB) or
    formed a second time in it. The backward pass needs a transient buffer of at most about 2.2 GB, which holds the gradient of the logits
    in bf16, the operand type of the two products that follow: their results are off by one rounding more (relative error against 64 bits
    2.3e-3; rounding the result alone gives 1.7e-3). Rows whose label is
    ignored take no part in any product. bf16 operands with ``H`` a multiple of 8 run on the kernels, which add the gradient of
    ``weight`` into its ``main_grad`` when the engine provides one; other types and sizes run as PyTorch operations in fp32 (fp64 operands
    in fp64), with the logits kept."""
    if x.is_cuda and x.dtype == torch.bfloat16 and x.dim() > 0 and weight.dim() == 2 and x.shape[-1] % 8 == 0:
        with site("loss.lm_head.log_probs"):
            out = native().linear_token_log_probs(
                x, weight, labels, logit_scale, ignore_index, return_entropy, _flce_chunk_rows(labels.numel(), weight.shape[0]),
                _KEEP_LOGITS_BYTES if keep_logits is None else (1 << 62) * bool(keep_logits), status_word(x.device))
        return tuple(out) if return_entropy else out[0]
    logit_scale = _check_logit_scale(logit_scale)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"hidden states [..., H] and a weight [V, H] are needed, got {tuple(x.shape)} and {tuple(weight.shape)}")
    if x.device != weight.device or x.dtype != weight.dtype or not x.is_floating_point():
        raise ValueError(f"hidden states and weight must be floating point of one type on one device, got {x.dtype} on {x.device} "
                         f"and {weight.dtype} on {weight.device}")
    _check_labels(labels, x.shape[:-1], x.device)
    note_fallback("fused_linear_token_log_probs", "the hidden size is not a multiple of 8", x, weight)
    # logits of fp32 as on the kernels, and rows that do not count are left out of the products: their values would reach the
    # weight's gradient as 0 * NaN
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    x = torch.where(_kept(labels.long(), ignore_index, weight.shape[0])[..., None], x, 0.0)
    return _token_log_probs_torch(F.linear(x.to(wide), weight.to(wide)), labels, logit_scale, ignore_index, return_entropy)


# ----------------------------------------------------------------------------- losses over packed answers
class PreferenceLossOutput(NamedTuple):
    loss: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor


class PolicyLossOutput(NamedTuple):
    loss: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


_PREFERENCE_KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}
_PREFERENCE_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_POLICY_REDUCTIONS = {"sum": 0, "token_mean": 1, "sequence_mean": 2}


def _check_like(t: torch.Tensor, like: torch.Tensor, name: str) -> torch.Tensor:
    if t.shape != like.shape or t.device != like.device or not t.is_floating_point():
        raise ValueError(f"{name} must be floating point, shaped {tuple(like.shape)} on {like.device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    if t.requires_grad:
        raise ValueError(f"{name} must not require a gradient (detach it): the loss is differentiated with respect to log_probs alone")
    return t


def _check_sequences(log_probs: torch.Tensor, cu_seqlens: torch.Tensor | None, mask: torch.Tensor | None) -> tuple[int, int]:
    """``(number of sequences, their length when there is no cu_seqlens)``."""
    if not log_probs.is_floating_point():
        raise ValueError(f"log_probs must be floating point, got {log_probs.dtype}")
    if mask is not None and (mask.shape != log_probs.shape or mask.device != log_probs.device or mask.is_floating_point()):
        raise ValueError(f"mask must be boolean or integer, shaped {tuple(log_probs.shape)} on {log_probs.device}, got {mask.dtype} "
                         f"{tuple(mask.shape)} on {mask.device}")
    if cu_seqlens is None:
        if log_probs.dim() != 2:
            raise ValueError(f"log_probs must be [sequences, length], or [tokens] with cu_seqlens, got {tuple(log_probs.shape)}")
        return log_probs.shape[0], log_probs.shape[1]
    if log_probs.dim() != 1:
        raise ValueError(f"with cu_seqlens log_probs must be [tokens], got {tuple(log_probs.shape)}")
    integers = cu_seqlens.dtype in (torch.int32, torch.int64)
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or not integers or cu_seqlens.device != log_probs.device:
        raise ValueError(f"cu_seqlens must be int32 or int64 [sequences + 1] on {log_probs.device}, got {cu_seqlens.dtype} "
                         f"{tuple(cu_seqlens.shape)} on {cu_seqlens.device}")
    return cu_seqlens.numel() - 1, 0


def _sequence_ids(count: int, length: int, cu_seqlens: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    """Sequence of each (flattened) token, ``count`` for tokens outside of all sequences."""
    t = torch.arange(like.numel(), device=like.device)
    if cu_seqlens is None:
        return t // max(length, 1)
    ids = torch.searchsorted(cu_seqlens[1:].long().contiguous(), t, right=True)
    return torch.where(t < cu_seqlens[0], count, ids)


def _preference_loss_torch(log_probs, reference, cu_seqlens, length, sequences, mask, kind, beta, label_smoothing, average, reduction):
    lp = log_probs.reshape(-1)
    d = lp if reference is None else lp - reference.reshape(-1)
    ids = _sequence_ids(sequences, length, cu_seqlens, lp)
    kept = ids < sequences if mask is None else (ids < sequences) & (mask.reshape(-1) != 0)
    d = torch.where(kept, d, 0.0)
    sums = torch.zeros(sequences + 1, dtype=d.dtype, device=d.device).index_add(0, ids, d)[:sequences]
    if average:
        tokens = torch.zeros(sequences + 1, dtype=d.dtype, device=d.device).index_add(0, ids, kept.to(d.dtype))[:sequences]
        sums = sums / tokens.clamp_min(1)
    chosen, rejected = sums.chunk(2)
    margin = beta * (chosen - rejected)
    if kind == 0:
        loss = (1 - label_smoothing) * F.softplus(-margin) + (label_smoothing * F.softplus(margin) if label_smoothing else 0.0)
    elif kind == 1:
        loss = torch.relu(1 - margin)
    else:
        loss = (chosen - rejected - 0.5 / beta).square()
    loss = loss if reduction == 0 else loss.sum() if reduction == 1 else loss.mean()
    return loss, (beta * sums).detach()


def preference_loss(log_probs: torch.Tensor, reference_log_probs: torch.Tensor | None, cu_seqlens: torch.Tensor | None = None, *,
                    beta: float = 0.1, loss_type: str = "sigmoid", label_smoothing: float = 0.0, average_log_probs: bool = False,
                    mask: torch.Tensor | None = None, reduction: str = "mean") -> PreferenceLossOutput:
    """Loss over pairs of answers from per-token log-probabilities of the policy and of a frozen reference.

    ``log_probs`` is packed ``[tokens]`` with ``cu_seqlens [2 * pairs + 1]`` or padded ``[2 * pairs, length]``: the chosen answers first,
    then the rejected ones in the same order. With ``s`` an answer's sum (``average_log_probs``: mean) of ``log_probs - reference``
    over the tokens that ``mask`` keeps and ``D = s_chosen - s_rejected``: ``sigmoid`` is ``(1 - e) softplus(-beta D) + e softplus(beta D)``
    with ``e = label_smoothing``, ``hinge`` is ``max(0, 1 - beta D)``, ``ipo`` is ``(D - 1 / (2 beta))^2``.
    ``reference_log_probs=None`` leaves the reference out.

    Returns the loss (reduced over pairs, or one per pair with ``reduction="none"``) and ``beta * s`` of the chosen and the rejected answers
    (no gradient). An answer without tokens has ``s = 0``. Masked tokens, and tokens outside of all sequences, are not looked at and get a
    gradient of 0."""
    if loss_type not in _PREFERENCE_KINDS or reduction not in _PREFERENCE_REDUCTIONS:
        raise ValueError(f"unexpected loss_type ({loss_type}) or reduction ({reduction})")
    if log_probs.is_cuda and log_probs.dtype in _LOGIT_TYPES:
        with site("preference_loss"):
            return PreferenceLossOutput(*native().preference_loss(
                log_probs, reference_log_probs, cu_seqlens, mask, _PREFERENCE_KINDS[loss_type], beta, label_smoothing, average_log_probs,
                _PREFERENCE_REDUCTIONS[reduction]))
    sequences, length = _check_sequences(log_probs, cu_seqlens, mask)
    if sequences == 0 or sequences % 2:
        raise ValueError(f"an even number of answers is needed (chosen, then rejected), got {sequences}")
    beta, label_smoothing = float(beta), float(label_smoothing)
    if not (math.isfinite(beta) and beta > 0):
        raise ValueError(f"beta must be positive and finite, got {beta}")
    if not 0 <= label_smoothing < 0.5 or (label_smoothing and loss_type != "sigmoid"):
        raise ValueError(f"label_smoothing must be in [0, 0.5) and goes with loss_type='sigmoid', got {label_smoothing} for {loss_type}")
    if reference_log_probs is not None:
        _check_like(reference_log_probs, log_probs, "reference_log_probs")
    args = (_PREFERENCE_KINDS[loss_type], beta, label_smoothing, bool(average_log_probs), _PREFERENCE_REDUCTIONS[reduction])
    wide = log_probs if log_probs.dtype == torch.float64 else log_probs.float()
    reference = None if reference_log_probs is None else reference_log_probs.to(wide.dtype)
    loss, rewards = _preference_loss_torch(wide, reference, cu_seqlens, length, sequences, mask, *args)
    pairs = sequences // 2
    return PreferenceLossOutput(loss, rewards[:pairs], rewards[pairs:])


def _policy_loss_torch(log_probs, old, reference, advantages, per_token, cu_seqlens, length, sequences, mask, clip_low, clip_high,
                       dual_clip, kl_coef, reduction):
    lp = log_probs.reshape(-1)
    ids = _sequence_ids(sequences, length, cu_seqlens, lp)
    kept = ids < sequences if mask is None else (ids < sequences) & (mask.reshape(-1) != 0)
    # neither values nor gradients of tokens that take no part may reach a sum, also where they are not finite
    own, old = torch.where(kept, lp, 0.0), torch.where(kept, old.reshape(-1), 0.0)
    adv = advantages.reshape(-1) if per_token else torch.cat([advantages, advantages.new_zeros(1)])[ids]
    adv = torch.where(kept, adv, 0.0)
    delta = own.double() - old.double()
    log_low, log_high = math.log1p(-clip_low) if clip_low < 1 else -math.inf, math.log1p(clip_high)
    clipped = ((adv > 0) & (delta > log_high)) | ((adv < 0) & (delta < log_low))
    ratio = torch.where(clipped | (adv == 0), 0.0, delta).exp().to(own.dtype)
    value = torch.where(clipped, -adv * torch.where(adv > 0, torch.full_like(adv, 1 + clip_high), 1 - clip_low), -adv * ratio)
    if dual_clip:
        bound = (adv < 0) & (value > -dual_clip * adv)
        value, clipped = torch.where(bound, -dual_clip * adv, value), clipped | bound
    kl = torch.zeros_like(value)
    if reference is not None:
        d = torch.where(kept, reference.reshape(-1), 0.0) - own
        kl = torch.expm1(d) - d
        if kl_coef:
            value = value + kl_coef * kl
    n = kept.sum().clamp_min(1)
    if reduction == 2:
        zeros = torch.zeros(sequences + 1, dtype=value.dtype, device=value.device)
        tokens = zeros.index_add(0, ids, kept.to(value.dtype))[:sequences]
        means = zeros.index_add(0, ids, value)[:sequences] / tokens.clamp_min(1)
        loss = means.sum() / (tokens > 0).sum().clamp_min(1)
    else:
        loss = value.sum() if reduction == 0 else value.sum() / n
    return loss, (kl.sum() / n).detach(), clipped.sum().to(value.dtype) / n


def policy_loss(log_probs: torch.Tensor, old_log_probs: torch.Tensor, advantages: torch.Tensor, *,
                reference_log_probs: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                clip_low: float = 0.2, clip_high: float = 0.2, dual_clip: float | None = None, kl_coef: float = 0.0,
                reduction: str = "token_mean") -> PolicyLossOutput:
    """Clipped policy-gradient loss with a KL term, from per-token log-probabilities of sampled answers.

    ``log_probs`` is packed ``[tokens]`` with ``cu_seqlens [sequences + 1]`` or padded ``[sequences, length]``; ``advantages`` is
    ``[sequences]``, one value per answer, or else has the shape of ``log_probs``. A token's loss is
    ``max(-A r, -A clip(r, 1 - clip_low, 1 + clip_high))`` with ``r = exp(log_probs - old_log_probs)``, bounded by ``-dual_clip A``
    where ``A < 0``, plus ``kl_coef (exp(k) - 1 - k)`` with ``k = reference - log_probs``. ``token_mean`` divides the sum by the
    number of tokens that ``mask`` keeps, ``sequence_mean`` averages the answers' token means over the answers that keep a token,
    ``sum`` does neither.

    Returns the loss, and over the kept tokens the mean of ``exp(k) - 1 - k`` (0 without a reference) and the share whose gradient
    was clipped (neither has a gradient). Masked tokens, and tokens outside of all sequences, are not looked at and get a gradient
    of 0; nothing kept gives 0."""
    if reduction not in _POLICY_REDUCTIONS:
        raise ValueError(f"unexpected reduction ({reduction})")
    if dual_clip is not None and not (math.isfinite(dual_clip) and dual_clip > 1):
        raise ValueError(f"dual_clip must be finite and above 1, got {dual_clip}")
    if log_probs.is_cuda and log_probs.dtype in _LOGIT_TYPES:
        with site("policy_loss"):
            return PolicyLossOutput(*native().policy_loss(
                log_probs, old_log_probs, advantages, reference_log_probs, cu_seqlens, mask, clip_low, clip_high, dual_clip or 0.0, kl_coef,
                _POLICY_REDUCTIONS[reduction]))
    sequences, length = _check_sequences(log_probs, cu_seqlens, mask)
    _check_like(old_log_probs, log_probs, "old_log_probs")
    if reference_log_probs is not None:
        _check_like(reference_log_probs, log_probs, "reference_log_probs")
    per_token = advantages.shape != (sequences,) and advantages.shape == log_probs.shape
    _check_like(advantages, log_probs if per_token else log_probs.new_empty(()).expand(sequences), "advantages")
    clip_low, clip_high, kl_coef = float(clip_low), float(clip_high), float(kl_coef)
    if not (0 <= clip_low <= 1 and clip_high >= 0):
        raise ValueError(f"clip_low must be in [0, 1] and clip_high at least 0, got {clip_low} and {clip_high}")
    if not (math.isfinite(kl_coef) and kl_coef >= 0):
        raise ValueError(f"kl_coef must be finite and at least 0, got {kl_coef}")
    if kl_coef and reference_log_probs is None:
        raise ValueError("kl_coef needs reference_log_probs")
    args = (clip_low, clip_high, float(dual_clip or 0.0), kl_coef, _POLICY_REDUCTIONS[reduction])
    wide = log_probs if log_probs.dtype == torch.float64 else log_probs.float()
    others = [None if t is None else t.to(wide.dtype) for t in (old_log_probs, reference_log_probs, advantages)]
    return PolicyLossOutput(*_policy_loss_torch(wide, *others, per_token, cu_seqlens, length, sequences, mask, *args))


# ----------------------------------------------------------------------------- embedding
def embedding_sorted(weight: torch.Tensor, ids: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[ids]`` whose weight gradient adds the rows of a token in an order fixed by the ids and the sizes: the same bits on
    every run, no fp32 copy of the whole table (``ops.embedding(sorted_gradient=True)``). Sums are fp32 for up to 128 rows of a 16-bit
    token and 64-bit otherwise. bf16, fp16 and fp32 tables of any width run on the kernels. The gradient has no derivative, and forward-mode
    differentiation is not available there.

    On the GPU an id outside of the table gives a row of zeros, takes no part in the gradient and raises the status word
    (``ops.check_status()``)."""
    if weight.is_cuda and weight.dtype in _LOGIT_TYPES:
        with site("embedding"):
            return native().embedding_sorted(weight, ids, scale, status_word(weight.device))
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"the embedding table must be floating point [V, H], got {weight.dtype} {tuple(weight.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be int64 or int32, got {ids.dtype}")
    if ids.device != weight.device:
        raise ValueError(f"ids must be on {weight.device}, got {ids.device}")
    out = F.embedding(ids, weight)
    return out if scale == 1.0 else out * scale
