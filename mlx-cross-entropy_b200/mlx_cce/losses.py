"""Losses on a head's per-token log-probabilities: policy and preference losses.

    logp = -linear_cross_entropy(hidden, weight, tokens, reduction="none")
    loss = policy_loss(logp, old_logp, advantages, ref_logp=ref_logp, kl_coef=0.04)

The reference ends at the cross-entropy; these are what its log-probabilities
are trained with after pre-training.  Both run on the CUDA kernels of
``csrc/token_loss.cu`` and are differentiable with respect to ``logp``; the
other tensors are constants.

Tokens come as padded rows ``[S, T]`` (a row is a sequence) or packed in one
dimension with ``cu_seqlens`` (int32 offsets ``[S + 1]``).  Tokens that
``mask`` leaves out, and packed tokens of no sequence, add nothing and get a
zero gradient, whatever they hold.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _ext

POLICY_REDUCTIONS = {"mean": _ext.CCE_REDUCE_MEAN, "sum": _ext.CCE_REDUCE_SUM,
                     "sequence": _ext.CCE_REDUCE_SEQUENCE, "none": _ext.CCE_REDUCE_NONE}
PREFERENCE_REDUCTIONS = {"mean": _ext.CCE_REDUCE_MEAN, "sum": _ext.CCE_REDUCE_SUM, "none": _ext.CCE_REDUCE_NONE}
PREFERENCE_LOSSES = {"sigmoid": _ext.CCE_PREF_SIGMOID, "hinge": _ext.CCE_PREF_HINGE, "ipo": _ext.CCE_PREF_IPO}


class PolicyStats(NamedTuple):
    """Over the tokens that count: mean KL term and share of clipped tokens (float32 scalars)."""
    kl: torch.Tensor
    clip_fraction: torch.Tensor


class PreferenceRewards(NamedTuple):
    """beta times the summed log-ratio of each pair's sequences (float32 [pairs])."""
    chosen: torch.Tensor
    rejected: torch.Tensor


# ---------------------------------------------------------------------------
# argument checks
# ---------------------------------------------------------------------------

def _offsets(what, cu_seqlens, dev):
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError(f"[{what}] cu_seqlens must be 1D with S + 1 offsets, got {tuple(cu_seqlens.shape)}")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"[{what}] cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
    if cu_seqlens.device != dev:
        raise ValueError(f"[{what}] cu_seqlens is on {cu_seqlens.device}, expected {dev}")
    return cu_seqlens.to(torch.int32).contiguous()


def _sequences(what, shape, cu_seqlens, dev):
    """(number of sequences, int32 offsets or None) of tokens of this shape."""
    if cu_seqlens is not None:
        if len(shape) != 1:
            raise ValueError(f"[{what}] packed tokens (cu_seqlens) must be 1D, got {tuple(shape)}")
        cu = _offsets(what, cu_seqlens, dev)
        return cu.numel() - 1, cu
    if len(shape) == 2:
        return shape[0], None
    if len(shape) == 1:
        return 1, None
    raise ValueError(f"[{what}] tokens must be [S, T], or 1D (with cu_seqlens for several sequences), "
                     f"got {tuple(shape)}")


def _like(what, name, t, logp):
    if t is None:
        return None
    if t.shape != logp.shape:
        raise ValueError(f"[{what}] {name} must have logp's shape {tuple(logp.shape)}, got {tuple(t.shape)}")
    if t.dtype != logp.dtype:
        raise ValueError(f"[{what}] {name} must have logp's dtype {logp.dtype}, got {t.dtype}")
    if t.device != logp.device:
        raise ValueError(f"[{what}] {name} is on {t.device}, expected {logp.device}")
    return t.detach().contiguous()


def _mask(what, mask, shape, dev):
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"[{what}] mask must be bool (or uint8), got {mask.dtype}")
    if mask.shape != shape:
        raise ValueError(f"[{what}] mask must have the tokens' shape {tuple(shape)}, got {tuple(mask.shape)}")
    if mask.device != dev:
        raise ValueError(f"[{what}] mask is on {mask.device}, expected {dev}")
    return mask.contiguous()


def _logp(what, logp):
    _ext.dtype_code(logp.dtype, what)
    if not logp.is_cuda:
        raise ValueError(f"[{what}] logp must be a CUDA tensor (no CPU implementation exists)")
    return logp.contiguous()


def _policy_params(what, clip, clip_high, dual_clip, kl_coef, reduction, per_token):
    if reduction not in POLICY_REDUCTIONS:
        raise ValueError(f"[{what}] Unknown reduction: {reduction}")
    high = clip if clip_high is None else clip_high
    if not (0 <= clip <= 1) or not high >= 0:
        raise ValueError(f"[{what}] clip must be in [0, 1] and clip_high >= 0, got {clip} and {clip_high}")
    if dual_clip is not None and not dual_clip > 1:
        raise ValueError(f"[{what}] dual_clip must be above 1, got {dual_clip}")
    if not math.isfinite(kl_coef):
        raise ValueError(f"[{what}] kl_coef must be finite, got {kl_coef}")
    return _ext.CcePolicyParams(clip, high, dual_clip or 0.0, kl_coef, POLICY_REDUCTIONS[reduction], int(per_token))


def _advantages(what, advantages, shape, S, dev):
    """(float32 advantages, one per token?)"""
    if advantages.shape == shape:
        per_token = True
    elif advantages.shape == (S,):
        per_token = False
    else:
        raise ValueError(f"[{what}] advantages must be per token {tuple(shape)} or per sequence ({S},), "
                         f"got {tuple(advantages.shape)}")
    if not advantages.is_floating_point():
        raise ValueError(f"[{what}] advantages must be floating point, got {advantages.dtype}")
    if advantages.device != dev:
        raise ValueError(f"[{what}] advantages are on {advantages.device}, expected {dev}")
    return advantages.detach().to(torch.float32).contiguous(), per_token


def _preference_params(what, beta, margin, loss_type, label_smoothing, length_normalize, reduction):
    if reduction not in PREFERENCE_REDUCTIONS:
        raise ValueError(f"[{what}] Unknown reduction: {reduction}")
    if loss_type not in PREFERENCE_LOSSES:
        raise ValueError(f"[{what}] Unknown loss_type: {loss_type!r}; expected one of {tuple(PREFERENCE_LOSSES)}")
    if not (beta > 0 and math.isfinite(beta)) or not math.isfinite(margin):
        raise ValueError(f"[{what}] beta must be positive and margin finite, got {beta} and {margin}")
    if not 0 <= label_smoothing <= 0.5:
        raise ValueError(f"[{what}] label_smoothing must be in [0, 0.5], got {label_smoothing}")
    if loss_type != "sigmoid" and label_smoothing:
        raise ValueError(f"[{what}] label_smoothing belongs to the sigmoid loss")
    if loss_type == "ipo" and margin:
        raise ValueError(f"[{what}] margin does not apply to the ipo loss")
    return _ext.CcePreferenceParams(beta, margin, label_smoothing, PREFERENCE_LOSSES[loss_type],
                                    PREFERENCE_REDUCTIONS[reduction], int(bool(length_normalize)))


def _pairs(what, shape, cu_seqlens, dev):
    """(pairs, offsets): sequence p is chosen over sequence pairs + p."""
    if cu_seqlens is None and len(shape) != 2:
        raise ValueError(f"[{what}] tokens must be [2 pairs, T], or 1D with cu_seqlens, got {tuple(shape)}")
    S, cu = _sequences(what, shape, cu_seqlens, dev)
    if S % 2:
        raise ValueError(f"[{what}] pairs need an even number of sequences (chosen, then rejected), got {S}")
    return S // 2, cu


def _reference(what, ref_logp, logp, S):
    """(per-token reference or None, per-sequence sums or None)"""
    if ref_logp is None:
        return None, None
    if ref_logp.shape == logp.shape:
        return _like(what, "ref_logp", ref_logp, logp), None
    if ref_logp.shape != (S,):
        raise ValueError(f"[{what}] ref_logp must be per token {tuple(logp.shape)} or per sequence ({S},), "
                         f"got {tuple(ref_logp.shape)}")
    if not ref_logp.is_floating_point() or ref_logp.device != logp.device:
        raise ValueError(f"[{what}] ref_logp must be floating point on {logp.device}")
    return None, ref_logp.detach().to(torch.float32).contiguous()


# ---------------------------------------------------------------------------
# autograd
# ---------------------------------------------------------------------------

class PolicyLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, old, ref, adv, mask, cu, S, params):
        loss, stats, coef = _ext.policy_forward(logp, old, ref, adv, mask, cu, S, params)
        ctx.save_for_backward(coef, cu)
        ctx.meta = (params.reduction, logp.numel(), S, logp.shape, logp.dtype)
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _grad_stats):
        if grad_loss is None:
            return (None,) * 8
        coef, cu = ctx.saved_tensors
        reduction, N, S, shape, dtype = ctx.meta
        g = grad_loss.to(torch.float32).contiguous()
        return (_ext.policy_backward(coef, g, reduction, cu, N, S, shape, dtype),) + (None,) * 7


class PreferenceLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, ref, ref_sums, mask, cu, pairs, params):
        loss, rewards, coef = _ext.preference_forward(logp, ref, ref_sums, mask, cu, pairs, params)
        ctx.save_for_backward(coef, mask, cu)
        ctx.meta = (params.reduction, logp.numel(), pairs, logp.shape, logp.dtype)
        ctx.mark_non_differentiable(rewards)
        ctx.set_materialize_grads(False)
        return loss, rewards

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _grad_rewards):
        if grad_loss is None:
            return (None,) * 7
        coef, mask, cu = ctx.saved_tensors
        reduction, N, pairs, shape, dtype = ctx.meta
        g = grad_loss.to(torch.float32).contiguous()
        return (_ext.preference_backward(coef, g, reduction, mask, cu, N, pairs, shape, dtype),) + (None,) * 6


# ---------------------------------------------------------------------------
# public entry points
# ---------------------------------------------------------------------------

def policy_loss(logp, old_logp, advantages, *, ref_logp=None, mask=None, cu_seqlens=None, clip=0.2, clip_high=None,
                dual_clip=None, kl_coef=0.0, reduction="mean", return_stats=False):
    """Clipped policy loss with a KL term, on per-token log-probabilities.

    With ratio ``r = exp(logp - old_logp)`` and advantage ``A`` a token's loss is
    ``-min(r A, clip(r, 1 - clip, 1 + clip_high) A) + kl_coef (exp(q) - 1 - q)``,
    ``q = ref_logp - logp``.

    Args:
        logp: log-probabilities of the sampled tokens, ``[S, T]`` or packed ``[N]``
            (float32, float16 or bfloat16; differentiable)
        old_logp: those of the policy that sampled them; None: the policy itself (r = 1)
        advantages: per token (logp's shape) or per sequence ``[S]``
        ref_logp: those of the reference policy, for the KL term; None: no such term
        mask: bool, logp's shape; False leaves a token out
        cu_seqlens: offsets ``[S + 1]`` of packed sequences
        clip, clip_high: the ratio is clipped to ``[1 - clip, 1 + clip_high]``
            (clip_high defaults to clip; ``inf`` leaves that side open)
        dual_clip: bounds a negative advantage's loss by ``-dual_clip * A``
        kl_coef: weight of the KL term
        reduction: "mean" over tokens, "sequence" (mean over the sequences that
            have a token of their tokens' means), "sum" or "none" (per token)
        return_stats: also return ``PolicyStats(kl, clip_fraction)``
    Returns:
        float32 loss (scalar, or logp's shape for reduction="none"); with
        ``return_stats`` a tuple ``(loss, stats)``.
    """
    what = "policy_loss"
    logp = _logp(what, logp)
    S, cu = _sequences(what, logp.shape, cu_seqlens, logp.device)
    adv, per_token = _advantages(what, advantages, logp.shape, S, logp.device)
    params = _policy_params(what, clip, clip_high, dual_clip, kl_coef, reduction, per_token)
    loss, stats = PolicyLossFunction.apply(logp, _like(what, "old_logp", old_logp, logp),
                                           _like(what, "ref_logp", ref_logp, logp), adv,
                                           _mask(what, mask, logp.shape, logp.device), cu, S, params)
    return (loss, PolicyStats(*stats.unbind())) if return_stats else loss


def preference_loss(logp, ref_logp=None, *, mask=None, cu_seqlens=None, beta=0.1, margin=0.0, loss_type="sigmoid",
                    label_smoothing=0.0, length_normalize=False, reduction="mean", return_rewards=False):
    """Preference loss of pairs of sequences from the log-ratios of their tokens.

    The first half of the sequences is chosen over the second half, in the same
    order.  With ``D`` the sum over a sequence's tokens of ``logp - ref_logp``,
    ``gap = D_chosen - D_rejected`` and ``h = beta * gap - margin`` a pair's loss is
    ``-log sigmoid(h)`` ("sigmoid"), ``max(0, 1 - h)`` ("hinge") or
    ``(gap - 1 / (2 beta))^2`` ("ipo").

    Args:
        logp: log-probabilities, ``[2 pairs, T]`` or packed ``[N]`` (float32,
            float16 or bfloat16; differentiable)
        ref_logp: the reference policy's, per token (logp's shape) or summed per
            sequence ``[2 pairs]``; None: none (reference-free losses)
        mask: bool, logp's shape; False leaves a token out (prompts, padding)
        cu_seqlens: offsets ``[2 pairs + 1]`` of packed sequences
        beta, margin: see above
        label_smoothing: probability that a pair's order is wrong ("sigmoid")
        length_normalize: divide ``D`` by the sequence's number of tokens
        reduction: "mean", "sum" or "none" over the pairs
        return_rewards: also return ``PreferenceRewards(chosen, rejected)``
    Returns:
        float32 loss (scalar, or ``[pairs]`` for reduction="none"); with
        ``return_rewards`` a tuple ``(loss, rewards)``.
    """
    what = "preference_loss"
    logp = _logp(what, logp)
    pairs, cu = _pairs(what, logp.shape, cu_seqlens, logp.device)
    params = _preference_params(what, beta, margin, loss_type, label_smoothing, length_normalize, reduction)
    ref, sums = _reference(what, ref_logp, logp, 2 * pairs)
    loss, rewards = PreferenceLossFunction.apply(logp, ref, sums, _mask(what, mask, logp.shape, logp.device), cu,
                                                 pairs, params)
    return (loss, PreferenceRewards(rewards[:pairs], rewards[pairs:])) if return_rewards else loss
