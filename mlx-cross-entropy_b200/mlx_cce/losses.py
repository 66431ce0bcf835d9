"""Losses on a head's log-probabilities: policy, preference and distillation losses.

    loss = linear_policy_loss(hidden, weight, tokens, old_logp, advantages, ref_logp=ref_logp, kl_coef=0.04)
    loss = linear_preference_loss(hidden, weight, tokens, ref_logp, cu_seqlens=offsets)
    loss = linear_distillation_loss(hidden, weight, teacher_ids, teacher_logprobs, temperature=2.0)

The reference ends at the cross-entropy; these are what a head is trained with
after pre-training.  ``linear_log_probs`` is the head's part of the first two
(log-probabilities of given tokens, the [N, V] logits never materialised);
``policy_loss`` and ``preference_loss`` take log-probabilities.  Hidden states,
classifier, bias and log-probabilities are differentiable, the other tensors
are constants.  Kernels: ``csrc/token_loss.cu``, ``csrc/rows_kernels.cu`` and
the GEMMs of ``csrc/tc_rows.cuh``.

The linear forms differ from ``linear_cross_entropy`` in two ways: the filter of
small softmax values is not applied (a policy gradient pushes the unlikely
tokens too: float16 heads lose what is below 2^-38 of a row's largest dlogit,
float32 heads below 2^-48), and rows that do not count are taken out before the
GEMMs.

Tokens come as padded rows ``[S, T]`` (a row is a sequence) or packed in one
dimension with ``cu_seqlens`` (int32 offsets ``[S + 1]``).  Advantages and
reference log-probabilities come per token or per sequence, told apart by their
shape; a packed batch of as many tokens as sequences fits both and is read per
token, with a warning, unless ``advantages_per_token`` or ``ref_per_token`` says
which it is.  Tokens that
``mask`` leaves out, and packed tokens of no sequence, add nothing and get a
zero gradient, whatever they hold.
"""

from __future__ import annotations

import math
import warnings
from typing import NamedTuple

import torch

from . import _ext

# The operators (csrc/torch_ops.cpp), called without the overload lookup.
_OPS = _ext.torch_ops()
_POLICY = _OPS.policy_loss.default
_PREFERENCE = _OPS.preference_loss.default
_LOG_PROBS = _OPS.log_probs.default
_LINEAR_POLICY = _OPS.linear_policy_loss.default
_LINEAR_PREFERENCE = _OPS.linear_preference_loss.default
_DISTILLATION = _OPS.distillation.default

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

def _untraced(what):
    """torch.compile breaks its graph here: the call runs as it is, between two graphs."""
    if torch.compiler.is_dynamo_compiling():
        raise RuntimeError(f"[{what}] cannot be part of a traced graph")


def _constant(t):
    """t as a kernel input: contiguous, cut from the graph."""
    if t.requires_grad:
        t = t.detach()
    return t.contiguous()


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


def _per_token(what, name, t, tokens, dtype=torch.float32):
    """t as a constant of the tokens' shape and the given dtype."""
    if t is None:
        return None
    if t.shape != tokens.shape:
        raise ValueError(f"[{what}] {name} must have the tokens' shape {tuple(tokens.shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"[{what}] {name} must be {dtype} (the log-probabilities' dtype), got {t.dtype}")
    if t.device != tokens.device:
        raise ValueError(f"[{what}] {name} is on {t.device}, expected {tokens.device}")
    return _constant(t)


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
    if not abs(kl_coef) <= torch.finfo(torch.float32).max:
        raise ValueError(f"[{what}] kl_coef must be finite in float32, got {kl_coef}")
    return [float(clip), float(high), float(dual_clip or 0.0), float(kl_coef)], POLICY_REDUCTIONS[reduction], per_token


def _is_per_token(what, name, got, shape, S, per_token, argument):
    """Whether values of shape ``got`` are one per token, not one per sequence."""
    tokens, seqs = got == shape, got == (S,)
    if per_token is not None:
        if not (tokens if per_token else seqs):
            raise ValueError(f"[{what}] {name} must be {tuple(shape) if per_token else (S,)} with {argument}="
                             f"{bool(per_token)}, got {tuple(got)}")
        return bool(per_token)
    if not (tokens or seqs):
        raise ValueError(f"[{what}] {name} must be per token {tuple(shape)} or per sequence ({S},), got {tuple(got)}")
    if tokens and seqs and S > 1:
        warnings.warn(f"[{what}] {name} of shape {tuple(got)} could be one per token or one per sequence and are read "
                      f"per token: say {argument}=True or False", stacklevel=4)
    return tokens


def _advantages(what, advantages, shape, S, dev, per_token=None):
    """(float32 advantages, one per token?)"""
    per_token = _is_per_token(what, "advantages", advantages.shape, shape, S, per_token, "advantages_per_token")
    if not advantages.is_floating_point():
        raise ValueError(f"[{what}] advantages must be floating point, got {advantages.dtype}")
    if advantages.device != dev:
        raise ValueError(f"[{what}] advantages are on {advantages.device}, expected {dev}")
    return _constant(advantages.to(torch.float32)), per_token


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
    return ([float(beta), float(margin), float(label_smoothing)], PREFERENCE_LOSSES[loss_type],
            PREFERENCE_REDUCTIONS[reduction], bool(length_normalize))


def _pairs(what, shape, cu_seqlens, dev):
    """(pairs, offsets): sequence p is chosen over sequence pairs + p."""
    if cu_seqlens is None and len(shape) != 2:
        raise ValueError(f"[{what}] tokens must be [2 pairs, T], or 1D with cu_seqlens, got {tuple(shape)}")
    S, cu = _sequences(what, shape, cu_seqlens, dev)
    if S % 2:
        raise ValueError(f"[{what}] pairs need an even number of sequences (chosen, then rejected), got {S}")
    return S // 2, cu


def _head(what, e, c, bias, rows_shape):
    """Checked (e [N, D], c, bias), contiguous."""
    if e.dim() < 2 or c.dim() != 2:
        raise ValueError(f"[{what}] e must be [..., D] and c [V, D], got {tuple(e.shape)} and {tuple(c.shape)}")
    if e.shape[:-1] != rows_shape:
        raise ValueError(f"[{what}] e holds rows {tuple(e.shape[:-1])}, expected {tuple(rows_shape)}")
    if e.shape[-1] != c.shape[1]:
        raise ValueError(f"[{what}] c.shape[1] ({c.shape[1]}) must equal e.shape[-1] ({e.shape[-1]})")
    if e.dtype != c.dtype:
        raise ValueError(f"[{what}] e and c must share a dtype, got {e.dtype} and {c.dtype}")
    _ext.dtype_code(e.dtype, what)
    if bias is not None:
        if bias.shape != (c.shape[0],):
            raise ValueError(f"[{what}] bias must be [V={c.shape[0]}], got {tuple(bias.shape)}")
        _ext.dtype_code(bias.dtype, what)
    if c.shape[0] == 0 or c.shape[1] == 0:
        raise ValueError(f"[{what}] c must not be empty, got {tuple(c.shape)}")
    for name, t in (("e", e), ("c", c), ("bias", bias)):
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"[{what}] {name} must be a CUDA tensor (no CPU implementation exists)")
        if t.device != e.device:
            raise ValueError(f"[{what}] {name} is on {t.device}, expected {e.device}")
    c = c.contiguous()
    if c.data_ptr() % 16:  # (a view at an odd element: the kernels' copies start on 16-byte boundaries)
        c = c.clone()
    return e.reshape(-1, e.shape[-1]).contiguous(), c, None if bias is None else bias.contiguous()


def _ids(what, name, t, dev):
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"[{what}] {name} must be int32 or int64, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"[{what}] {name} is on {t.device}, expected {dev}")
    return t.contiguous()


def _distill_params(what, temperature, tail, reduction):
    if reduction not in PREFERENCE_REDUCTIONS:
        raise ValueError(f"[{what}] Unknown reduction: {reduction}")
    if not 1e-30 <= temperature <= 1e30:  # (held in float32, and its reciprocal)
        raise ValueError(f"[{what}] temperature must be in [1e-30, 1e30], got {temperature}")
    return float(temperature), bool(tail), PREFERENCE_REDUCTIONS[reduction]


def _reference(what, ref_logp, tokens, dtype, S, per_token=None):
    """(per-token reference or None, per-sequence sums or None)"""
    if ref_logp is None:
        return None, None
    if _is_per_token(what, "ref_logp", ref_logp.shape, tokens.shape, S, per_token, "ref_per_token"):
        return _per_token(what, "ref_logp", ref_logp, tokens, dtype), None
    if not ref_logp.is_floating_point() or ref_logp.device != tokens.device:
        raise ValueError(f"[{what}] ref_logp must be floating point on {tokens.device}")
    return None, _constant(ref_logp.to(torch.float32))


# ---------------------------------------------------------------------------
# public entry points
# ---------------------------------------------------------------------------

def policy_loss(logp, old_logp, advantages, *, ref_logp=None, mask=None, cu_seqlens=None, clip=0.2, clip_high=None,
                dual_clip=None, kl_coef=0.0, reduction="mean", return_stats=False, advantages_per_token=None):
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
        kl_coef: weight of the KL term (0: it is measured for the statistics alone)
        reduction: "mean" over tokens, "sequence" (mean over the sequences that
            have a token of their tokens' means), "sum" or "none" (per token)
        return_stats: also return ``PolicyStats(kl, clip_fraction)``
        advantages_per_token: what advantages of a shape that fits both are (True,
            False; None: per token, with a warning)
    Returns:
        float32 loss (scalar, or logp's shape for reduction="none"); with
        ``return_stats`` a tuple ``(loss, stats)``.
    """
    what = "policy_loss"
    _untraced(what)
    logp = _logp(what, logp)
    S, cu = _sequences(what, logp.shape, cu_seqlens, logp.device)
    adv, per_token = _advantages(what, advantages, logp.shape, S, logp.device, advantages_per_token)
    params = _policy_params(what, clip, clip_high, dual_clip, kl_coef, reduction, per_token)
    loss, stats = _POLICY(logp, _per_token(what, "old_logp", old_logp, logp, logp.dtype),
                          _per_token(what, "ref_logp", ref_logp, logp, logp.dtype), adv,
                          _mask(what, mask, logp.shape, logp.device), cu, S, *params)
    return (loss, PolicyStats(*stats.unbind())) if return_stats else loss


def preference_loss(logp, ref_logp=None, *, mask=None, cu_seqlens=None, beta=0.1, margin=0.0, loss_type="sigmoid",
                    label_smoothing=0.0, length_normalize=False, reduction="mean", return_rewards=False,
                    ref_per_token=None):
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
        ref_per_token: what a ref_logp of a shape that fits both is (True, False; None:
            per token, with a warning)
    Returns:
        float32 loss (scalar, or ``[pairs]`` for reduction="none"); with
        ``return_rewards`` a tuple ``(loss, rewards)``.
    """
    what = "preference_loss"
    _untraced(what)
    logp = _logp(what, logp)
    pairs, cu = _pairs(what, logp.shape, cu_seqlens, logp.device)
    params = _preference_params(what, beta, margin, loss_type, label_smoothing, length_normalize, reduction)
    ref, sums = _reference(what, ref_logp, logp, logp.dtype, 2 * pairs, ref_per_token)
    loss, rewards = _PREFERENCE(logp, ref, sums, _mask(what, mask, logp.shape, logp.device), cu, pairs, *params)
    return (loss, PreferenceRewards(rewards[:pairs], rewards[pairs:])) if return_rewards else loss


def linear_log_probs(e, c, targets, bias=None, *, ignore_index=-100):
    """Log-probabilities ``log softmax(e c^T + bias)`` of the target tokens.

    Args:
        e: hidden states ``[..., D]`` (float32, float16 or bfloat16)
        c: classifier weights ``[V, D]`` in e's dtype
        targets: token ids ``[...]`` in ``[0, V)`` (int32 or int64)
        bias: optional classifier bias ``[V]``
        ignore_index: rows with this target are left out (None: none)
    Returns:
        float32, shaped like ``targets``; 0 for rows left out.  Accurate to
        float32 also for 16-bit inputs (``linear_cross_entropy`` is to 1e-3),
        differentiable with respect to e, c and bias.
    """
    what = "linear_log_probs"
    _untraced(what)
    e, c, bias = _head(what, e, c, bias, targets.shape)
    logp = _LOG_PROBS(e, c, bias, _ids(what, "targets", targets, e.device), ignore_index)
    return logp.view(targets.shape)


def linear_policy_loss(e, c, targets, old_logp, advantages, bias=None, *, ref_logp=None, cu_seqlens=None, clip=0.2,
                       clip_high=None, dual_clip=None, kl_coef=0.0, reduction="mean", ignore_index=-100,
                       return_stats=False, advantages_per_token=None):
    """``policy_loss`` of the head's log-probabilities of ``targets``.

    e ``[..., D]``, c ``[V, D]`` and bias as in ``linear_log_probs``; targets are the
    sampled tokens, ``[S, T]`` or packed ``[N]`` with ``cu_seqlens``; those equal to
    ignore_index do not count.  old_logp and ref_logp are float32, shaped like
    targets.  The other arguments and the result are those of ``policy_loss``.
    """
    what = "linear_policy_loss"
    _untraced(what)
    S, cu = _sequences(what, targets.shape, cu_seqlens, targets.device)
    adv, per_token = _advantages(what, advantages, targets.shape, S, targets.device, advantages_per_token)
    params = _policy_params(what, clip, clip_high, dual_clip, kl_coef, reduction, per_token)
    e, c, bias = _head(what, e, c, bias, targets.shape)
    targets = _ids(what, "targets", targets, e.device)
    loss, stats = _LINEAR_POLICY(e, c, bias, targets, ignore_index, _per_token(what, "old_logp", old_logp, targets),
                                 _per_token(what, "ref_logp", ref_logp, targets), adv, cu, S, *params)
    if reduction == "none":
        loss = loss.view(targets.shape)
    return (loss, PolicyStats(*stats.unbind())) if return_stats else loss


def linear_preference_loss(e, c, targets, ref_logp=None, bias=None, *, cu_seqlens=None, beta=0.1, margin=0.0,
                           loss_type="sigmoid", label_smoothing=0.0, length_normalize=False, reduction="mean",
                           ignore_index=-100, return_rewards=False, ref_per_token=None):
    """``preference_loss`` of the head's log-probabilities of ``targets``.

    e ``[..., D]``, c ``[V, D]`` and bias as in ``linear_log_probs``; targets are the
    tokens of the sequences, ``[2 pairs, T]`` or packed ``[N]`` with ``cu_seqlens``,
    chosen before rejected; those equal to ignore_index do not count.  ref_logp is
    float32 per token, or per sequence ``[2 pairs]``.  The other arguments and the
    result are those of ``preference_loss``.
    """
    what = "linear_preference_loss"
    _untraced(what)
    pairs, cu = _pairs(what, targets.shape, cu_seqlens, targets.device)
    params = _preference_params(what, beta, margin, loss_type, label_smoothing, length_normalize, reduction)
    e, c, bias = _head(what, e, c, bias, targets.shape)
    targets = _ids(what, "targets", targets, e.device)
    ref, sums = _reference(what, ref_logp, targets, torch.float32, 2 * pairs, ref_per_token)
    loss, rewards = _LINEAR_PREFERENCE(e, c, bias, targets, ignore_index, ref, sums, cu, pairs, *params)
    return (loss, PreferenceRewards(rewards[:pairs], rewards[pairs:])) if return_rewards else loss


def linear_distillation_loss(e, c, teacher_ids, teacher_logprobs, bias=None, *, temperature=1.0, tail=False, mask=None,
                             reduction="mean"):
    """KL divergence from a teacher known by its top K tokens to the head's softmax.

    With ``q = softmax((e c^T + bias) / temperature)`` over the whole vocabulary and
    the teacher's probabilities ``p`` of its K entries a row's loss is
    ``sum p (log p - log q)``; with ``tail`` also ``r (log r - log q_r)`` of the mass
    ``r = 1 - sum p`` that the entries leave over and the student's mass ``q_r``
    outside of them.  (No factor ``temperature**2``.)

    Args:
        e: hidden states ``[..., D]`` (float32, float16 or bfloat16)
        c: classifier weights ``[V, D]`` in e's dtype
        teacher_ids: token ids ``[..., K]`` (int32 or int64, K <= 1024), in any order;
            ids outside of ``[0, V)`` are absent entries (padding), entries of the
            same id add their probabilities
        teacher_logprobs: ``[..., K]`` log-probabilities or logits; p is their softmax
            over the K entries at the temperature.  With ``tail``: log-probabilities
            over the whole vocabulary at the temperature, used as they are
        bias: optional classifier bias ``[V]``
        temperature: in [1e-30, 1e30]
        mask: bool ``[...]``; False leaves a row out
        reduction: "mean" over the rows that have an entry, "sum" or "none"
    Returns:
        float32 loss (scalar, or the rows' shape for reduction="none"), differentiable
        with respect to e, c and bias.
    """
    what = "linear_distillation_loss"
    _untraced(what)
    params = _distill_params(what, temperature, tail, reduction)
    if teacher_ids.dim() < 1 or teacher_ids.shape != teacher_logprobs.shape:
        raise ValueError(f"[{what}] teacher_ids and teacher_logprobs must be [..., K] of one shape, got "
                         f"{tuple(teacher_ids.shape)} and {tuple(teacher_logprobs.shape)}")
    rows, K = teacher_ids.shape[:-1], teacher_ids.shape[-1]
    if not 1 <= K <= _ext.CCE_DISTILL_MAX_K:
        raise ValueError(f"[{what}] K must be in [1, {_ext.CCE_DISTILL_MAX_K}], got {K}")
    e2, c, bias = _head(what, e, c, bias, rows)
    ids = _ids(what, "teacher_ids", teacher_ids, e.device).view(-1, K)
    if not teacher_logprobs.is_floating_point() or teacher_logprobs.device != e.device:
        raise ValueError(f"[{what}] teacher_logprobs must be floating point on {e.device}")
    teacher = _constant(teacher_logprobs.to(torch.float32))
    loss = _DISTILLATION(e2, c, bias, ids, teacher, _mask(what, mask, rows, e.device), *params)
    return loss.view(rows) if reduction == "none" else loss
