"""The clipped policy loss of a batch of played actions, with a KL term
towards a reference policy and the gradient in the logits.

It takes the frames where ``loss_input`` leaves them: ``Sample.policy_mask``
is ``legal``, ``Sample.played_action`` the action, ``Sample.policy_loss_mask``
(over its sum) the weight.  No counterpart in the reference, whose policy
loss is the cross-entropy to the search's policy.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from . import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_ACTIONS = 262144


class PolicyLoss(NamedTuple):
    """``loss`` is a float32 scalar; ``log_prob``, ``kl`` (float32) and
    ``clipped`` (bool) have the rows' shape; ``grad_logits`` has the logits'
    shape and type."""

    loss: torch.Tensor
    log_prob: torch.Tensor
    clipped: torch.Tensor
    kl: torch.Tensor | None = None
    grad_logits: torch.Tensor | None = None


def _rows(t: torch.Tensor, actions: int) -> torch.Tensor:
    """[..., A] as rows [N, A] of unit column stride, a view where it can be."""
    if t.requires_grad:
        t = t.detach()
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= actions:
        return t
    t = t.reshape(-1, actions)
    return t if t.stride(1) == 1 and (t.stride(0) >= actions or t.shape[0] <= 1) else t.contiguous()


def clipped_policy_loss(logits: torch.Tensor, action: torch.Tensor, old_log_prob: torch.Tensor,
                        advantage: torch.Tensor, *, legal: torch.Tensor | None = None,
                        weight: torch.Tensor | None = None, reference_logits: torch.Tensor | None = None,
                        reference_log_prob: torch.Tensor | None = None, clip_low: float = 0.2,
                        clip_high: float = 0.2, kl_coefficient: float = 0.0, gradient: bool = True) -> PolicyLoss:
    """sum_i weight_i (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) +
    kl_coefficient KL_i) with r = exp(log pi(action) - old_log_prob), over
    the legal actions, and its gradient in ``logits``.

    ``logits`` [..., actions] is float32, bfloat16 or float16 on a CUDA
    device, up to 262144 actions; rows may be strided (a slice of a padded
    vocabulary).  ``action`` (int32 or int64), ``old_log_prob``,
    ``advantage`` and ``weight`` have the leading shape; ``weight`` is a
    row's share of the loss (a mask over its sum, say; 1 / rows if absent).
    Floating point of another type is rounded to float32 first.
    ``legal`` (bool) has the logits' shape; absent, every action is legal.

    The KL term is KL(pi || reference) over the legal actions where
    ``reference_logits`` (the logits' shape and type, finite where legal) is
    given, and its estimate exp(y) - 1 - y, y = reference - log pi(action),
    where ``reference_log_prob`` is; with a coefficient of 0 the KL is a
    statistic alone.  Rows without a legal action belong into ``legal``: one
    whose logits are all masked by the type's lowest value is the uniform
    policy, and where its reference is not masked likewise, fp32 and bfloat16
    have no gradient of the KL (NaN).

    A row of weight 0, or whose action is out of range, illegal or has a
    logit of -inf, adds nothing: its statistics and gradient are 0.  An
    illegal action's logit may hold anything; its gradient is 0.

    The gradient is returned, not recorded: ``logits.backward(grad_logits)``
    continues it.  It has the logits' type, and float16 ends at 6e-8: put a
    loss scale into ``weight`` where rows are many.  The call launches on the
    current stream, does not synchronise and can be captured into a CUDA
    graph.
    """
    if logits.device.type != "cuda":
        raise ValueError("clipped_policy_loss runs on the GPU: pass logits on a CUDA device")
    if logits.dtype not in DTYPES:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_ACTIONS:
        raise ValueError(f"logits must be [..., actions] with 1 to {MAX_ACTIONS} actions, got {tuple(logits.shape)}")
    if not (0.0 <= clip_low < 1.0) or not (0.0 <= clip_high < math.inf):
        raise ValueError(f"clip_low must be in [0, 1) and clip_high finite and >= 0, got {clip_low}, {clip_high}")
    if not math.isfinite(kl_coefficient):
        raise ValueError(f"kl_coefficient must be finite, got {kl_coefficient}")
    if reference_logits is not None and reference_log_prob is not None:
        raise ValueError("pass reference_logits or reference_log_prob, not both")
    if kl_coefficient != 0.0 and reference_logits is None and reference_log_prob is None:
        raise ValueError("a KL term needs reference_logits or reference_log_prob")
    dev, lead, A = logits.device, logits.shape[:-1], logits.shape[-1]
    if action.shape != lead or action.device != dev or action.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"action must be int32 or int64 of shape {tuple(lead)} on {dev}, got {action.dtype} "
                         f"{tuple(action.shape)} on {action.device}")
    if legal is not None and (legal.shape != logits.shape or legal.device != dev
                              or legal.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"legal must be bool of shape {tuple(logits.shape)} on {dev}, got {legal.dtype} "
                         f"{tuple(legal.shape)} on {legal.device}")
    if reference_logits is not None and (reference_logits.shape != logits.shape or reference_logits.device != dev
                                         or reference_logits.dtype != logits.dtype):
        raise ValueError(f"reference_logits must match the logits ({logits.dtype} {tuple(logits.shape)} on {dev}), "
                         f"got {reference_logits.dtype} {tuple(reference_logits.shape)} on "
                         f"{reference_logits.device}")
    old_log_prob = _per_row(old_log_prob, "old_log_prob", lead, dev)
    advantage = _per_row(advantage, "advantage", lead, dev)
    if weight is not None:
        weight = _per_row(weight, "weight", lead, dev)
    if reference_log_prob is not None:
        reference_log_prob = _per_row(reference_log_prob, "reference_log_prob", lead, dev)
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _launch(logits, action, old_log_prob, advantage, legal, weight, reference_logits,
                           reference_log_prob, clip_low, clip_high, kl_coefficient, gradient)
    return _launch(logits, action, old_log_prob, advantage, legal, weight, reference_logits, reference_log_prob,
                   clip_low, clip_high, kl_coefficient, gradient)


def _per_row(t: torch.Tensor, name: str, lead: torch.Size, dev: torch.device) -> torch.Tensor:
    if t.shape != lead:
        raise ValueError(f"{name} must have shape {tuple(lead)}, got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the logits on {dev}")
    if t.dtype != torch.float32:
        if not t.is_floating_point():
            raise ValueError(f"{name} must be floating point, got {t.dtype}")
        t = t.to(torch.float32)
    return t if t.is_contiguous() else t.contiguous()


@functools.lru_cache(maxsize=1)
def _workspace_floats() -> int:
    return -(-int(_lib.lib().scacchi_policy_loss_workspace_bytes()) // 4)


def _launch(logits, action, old_log_prob, advantage, legal, weight, reference_logits, reference_log_prob, clip_low,
            clip_high, kl_coefficient, gradient) -> PolicyLoss:
    dev, lead, A = logits.device, logits.shape[:-1], logits.shape[-1]
    if action.dtype == torch.int64:
        action = action.clamp(-1, A).to(torch.int32)  # an index past 32 bits stays out of range
    if not action.is_contiguous():
        action = action.contiguous()
    if legal is not None and not legal.is_contiguous():
        legal = legal.contiguous()
    x = _rows(logits, A)
    ref = None if reference_logits is None else _rows(reference_logits, A)
    N = x.shape[0]
    # (empty_like and new_empty cost the host half of what torch.empty does)
    loss, log_prob = old_log_prob.new_empty(()), torch.empty_like(old_log_prob)
    clipped = torch.empty_like(action, dtype=torch.bool)
    kl = None if ref is None and reference_log_prob is None else torch.empty_like(old_log_prob)
    grad = None
    if gradient:
        grad = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty(logits.shape)
    workspace = old_log_prob.new_empty((_workspace_floats(),))

    def at(t):
        return None if t is None else t.data_ptr()

    rows = _lib.PolicyRows(x.data_ptr(), at(ref), at(legal), action.data_ptr(), old_log_prob.data_ptr(),
                           advantage.data_ptr(), at(weight), at(reference_log_prob), max(x.stride(0), A),
                           A if ref is None else max(ref.stride(0), A))
    out = _lib.PolicyOut(loss.data_ptr(), log_prob.data_ptr(), at(kl), clipped.data_ptr(), at(grad))
    # (the stream's bare handle: a Stream object costs the host 2.4 us more)
    _lib.check(_lib.lib().scacchi_policy_loss(rows, out, N, A, DTYPES[logits.dtype], clip_low, clip_high,
                                              kl_coefficient, workspace.data_ptr(),
                                              torch._C._cuda_getCurrentRawStream(dev.index)), "policy_loss")
    return PolicyLoss(loss, log_prob, clipped, kl, grad)
