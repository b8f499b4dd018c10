"""The clipped policy loss of a batch of played actions, with a KL term
towards a reference policy and the gradient in the logits.

It takes the frames where ``loss_input`` leaves them: ``Sample.policy_mask``
is ``legal``, ``Sample.played_action`` the action, ``Sample.policy_loss_mask``
(over its sum) the weight.  No counterpart in the reference, whose policy
loss is the cross-entropy to the search's policy.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple

import torch

from . import _lib
from .dirichlet_mctx.tree import ptr, stream_handle

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
    ``legal`` (bool) has the logits' shape; absent, every action is legal.

    The KL term is KL(pi || reference) over the legal actions where
    ``reference_logits`` (the logits' shape and type, finite where legal) is
    given, and its estimate exp(y) - 1 - y, y = reference - log pi(action),
    where ``reference_log_prob`` is.

    A row of weight 0, or whose action is out of range, illegal or has a
    logit of -inf, adds nothing: its statistics and gradient are 0.  An
    illegal action's logit may hold anything; its gradient is 0.

    The gradient is returned, not recorded: ``logits.backward(grad_logits)``
    continues it.  The call launches on the current stream, does not
    synchronise and can be captured into a CUDA graph.
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

    def per_row(t, name):
        if t.shape != lead:
            raise ValueError(f"{name} must have shape {tuple(lead)}, got {tuple(t.shape)}")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the logits on {dev}")
        if not t.is_floating_point():
            raise ValueError(f"{name} must be floating point, got {t.dtype}")
        return t.to(torch.float32).contiguous()

    if action.shape != lead or action.device != dev or action.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"action must be int32 or int64 of shape {tuple(lead)} on {dev}, got {action.dtype} "
                         f"{tuple(action.shape)} on {action.device}")
    if action.dtype == torch.int64:
        action = action.clamp(-1, A).to(torch.int32)  # an index past 32 bits stays out of range
    action = action.contiguous()
    old_log_prob, advantage = per_row(old_log_prob, "old_log_prob"), per_row(advantage, "advantage")
    if weight is not None:
        weight = per_row(weight, "weight")
    if reference_log_prob is not None:
        reference_log_prob = per_row(reference_log_prob, "reference_log_prob")
    if legal is not None:
        if legal.shape != logits.shape or legal.device != dev or legal.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"legal must be bool of shape {tuple(logits.shape)} on {dev}, got {legal.dtype} "
                             f"{tuple(legal.shape)} on {legal.device}")
        legal = legal.contiguous()
    if reference_logits is not None:
        if (reference_logits.shape != logits.shape or reference_logits.device != dev
                or reference_logits.dtype != logits.dtype):
            raise ValueError(f"reference_logits must match the logits ({logits.dtype} {tuple(logits.shape)} on {dev}), "
                             f"got {reference_logits.dtype} {tuple(reference_logits.shape)} on "
                             f"{reference_logits.device}")
        reference_logits = _rows(reference_logits.detach(), A)
    x = _rows(logits.detach(), A)
    N = x.shape[0]
    f32 = torch.float32
    with_kl = reference_logits is not None or reference_log_prob is not None
    with torch.cuda.device(dev):
        loss = torch.empty((), dtype=f32, device=dev)
        log_prob = torch.empty(lead, dtype=f32, device=dev)
        clipped = torch.empty(lead, dtype=torch.bool, device=dev)
        kl = torch.empty(lead, dtype=f32, device=dev) if with_kl else None
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if gradient else None
        workspace = torch.empty((_workspace_bytes(),), dtype=torch.uint8, device=dev)
        rows = _lib.PolicyRows(ptr(x), ptr(reference_logits), ptr(legal), ptr(action), ptr(old_log_prob),
                               ptr(advantage), ptr(weight), ptr(reference_log_prob), max(x.stride(0), A),
                               A if reference_logits is None else max(reference_logits.stride(0), A))
        out = _lib.PolicyOut(ptr(loss), ptr(log_prob), ptr(kl), ptr(clipped), ptr(grad))
        _lib.check(_lib.lib().scacchi_policy_loss(C.byref(rows), C.byref(out), N, A, DTYPES[logits.dtype],
                                                  float(clip_low), float(clip_high), float(kl_coefficient),
                                                  ptr(workspace), stream_handle(dev)), "policy_loss")
    return PolicyLoss(loss=loss, log_prob=log_prob, clipped=clipped, kl=kl, grad_logits=grad)


_workspace = []


def _workspace_bytes() -> int:
    if not _workspace:
        _workspace.append(int(_lib.lib().scacchi_policy_loss_workspace_bytes()))
    return _workspace[0]
