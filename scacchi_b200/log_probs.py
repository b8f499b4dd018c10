"""Log-probabilities of played actions, with the rows' entropy and best
actions, and their gradient in the logits.

They stand before and beside ``policy_loss``: the behaviour policy's
``log_prob`` of ``Sample.played_action`` over ``Sample.policy_mask`` is that
loss's ``old_log_prob``; the entropy and its gradient are an entropy bonus;
the best actions are what a frame's analysis shows.  No counterpart in the
reference.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .policy_loss import DTYPES, MAX_ACTIONS, _per_row, _rows

MAX_TOP = 32


class LogProbs(NamedTuple):
    """Float32 of the rows' shape; ``top_log_prob`` (float32) and
    ``top_action`` (int32) have one more axis of ``top`` entries."""

    log_prob: torch.Tensor | None
    entropy: torch.Tensor
    max_logit: torch.Tensor
    log_sum: torch.Tensor
    top_log_prob: torch.Tensor | None = None
    top_action: torch.Tensor | None = None


def _check(what: str, logits: torch.Tensor, action: torch.Tensor, legal: torch.Tensor | None, temperature: float):
    if logits.device.type != "cuda":
        raise ValueError(f"{what} runs on the GPU: pass logits on a CUDA device")
    if logits.dtype not in DTYPES:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_ACTIONS:
        raise ValueError(f"logits must be [..., actions] with 1 to {MAX_ACTIONS} actions, got {tuple(logits.shape)}")
    dev, lead = logits.device, logits.shape[:-1]
    if action.shape != lead or action.device != dev or action.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"action must be int32 or int64 of shape {tuple(lead)} on {dev}, got {action.dtype} "
                         f"{tuple(action.shape)} on {action.device}")
    if legal is not None and (legal.shape != logits.shape or legal.device != dev
                              or legal.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"legal must be bool of shape {tuple(logits.shape)} on {dev}, got {legal.dtype} "
                         f"{tuple(legal.shape)} on {legal.device}")
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError(f"temperature must be in [1e-3, 1e3], got {temperature}")


def _at(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _struct(logits, action, legal):
    """The rows as the library takes them, and what holds their memory."""
    A = logits.shape[-1]
    if action.dtype == torch.int64:
        action = action.clamp(-1, A).to(torch.int32)  # an index past 32 bits stays out of range
    if not action.is_contiguous():
        action = action.contiguous()
    if legal is not None and not legal.is_contiguous():
        legal = legal.contiguous()
    x = _rows(logits, A)
    return _lib.LogProbRows(x.data_ptr(), _at(legal), action.data_ptr(), max(x.stride(0), A)), (x, legal, action)


def policy_log_probs(logits: torch.Tensor, action: torch.Tensor, *, legal: torch.Tensor | None = None,
                     temperature: float = 1.0, top: int = 0) -> LogProbs:
    """log softmax(logits / temperature)[action] over the legal actions, the
    distribution's entropy and its ``top`` likeliest actions.

    ``logits`` [..., actions] is float32, bfloat16 or float16 on a CUDA
    device, up to 262144 actions; rows may be strided (a slice of a padded
    vocabulary).  ``action`` (int32 or int64) has the leading shape,
    ``legal`` (bool) the logits'; absent, every action is legal.
    ``temperature`` is in [1e-3, 1e3], ``top`` in [0, 32].

    An action out of range (a padded frame's -1) has log-probability 0, one
    that is illegal or has a logit of -inf minus infinity.  Best actions come
    in order, the lower index first among equal logits, with -1 and minus
    infinity behind the last one that is legal and above -inf.  A row without
    any has entropy 0, ``max_logit`` and ``log_sum`` minus infinity; one
    whose logits all are the type's lowest value is uniform.  An illegal
    action's logit may hold anything; a NaN or +inf among the legal ones
    makes the row's numbers NaN (a log-probability stays 0 or minus infinity
    where the action has none), its best actions unspecified.

    ``max_logit`` and ``log_sum`` (log sum exp((x - max_logit) /
    temperature)) are what ``policy_log_probs_gradient`` needs.  The result
    is outside autograd.  The call launches on the current stream, does not
    synchronise and can be captured into a CUDA graph.
    """
    done = _lib.host().log_probs(logits, action, legal, temperature, top)
    if done is not None:
        return LogProbs(*done)
    _check("policy_log_probs", logits, action, legal, temperature)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be in [0, {MAX_TOP}], got {top}")
    if torch.cuda.current_device() != logits.device.index:
        with torch.cuda.device(logits.device):
            return _log_probs(logits, action, legal, temperature, top)
    return _log_probs(logits, action, legal, temperature, top)


def _log_probs(logits, action, legal, temperature, top) -> LogProbs:
    dev, lead = logits.device, logits.shape[:-1]
    rows, held = _struct(logits, action, legal)
    numbers = torch.empty((4, *lead), dtype=torch.float32, device=dev)
    log_prob, entropy, max_logit, log_sum = numbers.unbind(0)
    top_log_prob = top_action = None
    if top:
        top_log_prob = torch.empty((*lead, top), dtype=torch.float32, device=dev)
        top_action = torch.empty_like(top_log_prob, dtype=torch.int32)
    at = numbers.data_ptr()
    n = held[0].shape[0]
    out = _lib.LogProbOut(at, at + 4 * n, at + 8 * n, at + 12 * n, _at(top_log_prob), _at(top_action))
    _lib.check(_lib.lib().scacchi_log_probs(rows, out, n, logits.shape[-1], DTYPES[logits.dtype], temperature, top,
                                            torch._C._cuda_getCurrentRawStream(dev.index)), "policy_log_probs")
    return LogProbs(log_prob, entropy, max_logit, log_sum, top_log_prob, top_action)


def policy_log_probs_gradient(logits: torch.Tensor, action: torch.Tensor, out: LogProbs, *,
                              grad_log_prob: torch.Tensor | None = None, grad_entropy: torch.Tensor | None = None,
                              legal: torch.Tensor | None = None, temperature: float = 1.0) -> torch.Tensor:
    """The gradient in ``logits`` of sum(grad_log_prob log_prob +
    grad_entropy entropy), in their shape and type.

    ``out`` is what ``policy_log_probs`` gave for the same logits, actions,
    mask and temperature (its entropy, max_logit and log_sum are read).  The
    gradients are floating point of the rows' shape; either may be absent,
    not both.  An action without a log-probability (out of range, illegal,
    -inf) has no gradient of it; illegal actions and those of -inf have 0
    (in a row whose numbers or gradients are not finite it may be NaN
    throughout).

    The gradient is returned, not recorded: ``logits.backward(gradient)``
    continues it.  float16 ends at 6e-8: put a loss scale into the gradients
    where rows are many.  The call launches on the current stream, does not
    synchronise and can be captured into a CUDA graph.
    """
    done = _lib.host().log_probs_gradient(logits, action, legal, temperature, out.max_logit, out.log_sum, out.entropy,
                                          grad_log_prob, grad_entropy)
    if done is not None:
        return done
    _check("policy_log_probs_gradient", logits, action, legal, temperature)
    if grad_log_prob is None and grad_entropy is None:
        raise ValueError("pass grad_log_prob, grad_entropy or both")
    dev, lead = logits.device, logits.shape[:-1]
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _gradient(logits, action, out, grad_log_prob, grad_entropy, legal, temperature, dev, lead)
    return _gradient(logits, action, out, grad_log_prob, grad_entropy, legal, temperature, dev, lead)


def _gradient(logits, action, out, grad_log_prob, grad_entropy, legal, temperature, dev, lead) -> torch.Tensor:
    if grad_log_prob is not None:
        grad_log_prob = _per_row(grad_log_prob, "grad_log_prob", lead, dev)
    entropy = None
    if grad_entropy is not None:
        grad_entropy = _per_row(grad_entropy, "grad_entropy", lead, dev)
        entropy = _per_row(out.entropy, "out.entropy", lead, dev)
    max_logit = _per_row(out.max_logit, "out.max_logit", lead, dev)
    log_sum = _per_row(out.log_sum, "out.log_sum", lead, dev)
    rows, held = _struct(logits, action, legal)
    grad = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty(logits.shape)
    _lib.check(_lib.lib().scacchi_log_probs_gradient(
        rows, max_logit.data_ptr(), log_sum.data_ptr(), _at(entropy), _at(grad_log_prob), _at(grad_entropy),
        held[0].shape[0], logits.shape[-1], DTYPES[logits.dtype], temperature, grad.data_ptr(),
        torch._C._cuda_getCurrentRawStream(dev.index)), "policy_log_probs_gradient")
    return grad.detach()
