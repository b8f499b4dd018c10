"""AdamW over many tensors in one launch, with moments in 32 or in 8 bits,
and the norm of many gradients (the reference trains with Muon and Adam;
this is the part for whatever is no matrix).

``AdamW`` steps any float32 or bfloat16 tensors by name.  ``NetworkAdamW``
holds what ``muon.NetworkMuon`` leaves of the network's parameters: the
stem, the 1x1 convolutions, output vectors, biases and BatchNorm.

Moments lie in one buffer each, tensor after tensor at offsets that are
multiples of 256 (``AdamW.views``).  Those of 8 bits hold the first moment m
and the root r of the second, a block of 256 under one power of two: an
exponent byte E and a code c with the value

    2^(E - 127) f(c),   f = 2^(e - 14) (1 + t)  for e > 0, 2^-13 t  for e = 0

where r's eight bits are four of e and four of the fraction t, m's a sign,
four of e and three of t.  The block's largest element has e = 14; E = 255
marks a block that holds what is not finite, all of it NaN.  Codes are
rounded up or down by random bits, so that a moment moves by less than a
code's step a step on average; see ``AdamW``.
"""

from __future__ import annotations

import ctypes as C
import dataclasses
import functools
import math
from collections.abc import Iterable, Mapping

import numpy as np
import torch

from . import _lib
from .muon import DENSE
from .network import AZDirichletParams, BatchNormParams

GRADIENT_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
WEIGHT_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
BLOCK = 256
STATE_WORDS = 8  # int64 words of the step's count and scalars
TENSOR = np.dtype([("weight", np.uint64), ("gradient", np.uint64), ("count", np.int64), ("offset", np.int64),
                   ("weight_decay", np.float64), ("weight_dtype", np.int32), ("gradient_dtype", np.int32)])


@functools.lru_cache(maxsize=64)
def _norm_workspace_doubles(tensors: int) -> int:
    return -(-int(_lib.lib().scacchi_gradient_norm_workspace_bytes(tensors)) // 8)


def _norm(table: np.ndarray, device: torch.device) -> torch.Tensor:
    """The norm of a table's gradients, on the current device."""
    out = torch.empty((), dtype=torch.float32, device=device)
    workspace = torch.empty((_norm_workspace_doubles(len(table)),), dtype=torch.float64, device=device)
    _lib.check(_lib.lib().scacchi_gradient_norm(table.ctypes.data, len(table), out.data_ptr(), workspace.data_ptr(),
                                                torch._C._cuda_getCurrentRawStream(device.index)), "gradient_norm")
    return out


def gradient_norm(gradients: Iterable[torch.Tensor] | Mapping[str, torch.Tensor]) -> torch.Tensor:
    """sqrt(sum of squares) over all gradients, a float32 scalar.

    The gradients (float32, bfloat16 or float16, mixed as they come, of any
    shape; a mapping's values) are on one CUDA device.  Squares are summed in
    64 bits in an order that depends on the sizes alone; an infinity or a NaN
    in any of them gives an infinity or NaN.  A strided gradient is copied
    first.

    The call launches on the current stream, does not synchronise and can be
    captured into a CUDA graph.
    """
    grads = list(gradients.values() if isinstance(gradients, Mapping) else gradients)
    done = _lib.host().gradient_norm(grads)
    if done is not None:
        return done
    if not grads:
        raise ValueError("gradient_norm needs at least one gradient")
    for g in grads:
        if not isinstance(g, torch.Tensor):
            raise ValueError(f"gradients must be tensors, got {type(g).__name__}")
    device = grads[0].device
    if device.type != "cuda":
        raise ValueError("gradient_norm runs on the GPU: pass gradients on a CUDA device")
    index = device.index
    dtypes = [GRADIENT_DTYPES.get(g.dtype, -1) for g in grads]
    if -1 in dtypes:
        raise ValueError(f"gradients must be float32, bfloat16 or float16, got {grads[dtypes.index(-1)].dtype}")
    if any([g.get_device() != index for g in grads]):
        raise ValueError(f"gradients must be on one device, got {sorted({str(g.device) for g in grads})}")
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _gradient_norm(grads, dtypes, device)
    return _gradient_norm(grads, dtypes, device)


def _gradient_norm(grads: list, dtypes: list, device: torch.device) -> torch.Tensor:
    if not all([g.is_contiguous() for g in grads]):
        grads = [g.detach().contiguous() for g in grads]
    table = np.zeros(len(grads), TENSOR)
    table["gradient"] = [g.data_ptr() for g in grads]
    table["count"] = [g.numel() for g in grads]
    table["gradient_dtype"] = dtypes
    return _norm(table, device)


class AdamW:
    """AdamW over tensors by name, in place on them:

        g <- g max_norm / max(norm, max_norm)          (with max_norm)
        first <- beta1 first + (1 - beta1) g
        second <- beta2 second + (1 - beta2) g^2
        weight <- (1 - learning_rate weight_decay) weight - learning_rate
                  (first / (1 - beta1^t)) / (sqrt(second / (1 - beta2^t)) + eps)

    ``weights`` are contiguous float32 or bfloat16 tensors on one CUDA
    device that do not overlap; they are kept and changed in place.
    ``weight_decay`` is one number or one for each name.  ``state_bits`` is
    32, or 8 for moments of a byte an element and two in 256 elements.

    ``key`` (two 32-bit words, ``random.PRNGKey``) is what 8-bit moments and
    bfloat16 weights are rounded by: up or down at random, right on average,
    so that steps too small for a code or a bfloat16 add up.  The random bits
    depend on the key, the step's count and the element's place alone.  8-bit
    moments need one; without one bfloat16 weights round to nearest.

    A first moment that fades below 2^-17 of its block's largest is lost now
    and then; a root is never rounded to zero.

    Squares of gradients above 1.8e19 are infinite in 32 bits: the weight then
    rests (all but its decay), and 8-bit moments lose that block of 256, whose
    weights are NaN from the next step on.  ``max_norm`` keeps gradients below.
    """

    def __init__(self, weights: Mapping[str, torch.Tensor], *, learning_rate: float, beta1: float = 0.9,
                 beta2: float = 0.999, eps: float = 1e-8, weight_decay: float | Mapping[str, float] = 0.0,
                 max_norm: float | None = None, state_bits: int = 32, key=None):
        if not weights:
            raise ValueError("AdamW needs at least one weight")
        for name, b in (("beta1", beta1), ("beta2", beta2)):
            if not 0.0 <= b < 1.0:
                raise ValueError(f"{name} must be in [0, 1), got {b}")
        if not (eps == 0.0 or 1e-30 <= eps <= 1e30):
            raise ValueError(f"eps must be 0 or in [1e-30, 1e30], got {eps}")
        if not math.isfinite(learning_rate):
            raise ValueError(f"learning_rate must be finite, got {learning_rate}")
        if max_norm is not None and not 0.0 < max_norm < math.inf:
            raise ValueError(f"max_norm must be finite and > 0, got {max_norm}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if state_bits == 8 and key is None:
            raise ValueError("8-bit moments are rounded by random bits: pass a key")
        if isinstance(weight_decay, Mapping):
            if set(weight_decay) != set(weights):
                raise ValueError("weight_decay must have one number for each weight; differs in "
                                 f"{sorted(set(weight_decay) ^ set(weights))}")
            decay = [float(weight_decay[name]) for name in weights]
        else:
            decay = [float(weight_decay)] * len(weights)
        if not all(math.isfinite(d) for d in decay):
            raise ValueError(f"weight_decay must be finite, got {weight_decay}")
        device = next(iter(weights.values())).device
        if device.type != "cuda":
            raise ValueError("AdamW runs on the GPU: pass weights on a CUDA device")
        at, spans = 0, []
        table = np.zeros(len(weights), TENSOR)
        for i, (name, w) in enumerate(weights.items()):
            if w.dtype not in WEIGHT_DTYPES or w.device != device:
                raise ValueError(f"{name} must be float32 or bfloat16 on {device}, got {w.dtype} on {w.device}")
            if not w.is_contiguous():
                raise ValueError(f"{name} is updated in place and must be contiguous")
            n = w.numel()
            table[i] = (w.data_ptr(), 0, n, at, decay[i], WEIGHT_DTYPES[w.dtype], 0)
            at += -(-n // BLOCK) * BLOCK
            if n:
                spans.append((w.data_ptr(), w.data_ptr() + n * w.element_size(), name))
        spans.sort()
        for a, b in zip(spans, spans[1:]):
            if b[0] < a[1]:
                raise ValueError(f"{a[2]} and {b[2]} share memory")
        words = (0, 0) if key is None else tuple(int(k) & 0xFFFFFFFF for k in np.asarray(key, np.uint32).reshape(2))
        self.weights, self.device, self.state_bits = dict(weights), device, state_bits
        self.max_norm = None if max_norm is None else float(max_norm)
        self._names, self._tensors = tuple(weights), tuple(weights.values())
        self._shapes = [w.shape for w in self._tensors]
        self._table = table
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self.first = torch.zeros((at,), dtype=kind, device=device)
        self.second = torch.zeros((at,), dtype=kind, device=device)
        self.first_exponent = self.second_exponent = None
        if state_bits == 8:
            self.first_exponent = torch.full((at // BLOCK,), 27, dtype=torch.uint8, device=device)
            self.second_exponent = self.first_exponent.clone()
        self._state = torch.zeros((STATE_WORDS,), dtype=torch.int64, device=device)

        def ptr(t):
            return None if t is None else t.data_ptr()

        self._params = _lib.AdamWStep(
            state_bits, int(key is not None), float(learning_rate), float(beta1), float(beta2), float(max_norm or 0.0),
            float(eps), words[0], words[1], at, ptr(self.first), ptr(self.second), ptr(self.first_exponent),
            ptr(self.second_exponent), ptr(self._state), None, None)

    def _gradients(self, gradients: Mapping[str, torch.Tensor]) -> list:
        """The gradients in the weights' order, dense, None where there is none."""
        grads = list(map(gradients.get, self._names))
        unknown = set(gradients).difference(self._names)
        if unknown:
            raise ValueError(f"no such weights: {sorted(unknown)}; expected some of {sorted(self._names)}")
        index, dense = self.device.index, True
        for i, g in enumerate(grads):
            if g is None:
                continue
            if not isinstance(g, torch.Tensor):
                raise ValueError(f"the gradient of {self._names[i]} must be a tensor, got {type(g).__name__}")
            if g.shape != self._shapes[i] or g.get_device() != index or g.dtype not in GRADIENT_DTYPES:
                raise ValueError(f"the gradient of {self._names[i]} must be float32, bfloat16 or float16 "
                                 f"{tuple(self._shapes[i])} on {self.device}, got {g.dtype} {tuple(g.shape)} on "
                                 f"{g.device}")
            dense &= g.is_contiguous()
        if not dense:
            grads = [None if g is None else g.detach().contiguous() for g in grads]
        return grads

    def step(self, gradients: Mapping[str, torch.Tensor], *, norm: torch.Tensor | None = None,
             learning_rate: float | torch.Tensor | None = None) -> torch.Tensor | None:
        """One step with the gradients (float32, bfloat16 or float16, of the
        weights' shapes).  A weight without one stays as it is, and so do its
        moments; the count of steps is one for all.

        With ``max_norm`` the gradients are clipped by ``norm``, a float32
        scalar on the device (``gradient_norm`` of more than these gradients,
        say), or by their own norm.  A norm that is not finite skips the step
        as a whole, its count too.  Returns the norm, None without
        ``max_norm``.

        ``learning_rate`` replaces the constructor's; a float32 scalar on the
        device is read when the step runs, so a captured step can follow a
        schedule.  Gradients may not overlap the weights or the moments.  The
        call launches on the current stream, does not synchronise and can be
        captured into a CUDA graph.
        """
        done = _lib.host().adamw_step(self._names, self._tensors, gradients, self._table.ctypes.data,
                                      C.addressof(self._params), self.device.index, self.max_norm, norm, learning_rate)
        if done is not None:
            return done[0]
        grads = self._gradients(gradients)
        for name, t in (("norm", norm), ("learning_rate", learning_rate)):
            if isinstance(t, torch.Tensor) and (t.dtype != torch.float32 or t.numel() != 1 or t.device != self.device):
                raise ValueError(f"{name} must be one float32 on {self.device}, got {t.dtype} {tuple(t.shape)} on "
                                 f"{t.device}")
        if norm is not None and not isinstance(norm, torch.Tensor):
            raise ValueError(f"norm must be one float32 on {self.device}, got {type(norm).__name__}")
        if norm is not None and self.max_norm is None:
            raise ValueError("a norm is of use with max_norm alone")
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self._step(grads, norm, learning_rate)
        return self._step(grads, norm, learning_rate)

    def _step(self, grads: list, norm, learning_rate):
        table = self._table.copy()  # (the call lets other threads run, and they may step too)
        for name, w, row in zip(self._names, self._tensors, table):
            if (w.device != self.device or w.numel() != row["count"] or not w.is_contiguous()
                    or WEIGHT_DTYPES.get(w.dtype) != row["weight_dtype"]):
                raise ValueError(f"{name} has changed its device, size, type or layout since AdamW was made")
        table["weight"] = [w.data_ptr() for w in self._tensors]
        table["gradient"] = [0 if g is None else g.data_ptr() for g in grads]
        table["gradient_dtype"] = [0 if g is None else GRADIENT_DTYPES[g.dtype] for g in grads]
        if self.max_norm is not None and norm is None:
            norm = _norm(table[[g is not None for g in grads]], self.device)
        params = _lib.AdamWStep.from_buffer_copy(self._params)
        if norm is not None:
            params.norm, params.max_norm = norm.data_ptr(), float(self.max_norm)
        if isinstance(learning_rate, torch.Tensor):
            params.learning_rate_at = learning_rate.data_ptr()
        elif learning_rate is not None:
            if not math.isfinite(learning_rate):
                raise ValueError(f"learning_rate must be finite, got {learning_rate}")
            params.learning_rate = float(learning_rate)
        rc = _lib.lib().scacchi_adamw_step(C.byref(params), table.ctypes.data, len(table),
                                           torch._C._cuda_getCurrentRawStream(self.device.index))
        if rc == _lib.EINVAL:
            raise ValueError("a gradient, the norm or the learning rate overlaps a weight or the moments, or two "
                             "weights do")
        _lib.check(rc, "adamw_step")
        # a graph recorded before the step refuses to run backward through it
        torch.autograd.graph.increment_version([w for w, g in zip(self._tensors, grads) if g is not None])
        return norm

    def steps(self) -> int:
        """Steps taken; synchronises."""
        return int(self._state[0])

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(first moment, root of the second) of all tensors, in one buffer
        each (``views``).  Those of 8 bits come as the bfloat16 values that
        their codes stand for, without rounding; those of 32 as float32."""
        if self.state_bits == 32:
            return self.first.clone(), self.second.sqrt()
        done = _lib.host().adamw_moments(self.first, self.second, self.first_exponent, self.second_exponent)
        if done is not None:
            return done
        with torch.cuda.device(self.device):
            first = torch.empty(self.first.shape, dtype=torch.bfloat16, device=self.device)
            root = torch.empty_like(first)
            _lib.check(_lib.lib().scacchi_adamw_moments(
                self.first.data_ptr(), self.second.data_ptr(), self.first_exponent.data_ptr(),
                self.second_exponent.data_ptr(), self.first.numel(), first.data_ptr(), root.data_ptr(),
                torch._C._cuda_getCurrentRawStream(self.device.index)), "adamw_moments")
        return first, root

    def views(self, flat: torch.Tensor) -> dict[str, torch.Tensor]:
        """The parts of a moments' buffer by name, in the weights' shapes."""
        if flat.shape != self.first.shape:
            raise ValueError(f"expected a buffer of {tuple(self.first.shape)}, got {tuple(flat.shape)}")
        return {name: flat[int(row["offset"]):int(row["offset"] + row["count"])].view(w.shape)
                for name, w, row in zip(self._names, self._tensors, self._table)}

    def state_dict(self) -> dict:
        """The count of steps (synchronises) and the moments' buffers
        themselves: copy them before the next step if they are to stay."""
        out = dict(step=self.steps(), first=self.first, second=self.second)
        if self.state_bits == 8:
            out |= dict(first_exponent=self.first_exponent, second_exponent=self.second_exponent)
        return out

    def load_state_dict(self, state: Mapping) -> None:
        """Copies what ``state_dict`` gave for the same weights and bits."""
        own = dict(first=self.first, second=self.second)
        if self.state_bits == 8:
            own |= dict(first_exponent=self.first_exponent, second_exponent=self.second_exponent)
        if set(state) != {"step", *own}:
            raise ValueError(f"expected {sorted({'step', *own})}, got {sorted(state)}")
        if not 0 <= int(state["step"]) < 1 << 62:
            raise ValueError(f"step must not be negative, got {state['step']}")
        for name, t in own.items():
            if state[name].shape != t.shape or state[name].dtype != t.dtype:
                raise ValueError(f"{name} must be {t.dtype} {tuple(t.shape)}, got {state[name].dtype} "
                                 f"{tuple(state[name].shape)}")
        for name, t in own.items():
            t.copy_(state[name])
        self._state[0] = int(state["step"])


def _network_arrays(params: AZDirichletParams) -> dict[str, np.ndarray]:
    """What no matrix of NetworkMuon holds, by name: BatchNorm's scale and
    bias (its statistics are no parameters), blocks as "blocks.0.conv1_b"."""
    def parts(prefix, value):
        if isinstance(value, BatchNormParams):
            return {f"{prefix}.scale": value.scale, f"{prefix}.bias": value.bias}
        return {prefix: value}

    out = {}
    for field in dataclasses.fields(params):
        value = getattr(params, field.name)
        if field.name == "blocks":
            for i, blk in enumerate(value):
                for k, v in blk.items():
                    if k not in ("conv1_w", "conv2_w"):
                        out |= parts(f"blocks.{i}.{k}", v)
        elif field.name != "num_actions" and field.name not in DENSE:
            out |= parts(field.name, value)
    return out


class NetworkAdamW(AdamW):
    """AdamW over what ``NetworkMuon`` leaves of ``AZDirichletParams``:
    ``weights`` by name, BatchNorm as "policy_bn.scale", the blocks' as
    "blocks.0.bn1.bias".  ``weight_decay`` holds for the kernels (the stem,
    1x1 convolutions and output vectors); biases and BatchNorm have none.

    ``params`` gives the parameters with these weights in place; hand it
    ``NetworkMuon.params()`` for the whole network:
    ``adam.params(muon.params())``."""

    def __init__(self, params: AZDirichletParams, *, learning_rate: float, weight_decay: float = 0.0, device="cuda",
                 **settings):
        self._base = params
        weights = {k: torch.tensor(np.asarray(v, np.float32), device=device)
                   for k, v in _network_arrays(params).items()}
        decay = {k: float(weight_decay) if w.dim() > 1 else 0.0 for k, w in weights.items()}
        super().__init__(weights, learning_rate=learning_rate, weight_decay=decay, **settings)

    def params(self, base: AZDirichletParams | None = None) -> AZDirichletParams:
        base = self._base if base is None else base
        host = {k: w.detach().cpu().numpy() for k, w in self.weights.items()}

        def put(prefix, value):
            if isinstance(value, BatchNormParams):
                return dataclasses.replace(value, scale=host[f"{prefix}.scale"], bias=host[f"{prefix}.bias"])
            return host.get(prefix, value)

        changes = {f.name: put(f.name, getattr(base, f.name)) for f in dataclasses.fields(base)
                   if f.name not in ("blocks", "num_actions")}
        changes["blocks"] = [{k: put(f"blocks.{i}.{k}", v) for k, v in blk.items()}
                             for i, blk in enumerate(base.blocks)]
        return dataclasses.replace(base, **changes)
