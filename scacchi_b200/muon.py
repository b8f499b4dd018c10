"""Muon for the network's matrices: the orthogonalised update and the
weight's step (the reference trains with Muon and Adam; this is the part
for matrices).

A weight is a matrix [in, out] as flax stores it: the dense kernels of
``AZDirichletParams`` as they are, a convolution kernel [3, 3, in, out] as
its [9 in, out] reshape.  Leading axes stack matrices of one shape, which
one call updates together.

``NetworkMuon`` holds the network's matrices in that form (the blocks'
convolutions as one stack), steps them, and gives back the parameters that
``AZDirichletNet`` evaluates.
"""

from __future__ import annotations

import ctypes as C
import dataclasses
import functools
import math

import numpy as np
import torch

from . import _lib
from .dirichlet_mctx.tree import ptr, stream_handle
from .network import AZDirichletParams

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_SIDE = 131072
MAX_STACK = 65535


@functools.lru_cache(maxsize=64)
def _scale_exponent(a: float, b: float, c: float, steps: int) -> int:
    e = int(_lib.lib().scacchi_muon_scale_exponent(a, b, c, steps))
    if e < 0:
        raise ValueError(f"coefficients {(a, b, c)} diverge within {steps} steps from singular values in [0, 1], or "
                         "have 0 < 16 |c| < |b|")
    return e


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(batch: int, rows: int, cols: int) -> int:
    return int(_lib.lib().scacchi_muon_workspace_bytes(batch, rows, cols))


def check_waits(device=None) -> None:
    """Raises ScacchiError where a wait of these operators ran out on
    ``device`` (the current one if absent) since the last call, so that
    their results are not to be trusted.  Speaks of the work that is
    complete: synchronise first."""
    with torch.cuda.device(device):
        if _lib.muon_error():
            raise _lib.ScacchiError("a wait of an orthogonalised update ran out: its results are incomplete")


def _params(t: torch.Tensor, name: str, steps: int, coefficients, eps: float) -> _lib.NewtonSchulz:
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a CUDA device, got {t.device}")
    if t.dtype not in DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() < 2:
        raise ValueError(f"{name} must be [..., rows, cols], got {tuple(t.shape)}")
    rows, cols = t.shape[-2:]
    batch = math.prod(t.shape[:-2])
    if not (1 <= rows <= MAX_SIDE and 1 <= cols <= MAX_SIDE) or batch > MAX_STACK:
        raise ValueError(f"{name} must stack at most {MAX_STACK} matrices with sides of 1 to {MAX_SIDE}, got "
                         f"{tuple(t.shape)}")
    if not 1 <= steps <= 64:
        raise ValueError(f"steps must be in [1, 64], got {steps}")
    a, b, c = (float(v) for v in coefficients)
    if not all(math.isfinite(v) for v in (a, b, c)):
        raise ValueError(f"coefficients must be finite, got {tuple(coefficients)}")
    if not (0.0 <= eps < math.inf):
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    return _lib.NewtonSchulz(batch, rows, cols, DTYPES[t.dtype], int(steps), _scale_exponent(a, b, c, int(steps)),
                             a, b, c, float(eps))


def orthogonalize(matrix: torch.Tensor, *, steps: int = 5, coefficients=COEFFICIENTS,
                  eps: float = 1e-8) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of each matrix of [..., rows, cols].

    X = U / (|U|_F + eps), then ``steps`` times X <- a X + (b A + c A^2) X
    with A = X X^T on the narrow side; returns X in the input's shape and
    type (float32, bfloat16 or float16).  The products carry 32-bit
    accuracy whatever the type, and round once at the end.  A matrix of
    zeros gives zeros (NaN where ``eps`` is 0); one with an infinity or a
    NaN gives NaN, and leaves the others of its stack alone.  The result is
    outside autograd.

    The call launches on the current stream, does not synchronise and can
    be captured into a CUDA graph.  It cannot report a product whose wait
    ran out (2 s): the output then stays unwritten in part or as a whole,
    and ``check_waits``, at a point where the program synchronises, raises.
    """
    matrix = matrix.detach()
    params = _params(matrix, "matrix", steps, coefficients, eps)
    dev = matrix.device
    with torch.cuda.device(dev):
        x = matrix.contiguous()
        out = torch.empty_like(x)
        if x.numel():
            workspace = torch.empty((_workspace_bytes(params.batch, params.rows, params.cols),), dtype=torch.uint8,
                                    device=dev)
            _lib.check(_lib.lib().scacchi_orthogonalize(C.byref(params), ptr(x), ptr(out), ptr(workspace),
                                                        stream_handle(dev)), "orthogonalize")
    return out


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two dense tensors share memory."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    return (a.data_ptr() < b.data_ptr() + b.numel() * b.element_size()
            and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size())


def _span(t: torch.Tensor) -> torch.Tensor:
    """All memory from a tensor's first element to its last, as a dense one."""
    return t if t.is_contiguous() else t.as_strided((1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())),), (1,))


def muon_update(weight: torch.Tensor, gradient: torch.Tensor, momentum: torch.Tensor, *, learning_rate: float,
                beta: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, scale: float | None = None,
                steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-8) -> None:
    """Muon's step, in place on ``weight`` and ``momentum``:

        momentum <- beta momentum + (1 - beta) gradient
        u = (1 - beta) gradient + beta momentum   (nesterov; else momentum)
        weight <- (1 - learning_rate weight_decay) weight
                  - learning_rate scale orthogonalize(u)

    ``weight`` and ``momentum`` are contiguous float32 [..., in, out] of one
    shape (state is kept in 32 bits); ``gradient`` has that shape in
    float32, bfloat16 or float16.  ``scale`` defaults to
    sqrt(max(1, out / in)).  The three may not overlap.

    The call launches on the current stream, does not synchronise and can
    be captured into a CUDA graph.  It cannot report a product whose wait
    ran out (2 s): ``momentum`` is then the step's, ``weight`` unwritten in
    part or as a whole, and ``check_waits``, at a point where the program
    synchronises, raises.
    """
    gradient = gradient.detach()
    params = _params(gradient, "gradient", steps, coefficients, eps)
    dev = gradient.device
    for name, t in (("weight", weight), ("momentum", momentum)):
        if t.dtype != torch.float32 or t.shape != gradient.shape or t.device != dev:
            raise ValueError(f"{name} must be float32 {tuple(gradient.shape)} on {dev}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} is updated in place and must be contiguous")
    g = gradient.contiguous()
    if _overlap(weight, g) or _overlap(weight, momentum) or _overlap(g, momentum):
        raise ValueError("weight, gradient and momentum may not overlap")
    if not 0.0 <= beta < 1.0:
        raise ValueError(f"beta must be in [0, 1), got {beta}")
    if scale is None:
        scale = math.sqrt(max(1.0, params.cols / params.rows))
    decay, step = 1.0 - learning_rate * weight_decay, learning_rate * scale
    if not (math.isfinite(decay) and math.isfinite(step)):
        raise ValueError(f"learning_rate, weight_decay and scale must be finite, got {learning_rate}, {weight_decay}, "
                         f"{scale}")
    if weight.numel() == 0:
        return
    with torch.cuda.device(dev):
        workspace = torch.empty((_workspace_bytes(params.batch, params.rows, params.cols),), dtype=torch.uint8,
                                device=dev)
        _lib.check(_lib.lib().scacchi_muon_update(C.byref(params), ptr(g), ptr(momentum), ptr(weight), float(beta),
                                                  int(bool(nesterov)), decay, step, ptr(workspace),
                                                  stream_handle(dev)), "muon_update")
    # a graph recorded before the step refuses to run backward through it
    torch.autograd.graph.increment_version((weight, momentum))


# the dense kernels; the blocks' convolutions are the stack "convs"
DENSE = ("policy_w", "value_w", "q_dir_w", "q_dir_out_w", "q_conc_w", "q_conc_out_w")


class NetworkMuon:
    """Muon over the matrices of ``AZDirichletParams``: the blocks'
    convolutions as one stack ``convs`` [2 blocks, 9 channels, channels] (in
    order: block 0's first, its second, block 1's first, ...) and the dense
    kernels of DENSE by their names.

    ``step`` takes gradients of any of them, in their shapes; ``params``
    gives the updated parameters, and raises ScacchiError where a wait of a
    step ran out (``check_waits``).  The stem, the 1x1 convolutions, the
    output vectors, biases and BatchNorm are not matrices to orthogonalise
    and stay as they were given (``adamw.NetworkAdamW`` steps them beside it).
    """

    def __init__(self, params: AZDirichletParams, *, learning_rate: float, beta: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-8,
                 device="cuda"):
        self._params = params
        self.settings = dict(learning_rate=learning_rate, beta=beta, nesterov=nesterov, weight_decay=weight_decay,
                             steps=steps, coefficients=coefficients, eps=eps)
        kernels = [blk[k] for blk in params.blocks for k in ("conv1_w", "conv2_w")]
        convs = np.stack([k.reshape(-1, k.shape[-1]) for k in kernels])
        host = {"convs": convs, **{name: getattr(params, name) for name in DENSE}}
        self.matrices = {k: torch.tensor(np.asarray(v, np.float32), device=device) for k, v in host.items()}
        self.momentum = {k: torch.zeros_like(v) for k, v in self.matrices.items()}

    def step(self, gradients: dict) -> None:
        unknown = sorted(set(gradients) - set(self.matrices))
        if unknown:
            raise ValueError(f"no such matrices: {unknown}; expected some of {sorted(self.matrices)}")
        for name, gradient in gradients.items():  # all of them before the first is applied
            m = self.matrices[name]
            if gradient.shape != m.shape or gradient.device != m.device or gradient.dtype not in DTYPES:
                raise ValueError(f"the gradient of {name} must be float32, bfloat16 or float16 {tuple(m.shape)} on "
                                 f"{m.device}, got {gradient.dtype} {tuple(gradient.shape)} on {gradient.device}")
            # (a strided one is copied before its update, but after the others')
            if any(_overlap(_span(gradient), t) for t in (*self.matrices.values(), *self.momentum.values())):
                raise ValueError(f"the gradient of {name} overlaps a matrix or a momentum, which the step changes")
        for name, gradient in gradients.items():
            muon_update(self.matrices[name], gradient, self.momentum[name], **self.settings)

    def params(self) -> AZDirichletParams:
        host = {k: v.cpu().numpy() for k, v in self.matrices.items()}
        device = self.matrices["convs"].device
        if device.type == "cuda":
            check_waits(device)  # after the copies, which waited for the steps
        blocks = [dict(blk) for blk in self._params.blocks]
        for i, blk in enumerate(blocks):
            for j, k in enumerate(("conv1_w", "conv2_w")):
                blk[k] = host["convs"][2 * i + j].reshape(blk[k].shape)
        return dataclasses.replace(self._params, blocks=blocks, **{name: host[name] for name in DENSE})
