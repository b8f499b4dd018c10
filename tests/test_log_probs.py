"""Log-probabilities and their gradient refuse what they cannot compute,
before any launch (no GPU needed)."""

import ctypes as C

import pytest
import torch

from scacchi_b200 import _lib
from scacchi_b200.log_probs import LogProbs, policy_log_probs, policy_log_probs_gradient

A = 1 << 20  # a made-up aligned address: a refused call reads none


def _rows(**kw):
    d = dict(logits=A, legal=None, action=A, stride=8)
    d.update(kw)
    return _lib.LogProbRows(*d.values())


def _out(**kw):
    d = dict(log_prob=A, entropy=A, max_logit=A, log_sum=A, top_log_prob=A, top_action=A)
    d.update(kw)
    return _lib.LogProbOut(*d.values())


def _forward(rows=None, out=None, n=4, actions=8, dtype=0, temperature=1.0, top=0):
    return _lib.lib().scacchi_log_probs(rows or _rows(), out or _out(), n, actions, dtype, temperature, top, None)


def _backward(rows=None, at=(A, A, A, A, A), n=4, actions=8, dtype=0, temperature=1.0, grad=A):
    return _lib.lib().scacchi_log_probs_gradient(rows or _rows(), *at, n, actions, dtype, temperature, grad, None)


SIZES = [dict(n=-1), dict(actions=0), dict(actions=262145), dict(dtype=3), dict(dtype=-1), dict(temperature=0.0),
         dict(temperature=float("nan")), dict(temperature=9e-4), dict(temperature=1001.0), dict(n=(1 << 31) + 1),
         dict(actions=9)]


@pytest.mark.parametrize("kw", SIZES, ids=str)
def test_library_rejects_bad_sizes(kw):
    before = _lib.lib().scacchi_log_probs_launch_count()
    assert _forward(**kw) == _lib.EINVAL
    assert _backward(**kw) == _lib.EINVAL
    assert _lib.lib().scacchi_log_probs_launch_count() == before


def test_library_rejects_bad_pointers():
    for kw in (dict(logits=None), dict(logits=A + 2), dict(action=None), dict(action=A + 2), dict(stride=7)):
        assert _forward(rows=_rows(**kw)) == _lib.EINVAL
        assert _backward(rows=_rows(**kw)) == _lib.EINVAL
    assert _forward(rows=_rows(logits=A + 1), dtype=1) == _lib.EINVAL
    for name in ("log_prob", "entropy", "max_logit", "log_sum"):
        assert _forward(out=_out(**{name: None})) == _lib.EINVAL
        assert _forward(out=_out(**{name: A + 2})) == _lib.EINVAL
    for name in ("top_log_prob", "top_action"):
        assert _forward(out=_out(**{name: None}), top=1) == _lib.EINVAL
        assert _forward(out=_out(**{name: A + 1}), top=1) == _lib.EINVAL
    assert _forward(top=33) == _lib.EINVAL and _forward(top=-1) == _lib.EINVAL
    assert _lib.lib().scacchi_log_probs(None, _out(), 4, 8, 0, 1.0, 0, None) == _lib.EINVAL
    assert _lib.lib().scacchi_log_probs(_rows(), None, 4, 8, 0, 1.0, 0, None) == _lib.EINVAL
    for at in ((None, A, A, A, A), (A, None, A, A, A), (A, A, None, A, A), (A + 1, A, A, A, A), (A, A + 2, A, A, A),
               (A, A, A + 2, A, A), (A, A, A, A + 1, A), (A, A, A, A, A + 3)):
        assert _backward(at=at) == _lib.EINVAL
    assert _backward(grad=None) == _lib.EINVAL and _backward(grad=A + 2) == _lib.EINVAL
    assert _backward(grad=A + 1, dtype=2) == _lib.EINVAL


def test_no_rows_are_no_work():
    before = _lib.lib().scacchi_log_probs_launch_count()
    empty = _rows(logits=None, action=None)
    assert _forward(rows=empty, n=0) == _lib.OK and _backward(rows=empty, n=0) == _lib.OK
    assert _lib.lib().scacchi_log_probs_launch_count() == before


def test_python_rejects_cpu_tensors():
    x, k = torch.zeros((3, 5)), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        policy_log_probs(x, k)
    with pytest.raises(ValueError, match="CUDA"):
        policy_log_probs_gradient(x, k, LogProbs(*[torch.zeros(3)] * 4), grad_log_prob=torch.zeros(3))


def test_struct_sizes():
    assert C.sizeof(_lib.LogProbRows) == 32 and C.sizeof(_lib.LogProbOut) == 48


def test_limits_are_the_library_s():
    import os
    import re

    from scacchi_b200 import _build
    from scacchi_b200.log_probs import MAX_ACTIONS, MAX_TOP

    header = open(os.path.join(_build.ROOT, "include", "scacchi_b200.h")).read()
    for name, value in (("SCACCHI_MAX_ACTIONS", MAX_ACTIONS), ("SCACCHI_MAX_TOP", MAX_TOP)):
        assert re.findall(rf"#define {name} (\d+)", header) == [str(value)]
    assert _forward(rows=_rows(stride=MAX_ACTIONS + 1), actions=MAX_ACTIONS + 1) == _lib.EINVAL
    assert _forward(top=MAX_TOP + 1) == _lib.EINVAL
