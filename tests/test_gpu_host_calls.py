"""The extension module's calls (csrc/host.cpp): what the library refuses is
left to Python, and what fails behind a launch is an error at once."""

import ctypes as C
import math

import pytest
import torch

from scacchi_b200 import _lib
from scacchi_b200.adamw import AdamW, gradient_norm
from scacchi_b200.log_probs import policy_log_probs, policy_log_probs_gradient

pytestmark = pytest.mark.gpu


@pytest.fixture
def failing(cuda, monkeypatch):
    """Replaces an entry point of the library under the extension module by one that returns a status."""
    kept = []

    def replace(name, status):
        calls = []

        def fake(*args):
            calls.append(name)
            return status

        kept.append(C.CFUNCTYPE(C.c_int, *_lib.SIGNATURES[name])(fake))
        _lib.bind_host(_lib.host(), {name: C.cast(kept[-1], C.c_void_p).value})
        return calls

    yield replace
    _lib.bind_host(_lib.host())


def test_a_step_that_failed_is_not_taken_again(failing):
    """A launch may have failed behind the one that counts the step."""
    w = {"a": torch.ones((8,), device="cuda")}
    opt = AdamW(w, learning_rate=0.1)
    calls = failing("scacchi_adamw_step", 2)
    with pytest.raises(_lib.ScacchiError, match="adamw_step"):
        opt.step({"a": torch.ones((8,), device="cuda")})
    assert len(calls) == 1 and opt.steps() == 0 and bool((w["a"] == 1).all())


def test_other_calls_that_failed_are_errors(failing):
    x, k = torch.zeros((3, 5), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    out, one = policy_log_probs(x, k), torch.ones(3, device="cuda")
    opt = AdamW({"a": torch.ones((8,), device="cuda")}, learning_rate=0.1, max_norm=1.0, state_bits=8, key=(1, 2))
    for name, call in (("scacchi_log_probs", lambda: policy_log_probs(x, k)),
                       ("scacchi_log_probs_gradient", lambda: policy_log_probs_gradient(x, k, out, grad_log_prob=one)),
                       ("scacchi_adamw_moments", lambda: opt.moments()),
                       ("scacchi_gradient_norm", lambda: gradient_norm([one])),
                       ("scacchi_gradient_norm", lambda: opt.step({"a": torch.ones((8,), device="cuda")}))):
        calls = failing(name, 2)
        with pytest.raises(_lib.ScacchiError, match=name.removeprefix("scacchi_")):
            call()
        assert len(calls) == 1
    assert opt.steps() == 0


def test_what_the_library_refuses_is_left_to_python(failing):
    calls = failing("scacchi_adamw_step", _lib.EINVAL)
    opt = AdamW({"a": torch.ones((8,), device="cuda")}, learning_rate=0.1)
    opt.step({"a": torch.ones((8,), device="cuda")})
    assert len(calls) == 1 and opt.steps() == 1
