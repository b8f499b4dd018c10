"""The extension module's calls (csrc/host.cpp): what the library refuses is
left to Python, and what fails behind a launch is an error at once."""

import ctypes as C
import math
import threading

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


def _calls():
    """(host function, arguments that it must decline, the public call, which refuses them) each."""
    x, k = torch.zeros((3, 5), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    out, one = policy_log_probs(x, k), torch.ones(3, device="cuda")
    legal = torch.ones((3, 5), dtype=torch.bool, device="cuda")
    rows = [dict(logits=x.double()), dict(logits=x.cpu()), dict(logits=x[:, :0]), dict(logits=x[0, 0], action=k[0]),
            dict(action=k[:2]), dict(action=k.float()), dict(action=k.cpu()), dict(legal=legal[:, :4]), dict(legal=x),
            dict(legal=legal.cpu()), dict(temperature=0.0), dict(temperature=math.nan), dict(temperature=2e3),
            dict(logits=torch.zeros((1, 262145), device="cuda"), action=k[:1]), dict(logits=None), dict(action=None)]
    for bad in rows:
        kw = dict(dict(logits=x, action=k, legal=None, temperature=1.0), **bad)
        args = tuple(kw.values())
        yield "log_probs", (*args, 2), lambda kw=kw: policy_log_probs(**kw)
        yield ("log_probs_gradient", (*args, out.max_logit, out.log_sum, out.entropy, one, one),
               lambda kw=kw: policy_log_probs_gradient(out=out, grad_log_prob=one, grad_entropy=one, **kw))
    for top in (-1, 33, 1 << 80):
        yield "log_probs", (x, k, None, 1.0, top), lambda top=top: policy_log_probs(x, k, top=top)
    yield ("log_probs_gradient", (x, k, None, 1.0, *out[2:4], out.entropy, None, None),
           lambda: policy_log_probs_gradient(x, k, out))
    for bad in (one[:2], one.cpu(), one.int(), one.view(3, 1)):
        yield ("log_probs_gradient", (x, k, None, 1.0, *out[2:4], out.entropy, bad, None),
               lambda bad=bad: policy_log_probs_gradient(x, k, out, grad_log_prob=bad))
        yield ("log_probs_gradient", (x, k, None, 1.0, bad, out.log_sum, out.entropy, one, None),
               lambda bad=bad: policy_log_probs_gradient(x, k, out._replace(max_logit=bad), grad_log_prob=one))
    for bad in ([], [x, x.cpu()], [x.double()], [x, x.int()], [None], [1.0]):
        yield "gradient_norm", bad, lambda bad=bad: gradient_norm(bad)


def test_what_python_refuses_the_extension_declines(cuda):
    """Every check of arguments stands twice; none of these calls is taken by either."""
    launches = _lib.launch_count()
    made = 0
    for name, args, call in list(_calls()):
        fn = getattr(_lib.host(), name)
        before = _lib.launch_count()
        assert (fn(args) if name == "gradient_norm" else fn(*args)) is None, (name, args)
        with pytest.raises((ValueError, AttributeError, TypeError)):
            call()
        assert _lib.launch_count() == before
        made += 1
    assert made > 45 and _lib.launch_count() - launches < 10


def test_steps_that_python_refuses_the_extension_declines(cuda):
    w = torch.zeros((10, 10), device="cuda")
    good = torch.ones((10, 10), device="cuda")
    opt, clipped = AdamW({"a": w}, learning_rate=0.1), AdamW({"a": w}, learning_rate=0.1, max_norm=1.0)
    one = torch.ones((), device="cuda")

    def step(o, grads, norm=None, rate=None):
        return (o._names, o._tensors, grads, o._table.ctypes.data, C.addressof(o._params), o.device.index, o.max_norm,
                norm, rate)

    bad = [(opt, dict(grads={"a": g})) for g in (good[:9], good.double(), good.cpu(), good.view(100), 1.0, w)]
    bad += [(opt, dict(grads=g)) for g in ({"b": good}, {"a": good, "b": good})]
    bad += [(opt, dict(grads={"a": good}, norm=one))]
    rates = (math.nan, math.inf, one.cpu(), one.double(), good, w[0, 0])
    bad += [(opt, dict(grads={"a": good}, rate=r)) for r in rates]
    bad += [(clipped, dict(grads={"a": good}, norm=n)) for n in (one.cpu(), one.double(), good, 1.0)]
    for o, kw in bad:
        before = _lib.launch_count()
        assert _lib.host().adamw_step(*step(o, **kw)) is None, kw
        assert o is clipped or _lib.launch_count() == before
        with pytest.raises(ValueError):
            o.step(kw["grads"], norm=kw.get("norm"), learning_rate=kw.get("rate"))
    assert opt.steps() == clipped.steps() == 0 and not bool(w.any())


def test_calls_from_many_threads_at_once(cuda):
    """Each thread on a stream of its own, by the extension module and through Python (strided gradients, an int64
    action), gives what one thread gives."""
    N, A, T = 300, 700, 8
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn((T, N, A), generator=gen, device="cuda")
    action = torch.randint(0, A, (N,), generator=gen, device="cuda", dtype=torch.int32)
    grads = torch.randn((T, 64, 48), generator=gen, device="cuda")

    def work(i, res):
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_event(ready)
            w = {k: torch.ones(s, device="cuda") for k, s in (("a", (64, 48)), ("b", (48, 64)))}
            opt = AdamW(w, learning_rate=0.01, max_norm=1.0, state_bits=8 if i % 2 else 32, key=(3, 4))
            for _ in range(20):
                a = action if i % 3 else action.long()
                out = policy_log_probs(logits[i], a, top=5)
                grad = policy_log_probs_gradient(logits[i], a, out, grad_log_prob=out.entropy)
                opt.step({"a": grads[i], "b": grads[i].t() if i % 4 else grads[i].t().contiguous()})
            norm = gradient_norm([grad, grads[i]])
            torch.cuda.current_stream().synchronize()
            res[i] = [*out, grad, norm, *w.values(), opt.first, opt.second]

    ready = torch.cuda.Event()
    ready.record()
    want, got = {}, {}
    for i in range(T):
        work(i, want)
    threads = [threading.Thread(target=work, args=(i, got)) for i in range(T)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(T):
        assert len(want[i]) == len(got[i])
        for a, b in zip(want[i], got[i]):
            assert torch.equal(a, b)
