"""AdamW and the gradient norm refuse what they cannot compute, before any
launch (no GPU needed)."""

import ctypes as C
import dataclasses

import numpy as np
import pytest
import torch

from scacchi_b200 import _lib
from scacchi_b200.adamw import TENSOR, AdamW, _network_arrays, gradient_norm
from scacchi_b200.muon import DENSE
from scacchi_b200.network import init_params

A = 1 << 20  # made-up aligned addresses, a MiB apart: a refused call reads none


def _params(**kw):
    d = dict(state_bits=32, stochastic=0, learning_rate=1e-3, beta1=0.9, beta2=0.999, max_norm=1.0, eps=1e-8, key0=1,
             key1=2, moments=512, first=10 * A, second=11 * A, first_exponent=None, second_exponent=None, state=14 * A,
             norm=None, learning_rate_at=None)
    d.update(kw)
    return _lib.AdamWStep(*d.values())


def _table(*rows):
    """(weight, gradient, count, offset, weight_decay, weight_dtype, gradient_dtype) each"""
    return np.array(list(rows) or [(1 * A, 2 * A, 300, 0, 0.0, 0, 0)], TENSOR)


def _step(params=None, table=None, n=None):
    table = _table() if table is None else table
    return _lib.lib().scacchi_adamw_step(C.byref(params or _params()), table.ctypes.data, len(table) if n is None else n,
                                         None)


NAN, INF = float("nan"), float("inf")
BAD = [dict(state_bits=16), dict(state_bits=8), dict(state_bits=8, stochastic=1), dict(beta1=1.0), dict(beta1=-0.1),
       dict(beta1=NAN), dict(beta2=1.0), dict(beta2=NAN), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF),
       dict(learning_rate=NAN), dict(learning_rate=INF), dict(moments=-256), dict(moments=511), dict(moments=256),
       dict(first=None), dict(second=None), dict(first=10 * A + 8), dict(second=11 * A + 4), dict(state=None),
       dict(state=14 * A + 4), dict(norm=15 * A + 2), dict(norm=15 * A, max_norm=0.0), dict(norm=15 * A, max_norm=INF),
       dict(norm=15 * A, max_norm=NAN), dict(learning_rate_at=15 * A + 1), dict(first=1 * A), dict(second=10 * A),
       dict(first=2 * A), dict(state=2 * A), dict(state=10 * A + 64), dict(norm=1 * A), dict(learning_rate_at=11 * A)]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_library_rejects_bad_parameters(kw):
    before = _lib.lib().scacchi_adamw_launch_count()
    assert _step(_params(**kw)) == _lib.EINVAL
    assert _lib.lib().scacchi_adamw_launch_count() == before


ROWS = [(None, 2 * A, 300, 0, 0.0, 0, 0), (A + 2, 2 * A, 300, 0, 0.0, 0, 0), (A + 1, 2 * A, 300, 0, 0.0, 1, 0),
        (A, 2 * A + 2, 300, 0, 0.0, 0, 0), (A, 2 * A + 1, 300, 0, 0.0, 0, 1), (A, 2 * A, -1, 0, 0.0, 0, 0),
        (A, 2 * A, 513, 0, 0.0, 0, 0), (A, 2 * A, 300, 255, 0.0, 0, 0), (A, 2 * A, 300, -256, 0.0, 0, 0),
        (A, 2 * A, 300, 256, 0.0, 0, 0), (A, 2 * A, 300, 0, NAN, 0, 0), (A, 2 * A, 300, 0, 0.0, 2, 0),
        (A, 2 * A, 300, 0, 0.0, -1, 0), (A, 2 * A, 300, 0, 0.0, 0, 3), (A, 2 * A, 300, 0, 0.0, 0, -1),
        (A, A + 1196, 300, 0, 0.0, 0, 0), (A, A - 1196, 300, 0, 0.0, 0, 0), (A, A - 596, 300, 0, 0.0, 0, 1)]


@pytest.mark.parametrize("row", ROWS, ids=str)
def test_library_rejects_bad_tensors(row):
    row = tuple(0 if v is None else v for v in row)
    assert _step(table=_table(row)) == _lib.EINVAL


def test_library_rejects_bad_lists():
    a, b = (A, 2 * A, 200, 0, 0.0, 0, 0), (3 * A, 4 * A, 200, 256, 0.0, 0, 0)
    assert _step(table=_table(b, a)) == _lib.EINVAL  # offsets descend
    assert _step(table=_table(a, (3 * A, 4 * A, 200, 0, 0.0, 0, 0))) == _lib.EINVAL  # moments of two tensors
    assert _step(table=_table(a, (A + 796, 4 * A, 200, 256, 0.0, 0, 0))) == _lib.EINVAL  # weights meet
    assert _step(table=_table(a, (3 * A, A, 200, 256, 0.0, 0, 0))) == _lib.EINVAL  # one's gradient is the other's weight
    assert _step(n=-1) == _lib.EINVAL
    lib = _lib.lib()
    assert lib.scacchi_adamw_step(None, _table().ctypes.data, 1, None) == _lib.EINVAL
    assert lib.scacchi_adamw_step(C.byref(_params()), None, 1, None) == _lib.EINVAL


def test_library_rejects_bad_norms():
    lib = _lib.lib()
    call = lambda t, n=1, norm=5 * A, ws=6 * A: lib.scacchi_gradient_norm(t.ctypes.data, n, norm, ws, None)
    for row in ((0, 0, 300, 0, 0.0, 0, 0), (0, A + 2, 300, 0, 0.0, 0, 0), (0, A + 1, 300, 0, 0.0, 0, 2),
                (0, A, -1, 0, 0.0, 0, 0), (0, A, 300, 0, 0.0, 0, 3), (0, A, 300, 0, 0.0, 0, -1)):
        assert call(_table(row)) == _lib.EINVAL
    good = _table((0, A, 300, 0, 0.0, 0, 0))
    assert call(good, n=-1) == _lib.EINVAL and call(good, norm=None) == _lib.EINVAL
    assert call(good, norm=5 * A + 2) == _lib.EINVAL and call(good, ws=None) == _lib.EINVAL
    assert call(good, ws=6 * A + 4) == _lib.EINVAL
    assert lib.scacchi_gradient_norm(None, 1, 5 * A, 6 * A, None) == _lib.EINVAL
    assert lib.scacchi_gradient_norm_workspace_bytes(-1) == 0
    assert lib.scacchi_gradient_norm_workspace_bytes(0) > 0
    assert lib.scacchi_gradient_norm_workspace_bytes(5000) >= 10 * lib.scacchi_gradient_norm_workspace_bytes(0) // 2


def test_library_rejects_bad_moments():
    call = _lib.lib().scacchi_adamw_moments
    good = [A, 2 * A, 3 * A, 4 * A, 512, 5 * A, 6 * A, None]
    for i, bad in ((0, None), (1, None), (2, None), (3, None), (5, None), (6, None), (0, A + 8), (1, 2 * A + 1),
                   (5, 5 * A + 2), (6, 6 * A + 8), (4, -256), (4, 100)):
        args = list(good)
        args[i] = bad
        assert call(*args) == _lib.EINVAL
    assert call(None, None, None, None, 0, None, None, None) == _lib.OK


def test_python_refuses():
    w = {"w": torch.zeros(4)}
    with pytest.raises(ValueError, match="CUDA"):
        AdamW(w, learning_rate=0.1)
    with pytest.raises(ValueError, match="CUDA"):
        gradient_norm([torch.zeros(4)])
    with pytest.raises(ValueError, match="at least one"):
        gradient_norm([])
    with pytest.raises(ValueError, match="at least one"):
        AdamW({}, learning_rate=0.1)
    for kw, match in ((dict(beta1=1.0), "beta1"), (dict(beta2=-0.5), "beta2"), (dict(eps=-1e-8), "eps"),
                      (dict(eps=NAN), "eps"), (dict(learning_rate=NAN), "learning_rate"), (dict(max_norm=0.0), "max_norm"),
                      (dict(max_norm=INF), "max_norm"), (dict(state_bits=16), "state_bits"), (dict(state_bits=8), "key"),
                      (dict(weight_decay=INF), "weight_decay"), (dict(weight_decay={"v": 0.1}), "weight_decay")):
        with pytest.raises(ValueError, match=match):
            AdamW(w, **{"learning_rate": 0.1, **kw})


def test_struct_sizes():
    assert TENSOR.itemsize == 48
    assert C.sizeof(_lib.AdamWStep) == 120


def test_network_arrays_are_what_muon_leaves():
    params = init_params(0)
    arrays = _network_arrays(params)
    assert len(arrays) == 66 and not set(arrays) & set(DENSE)
    held = sum(v.size for v in arrays.values()) + sum(getattr(params, n).size for n in DENSE)
    held += sum(blk[k].size for blk in params.blocks for k in ("conv1_w", "conv2_w"))

    def size(v):
        if isinstance(v, np.ndarray):
            return v.size
        if dataclasses.is_dataclass(v):
            return v.scale.size + v.bias.size
        if isinstance(v, list):
            return sum(size(x) for blk in v for x in blk.values())
        return 0

    assert held == sum(size(getattr(params, f.name)) for f in dataclasses.fields(params))


def test_a_weight_that_left_its_device_is_refused():
    """``w.data = w.data.cpu()`` (a module moved behind the optimiser's back): its address is no longer the GPU's."""
    launches = _lib.lib().scacchi_adamw_launch_count()
    opt = AdamW.__new__(AdamW)
    opt.device, opt.max_norm = torch.device("cuda", 0), None
    opt._names, opt._tensors = ("a",), (torch.zeros(300),)
    opt._table, opt._params = _table(), _params()
    with pytest.raises(ValueError, match="a has changed its device"):
        opt._step([torch.zeros(300)], None, None)
    assert _lib.lib().scacchi_adamw_launch_count() == launches


def test_library_rejects_norms_of_more_than_the_workspace_holds():
    """A gradient of 2^42 elements fills half of a launch's grid, and listed
    three times two launches: more partial sums than three tensors have room for."""
    launches = _lib.lib().scacchi_adamw_launch_count()
    for n, count in ((3, 1 << 42), (2, (1 << 42) + 1), (1, (1 << 43) + 1), (1, (1 << 63) - 1)):
        table = _table(*[(0, A, count, 0, 0.0, 0, 1)] * n)
        assert _lib.lib().scacchi_gradient_norm(table.ctypes.data, n, 5 * A, 6 * A, None) == _lib.EINVAL
    assert _lib.lib().scacchi_adamw_launch_count() == launches


def test_what_is_no_tensor_is_refused():
    opt = AdamW.__new__(AdamW)
    opt.device, opt.max_norm, opt._names, opt._shapes = torch.device("cuda", 0), 1.0, ("a",), [torch.Size([3])]
    opt._tensors, opt._table, opt._params = (torch.zeros(3),), _table(), _params()
    for bad in (np.zeros(3, np.float32), [0.0, 0.0, 0.0]):
        with pytest.raises(ValueError, match="gradient of a must be a tensor"):
            opt.step({"a": bad})
        with pytest.raises(ValueError, match="must be tensors"):
            gradient_norm([bad])
    with pytest.raises(ValueError, match="norm must be one float32"):
        opt.step({"a": None}, norm=5.0)


def test_a_call_has_a_table_of_its_own(monkeypatch):
    """The library's call lets other threads run: what it reads is not written by another step."""
    opt = AdamW.__new__(AdamW)
    opt.device, opt.max_norm, opt._names, opt._tensors = torch.device("cpu"), None, ("a",), (torch.zeros(300),)
    opt._table, opt._params = _table((0, 0, 300, 0, 0.0, 0, 0)), _params()
    before, seen = opt._table.copy(), []

    class Library:
        @staticmethod
        def scacchi_adamw_step(params, table, count, stream):
            seen.append(table)
            return _lib.EINVAL

    monkeypatch.setattr(_lib, "lib", lambda: Library)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    with pytest.raises(ValueError, match="overlaps"):
        opt._step([torch.zeros(300)], None, None)
    assert seen[0] != opt._table.ctypes.data and np.array_equal(opt._table, before)
