"""The orthogonalised update and Muon's step refuse what they cannot
compute, before any launch, and choose the operands' scale (no GPU needed)."""

import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from scacchi_b200 import _lib
from scacchi_b200.muon import COEFFICIENTS, MAX_SIDE, NetworkMuon, muon_update, orthogonalize
from scacchi_b200.network import init_params

A = 1 << 20  # a made-up aligned address: a refused call reads none


def _params(**kw):
    d = dict(batch=1, rows=8, cols=8, dtype=0, steps=5, scale_exponent=14, a=3.4445, b=-4.775, c=2.0315, eps=1e-8)
    d.update(kw)
    return _lib.NewtonSchulz(**d)


BAD = [dict(batch=-1), dict(batch=65536), dict(rows=0), dict(cols=0), dict(rows=MAX_SIDE + 1),
       dict(cols=MAX_SIDE + 1), dict(dtype=3), dict(dtype=-1), dict(steps=0), dict(steps=65),
       dict(scale_exponent=-1), dict(scale_exponent=16), dict(a=float("nan")), dict(b=float("inf")),
       dict(c=float("nan")), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf"))]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_library_rejects_bad_parameters(kw):
    lib, p = _lib.lib(), _params(**kw)
    before = lib.scacchi_muon_launch_count()
    assert lib.scacchi_orthogonalize(C.byref(p), A, A, A, None) == _lib.EINVAL
    assert lib.scacchi_muon_update(C.byref(p), A, A, A, 0.9, 1, 1.0, 0.1, A, None) == _lib.EINVAL
    assert lib.scacchi_muon_launch_count() == before


def test_library_rejects_bad_pointers():
    lib, p, half = _lib.lib(), _params(), _params(dtype=1)
    for args in ((None, A, A), (A, None, A), (A, A, None), (A + 2, A, A), (A, A + 1, A), (A, A, A + 128)):
        assert lib.scacchi_orthogonalize(C.byref(p), *args, None) == _lib.EINVAL
    assert lib.scacchi_orthogonalize(C.byref(half), A + 1, A, A, None) == _lib.EINVAL
    assert lib.scacchi_orthogonalize(None, A, A, A, None) == _lib.EINVAL
    for args in ((None, A, A), (A, None, A), (A, A, None), (A, A + 2, A), (A, A, A + 2)):
        assert lib.scacchi_muon_update(C.byref(p), *args, 0.9, 1, 1.0, 0.1, A, None) == _lib.EINVAL
    for beta, decay, step in ((1.0, 1.0, 0.1), (-0.1, 1.0, 0.1), (float("nan"), 1.0, 0.1),
                              (0.9, float("nan"), 0.1), (0.9, 1.0, float("inf"))):
        assert lib.scacchi_muon_update(C.byref(p), A, A, A, beta, 1, decay, step, A, None) == _lib.EINVAL
    assert lib.scacchi_muon_update(C.byref(p), A, A, A, 0.9, 1, 1.0, 0.1, None, None) == _lib.EINVAL


def test_python_rejects_cpu_tensors():
    x = torch.zeros((4, 4))
    with pytest.raises(ValueError, match="CUDA"):
        orthogonalize(x)
    with pytest.raises(ValueError, match="CUDA"):
        muon_update(x, x.clone(), x.clone(), learning_rate=0.1)


def test_scale_keeps_operands_in_half_precision():
    """Largest operand of every step, followed on a finer grid of singular
    values, stays within fp16 at the scale; a doubled scale would not do or
    is fp16's own exponent limit."""
    f = _lib.lib().scacchi_muon_scale_exponent
    for coefficients, steps in ((COEFFICIENTS, 5), (COEFFICIENTS, 64), ((1.5, -0.5, 0.0), 12), ((2.0, -1.5, 0.5), 9)):
        e = f(*coefficients, steps)
        a, b, c = coefficients
        s = torch.linspace(0, 1, 100003, dtype=torch.float64)
        most = 1.0
        for _ in range(steps):
            p = a + b * s ** 2 + c * s ** 4
            most = max(most, float(s.abs().max()), float((s ** 2).max()), float(p.abs().max()))
            s = s * p
        assert 6 <= e <= 15 and most * 2 ** e < 65504
        assert e == 15 or 1.11 * most * 2 ** (e + 1) > 65504
    assert f(30.0, -1.5, 0.5, 5) == -1 and f(3.4445, -4.775, 2.0315, 0) == -1 and f(float("nan"), 0, 0, 5) == -1


def test_workspace_size():
    f = _lib.lib().scacchi_muon_workspace_bytes
    assert f(0, 4, 4) == 0 and f(1, 0, 4) == 0
    # two copies of the stack and two of its narrow square as fp16 pairs
    assert f(12, 1152, 128) >= 12 * (2 * 1152 * 128 + 2 * 128 * 128) * 4
    assert f(1, 3, 5) % 256 == 0
    assert f(2, 65536, 65536) > 2 ** 36


def test_network_muon_refuses_a_step_as_a_whole():
    """One bad gradient, and no matrix has moved."""
    opt = NetworkMuon(init_params(4, num_blocks=1), learning_rate=0.1, device="cpu")
    before = {k: v.clone() for k, v in opt.matrices.items()}
    good = {k: torch.ones_like(v) for k, v in opt.matrices.items()}
    for bad in (torch.ones((3, 3)), torch.ones_like(good["value_w"], dtype=torch.int32),
                torch.ones_like(good["value_w"]).double()):
        with pytest.raises(ValueError, match="gradient of value_w"):
            opt.step({**good, "value_w": bad})
    with pytest.raises(ValueError, match="no such matrices"):
        opt.step({**good, "stem_w": torch.ones((3, 3))})
    assert all(torch.equal(v, before[k]) for k, v in opt.matrices.items())


def _kernel(name):
    source = (Path(__file__).parents[1] / "scacchi_b200" / "csrc" / "muon.cu").read_text()
    kernel = source[source.index(name + "(const __grid_constant__"):]
    return kernel[:kernel.index("\n}\n")]


def test_no_wait_goes_unheeded():
    """A bounded wait that ran out leaves a product unfinished, so every
    kernel looks at what its waits return.  Read from the source: no input
    makes a wait run out."""
    for name in ("ns_pair_kernel", "ns_tile_kernel", "ns_narrow_kernel"):
        statements = [text.strip() for text in re.split("[;{}]", _kernel(name))]
        assert any("mbar_wait" in text for text in statements)
        assert not [text for text in statements if text.startswith("mbar_wait")], name


def test_a_narrow_matrix_is_written_whole_or_not_at_all():
    """In the last step the cluster's CTAs meet, and none writes where a wait
    of any of them ran out; an unfinished product is drained before TMEM goes."""
    kernel = _kernel("ns_narrow_kernel")
    update = kernel[kernel.index("// X <- M X"):]
    meet, leave, write = update.find("cluster.sync()"), update.find("if (*abort_flag) break;"), update.index("narrow_out(")
    assert 0 <= meet < leave < write
    assert "map_shared_rank(const_cast<int *>(abort_flag)" in kernel
    assert update.index("mbar_drain(") < update.index("tmem_dealloc(")


def test_products_after_an_unfinished_one_write_no_weights():
    """A call's products are launched in a row, so the last one has to learn
    that an earlier one gave up: a wait that runs out raises the call's flag,
    the first kernel clears it, and nothing is written to the user's matrix
    where it stands."""
    for name in ("ns_pair_kernel", "ns_tile_kernel"):
        kernel = _kernel(name)
        for wait in re.findall(r"mbar_wait\w*\((.*?)\)", kernel):
            assert wait.endswith("q.failed"), (name, wait)
        for at in re.finditer("emit<", kernel):
            assert "may_write(q)" in kernel[kernel.rindex("if (", 0, at.start()):at.start()], name
    source = (Path(__file__).parents[1] / "scacchi_b200" / "csrc" / "muon.cu").read_text()
    norm = source[source.index("ns_norm_kernel(Source"):]
    assert "*failed = 0" in norm[:norm.index("\n}\n")]


def test_network_muon_refuses_gradients_that_the_step_changes():
    """A gradient that lies in a matrix or a momentum, its own or another's,
    would change between the updates: refused before the first of them."""
    opt = NetworkMuon(init_params(4, num_blocks=1), learning_rate=0.1, device="cpu")
    before = {k: v.clone() for k, v in opt.matrices.items()}
    good = {k: torch.ones_like(v) for k, v in opt.matrices.items()}
    square = opt.matrices["convs"].shape[-1]
    strided = opt.matrices["convs"][0, :square].T  # of no matrix's shape but its own
    for name, bad in (("value_w", opt.matrices["value_w"]), ("policy_w", opt.momentum["policy_w"]),
                      ("convs", opt.matrices["convs"].detach())):
        with pytest.raises(ValueError, match=f"gradient of {name} overlaps"):
            opt.step({**good, name: bad})
    opt.matrices["policy_w"], opt.momentum["policy_w"] = torch.zeros((square, square)), torch.zeros((square, square))
    with pytest.raises(ValueError, match="gradient of policy_w overlaps"):
        opt.step({"convs": good["convs"], "policy_w": strided})
    assert all(torch.equal(opt.matrices[k], v) for k, v in before.items() if k != "policy_w")
