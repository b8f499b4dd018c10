"""The orthogonalised update and Muon's step against the definition in 64
bits.

Tolerances.  A product of operands held as fp16 pairs (22 bits) carries,
per entry, at most

    d = (3 * 2^-22 + (3 K / 16 + 1) 2^-23) (|A| |B|)_ij

three halves' rounding of the operands (hi + lo of each, and the lo lo term
that is left out), and one fp32 rounding per MMA that is added (three per 16
of K) and one at the end.  What such errors become after the steps depends
on the matrix, so the tests follow them: the 64-bit iteration is run with
every product disturbed by d with random signs, and the kernel has to be
within twice what the worst of three such runs moves the result by (in the
Frobenius norm), plus the rounding to the output's type.
"""

import math

import pytest
import torch

from scacchi_b200 import _lib
from scacchi_b200.muon import COEFFICIENTS, muon_update, orthogonalize

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _exact(u, steps=5, coefficients=COEFFICIENTS, eps=1e-8, gen=None):
    """The iteration in 64 bits; with `gen`, every product disturbed."""
    a, b, c = coefficients
    u = u.double()
    tall = u.shape[-2] > u.shape[-1]
    x = u.mT if tall else u
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + eps)

    def mul(p, q):
        r = p @ q
        if gen is not None:
            d = 3 * 2.0 ** -22 + (3 * math.ceil(p.shape[-1] / 16) + 1) * 2.0 ** -23
            sign = torch.randint(0, 2, r.shape, generator=gen, device=r.device, dtype=torch.int8).double() * 2 - 1
            r = r + d * sign * (p.abs() @ q.abs())
        return r

    eye = torch.eye(x.shape[-2], dtype=x.dtype, device=x.device)
    for _ in range(steps):
        gram = mul(x, x.mT)
        x = mul(a * eye + b * gram + c * mul(gram, gram), x)
    return x.mT if tall else x


def _bound(u, want, **kw):
    """Per matrix: how far the kernel's result may be, in the Frobenius norm."""
    g = torch.Generator(device=u.device).manual_seed(5)
    norm = lambda t: torch.linalg.vector_norm(t, dim=(-2, -1))
    moved = torch.stack([norm(_exact(u, gen=g, **kw) - want) for _ in range(3)]).amax(0)
    eps = torch.finfo(u.dtype).eps / 2
    return 2 * moved + eps * norm(want) + 1e-30


def _matrix(shape, dtype, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * shape[-1] + shape[-2])
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    *lead, m, n = shape
    if kind == "normal":
        x = rnd(*shape)
    elif kind == "low_rank":
        r = max(1, min(m, n) // 8)
        x = rnd(*lead, m, r) @ rnd(*lead, r, n) + 0.05 * rnd(*shape)
    elif kind == "rank_one":
        x = rnd(*lead, m, 1) * rnd(*lead, 1, n)
    return x.to(DT[dtype])


def _check(u, **kw):
    got = orthogonalize(u, **kw)
    torch.cuda.synchronize()
    assert got.shape == u.shape and got.dtype == u.dtype
    want = _exact(u, **kw)
    err = torch.linalg.vector_norm(got.double() - want, dim=(-2, -1))
    tol = _bound(u, want, **kw)
    assert torch.isfinite(got).all()
    assert bool((err <= tol).all()), f"off by {err.max():.3g}, bound {tol.min():.3g}, norm {want.norm():.3g}"
    return got


SHAPES = [(1, 1), (1, 9), (9, 1), (2, 3), (5, 64), (16, 16), (63, 65), (82, 162), (162, 82), (81, 128), (128, 82),
          (36, 128), (127, 129), (128, 128), (129, 127), (128, 1152), (1152, 128), (257, 1001), (1001, 257),
          (300, 300), (640, 520), (1, 5000), (4099, 3), (200, 4100), (1024, 1024), (1000, 2050)]


@pytest.mark.parametrize("kind", ["normal", "low_rank"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize_matches_definition(cuda, shape, kind):
    _check(_matrix(shape, "fp32", kind))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(82, 162), (1152, 128), (257, 1001), (520, 640), (3, 4099)], ids=str)
def test_orthogonalize_types(cuda, shape, dtype):
    _check(_matrix(shape, dtype, "normal"))
    _check(_matrix(shape, dtype, "low_rank", seed=1))


@pytest.mark.parametrize("shape", [(12, 1152, 128), (3, 257, 1001), (2, 3, 40, 33), (200, 20, 30), (5, 1, 1),
                                   (40, 130, 128), (2, 600, 500)], ids=str)
def test_orthogonalize_stacks(cuda, shape):
    """Each matrix of a stack is normalised and orthogonalised by itself."""
    x = _matrix(shape, "fp32", "normal", seed=2)
    scale = torch.logspace(-6, 6, x[..., 0, 0].numel(), device="cuda").reshape(*shape[:-2], 1, 1)
    _check(x * scale)


def test_orthogonalize_large(cuda):
    _check(_matrix((2048, 2304), "fp32", "normal", seed=3))
    _check(_matrix((5000, 1100), "bf16", "low_rank", seed=3))


@pytest.mark.parametrize("kw", [dict(steps=1), dict(steps=2), dict(steps=9), dict(coefficients=(1.5, -0.5, 0.0), steps=8),
                                dict(coefficients=(2.0, -1.5, 0.5), steps=6), dict(eps=0.0), dict(eps=10.0)], ids=str)
@pytest.mark.parametrize("shape", [(100, 90), (300, 700)], ids=str)
def test_orthogonalize_parameters(cuda, shape, kw):
    _check(_matrix(shape, "fp32", "normal", seed=4), **kw)


def test_singular_values_come_near_one(cuda):
    x = _matrix((4, 128, 256), "fp32", "normal", seed=5)
    s = torch.linalg.svdvals(orthogonalize(x).double())
    assert float(s.min()) > 0.5 and float(s.max()) < 1.3


@pytest.mark.parametrize("shape", [(2, 90, 70), (2, 300, 260)], ids=str)
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_scale_of_the_update(cuda, shape, scale):
    """Norms whose squares leave fp32, both ways."""
    _check(_matrix(shape, "fp32", "normal", seed=6) * scale, eps=0.0)


@pytest.mark.parametrize("shape", [(3, 90, 70), (3, 300, 260)], ids=str)
def test_zeros_and_what_is_not_finite(cuda, shape):
    x = _matrix(shape, "fp32", "normal", seed=7)
    clean = orthogonalize(x)
    for value in (math.nan, math.inf):
        y = x.clone()
        y[1, 5, 6] = value
        y[2] = 0.0
        out = orthogonalize(y)
        assert torch.equal(out[0], clean[0])
        assert torch.isnan(out[1]).all()
        assert not out[2].any()
    _check(_matrix(shape, "fp32", "rank_one", seed=8))


def test_views_and_streams(cuda):
    """Transposed and sliced inputs, another stream, repeats: the same bits."""
    x = _matrix((3, 200, 150), "fp32", "normal", seed=9)
    want = orthogonalize(x)
    wide = torch.full((3, 210, 160), math.nan, device="cuda")
    wide[:, 5:205, 4:154] = x
    assert torch.equal(orthogonalize(wide[:, 5:205, 4:154]), want)
    assert torch.equal(orthogonalize(x.mT.contiguous().mT), want)
    odd = torch.empty(x.numel() + 1, device="cuda")[1:].view(x.shape)  # 4-byte aligned alone
    odd.copy_(x)
    assert torch.equal(orthogonalize(odd), want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            other = orthogonalize(x)
    side.synchronize()
    assert torch.equal(other, want)


def test_empty_stacks(cuda):
    assert orthogonalize(torch.zeros((0, 4, 5), device="cuda")).shape == (0, 4, 5)
    z = torch.zeros((0, 4, 5), device="cuda")
    muon_update(z, z.clone(), z.clone(), learning_rate=0.1)


def _muon64(w, g, m, lr, beta, nesterov, decay, scale, **kw):
    g, m, w = g.double(), m.double(), w.double()
    m = beta * m + (1 - beta) * g
    u = (1 - beta) * g + beta * m if nesterov else m
    return (1 - lr * decay) * w - lr * scale * _exact(u, **kw), m, u


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(12, 1152, 128), (162, 82), (81, 128), (128, 164), (36, 128), (3, 257, 301),
                                   (700, 1300)], ids=str)
def test_muon_matches_definition(cuda, shape, dtype, nesterov):
    w, m = _matrix(shape, "fp32", "normal", seed=10), _matrix(shape, "fp32", "normal", seed=11)
    for t in range(2):
        g = _matrix(shape, dtype, "normal", seed=12 + t)
        lr, decay, beta = 0.03, 0.1, 0.9
        scale = math.sqrt(max(1.0, shape[-1] / shape[-2]))
        want_w, want_m, u = _muon64(w, g, m, lr, beta, nesterov, decay, scale)
        # the momentum: two fp32 products and their sum; the direction one
        # more of each, which moves the result as any relative 2^-22 of it
        m_tol = 3 * 2.0 ** -24 * (m.double().abs() * beta + g.double().abs() * (1 - beta))
        o_tol = _bound(u.float(), _exact(u)) + 2.0 ** -20 * torch.linalg.vector_norm(_exact(u), dim=(-2, -1))
        muon_update(w, g, m, learning_rate=lr, beta=beta, nesterov=nesterov, weight_decay=decay)
        torch.cuda.synchronize()
        assert bool(((m.double() - want_m).abs() <= m_tol + 1e-30).all())
        err = torch.linalg.vector_norm(w.double() - want_w, dim=(-2, -1))
        tol = lr * scale * o_tol + 3 * 2.0 ** -24 * torch.linalg.vector_norm(want_w, dim=(-2, -1))
        assert bool((err <= tol).all()), (err / tol).max()


def test_muon_graph_and_concurrent_calls(cuda):
    """Two captured steps replayed at once on two streams end where eager
    steps do."""
    start, graphs, held = [], [], []
    for shape, seed in (((12, 1152, 128), 20), ((2, 300, 500), 30)):
        start.append([_matrix(shape, "fp32", "normal", seed=seed + k) for k in range(3)])
    eager = []
    for w, g, m in start:
        w, m = w.clone(), m.clone()
        for _ in range(6):
            muon_update(w, g, m, learning_rate=0.02)
        eager.append((w, m))
    for w, g, m in start:
        w, m = w.clone(), m.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            muon_update(w, g, m, learning_rate=0.02)
        graphs.append(graph)
        held.append((w, m))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(6):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for (a, b), (c, d) in zip(eager, held):
        assert torch.equal(a, c) and torch.equal(b, d)
    assert _lib.muon_error() == 0


def test_step_marks_the_weight_changed(cuda):
    w = torch.randn((20, 30), device="cuda", requires_grad=True)
    loss = (w * w).sum()
    muon_update(w, torch.randn_like(w), torch.zeros((20, 30), device="cuda"), learning_rate=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals(cuda):
    x = torch.randn((8, 12), device="cuda")
    before = _lib.launch_count()
    for bad in (x.double(), x[0], x.int(), torch.empty((0, 5), device="cuda"), torch.empty((3, 131073), device="cuda")):
        with pytest.raises(ValueError):
            orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=65), dict(coefficients=(math.nan, 1.0, 1.0)), dict(eps=-1.0),
               dict(eps=math.inf), dict(coefficients=(30.0, -1.0, 0.5))):
        with pytest.raises(ValueError):
            orthogonalize(x, **kw)
    good = dict(weight=x.clone(), gradient=x, momentum=torch.zeros_like(x), learning_rate=0.1)
    for kw in (dict(weight=x.clone().bfloat16()), dict(momentum=torch.zeros((12, 8), device="cuda").T),
               dict(momentum=torch.zeros((8, 11), device="cuda")), dict(weight=x.cpu()), dict(weight=x),
               dict(momentum=good["weight"]), dict(beta=1.0), dict(beta=-0.1), dict(learning_rate=math.nan),
               dict(scale=math.inf), dict(gradient=x.double())):
        with pytest.raises(ValueError):
            muon_update(**{**good, **kw})
    assert _lib.launch_count() == before


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(2, 264, 304), (2, 160, 301), (3, 129, 131), (2, 72, 96)], ids=str)
def test_muon_at_any_alignment(cuda, shape, dtype):
    """Tensors that start on their element alone give the bits of aligned ones."""
    def odd(t):
        at = torch.full((t.numel() + 2,), 7.0, dtype=t.dtype, device="cuda")
        at[1:-1].view(t.shape).copy_(t)
        return at

    w, m = _matrix(shape, "fp32", "normal", seed=21), _matrix(shape, "fp32", "normal", seed=22)
    g = _matrix(shape, dtype, "normal", seed=23)
    w2, m2, g2 = odd(w), odd(m), odd(g)
    view = lambda t: t[1:-1].view(shape)
    muon_update(w, g, m, learning_rate=0.05, weight_decay=0.1)
    muon_update(view(w2), view(g2), view(m2), learning_rate=0.05, weight_decay=0.1)
    assert torch.equal(view(w2), w) and torch.equal(view(m2), m)
    for t in (w2, m2, g2):  # and nothing beside them is written
        assert float(t[0]) == 7.0 and float(t[-1]) == 7.0


def test_a_wait_that_ran_out_is_reported(cuda, monkeypatch):
    """The flag of the device in question, once the steps are complete."""
    from scacchi_b200 import muon
    from scacchi_b200.network import init_params

    opt = muon.NetworkMuon(init_params(5, num_blocks=1), learning_rate=0.1)
    opt.step({k: torch.ones_like(v) for k, v in opt.matrices.items()})
    opt.params()
    muon.check_waits()
    asked = []
    monkeypatch.setattr(_lib, "muon_error", lambda: asked.append(torch.cuda.current_device()) or 1)
    for report in (opt.params, muon.check_waits, lambda: muon.check_waits("cuda:0")):
        with pytest.raises(_lib.ScacchiError, match="wait"):
            report()
    assert asked == [0, 0, 0]
