"""The clipped policy loss kernel (scacchi_policy_loss) against the plain
definition in 64 bits.

Tolerances, from the kernel's arithmetic (32-bit row sums finished in 64
bits): the row's sum of exponentials has relative error at most E = 3e-6
(2^-24 |x - m| + 2 ulp per term, weighted by p with sum p |x - m| <= 13,
and 32 rounded adds per thread plus the tree), so log_prob is off by at
most E and its rounding to fp32, ratio by E + 2^-22 relative, p by
2 E relative; a difference d = x - r carries 2^-24 of its size, as does
mean(d).  The gradient then rounds once more to its own type, by at most
eps / 2 of it (and half the smallest subnormal).
"""

import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from scacchi_b200 import _lib
from scacchi_b200.policy_loss import clipped_policy_loss

pytestmark = pytest.mark.gpu

E = 3e-6
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _inputs(N, A, dtype, legal, kl, seed=0, spread=2.0, ref_spread=0.3):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + 7 * A + N)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    logits = (spread * rnd(N, A)).to(DT[dtype])
    mask = None
    if legal:
        mask = torch.rand((N, A), generator=g, device="cuda") < 0.7
        mask[:, 0] |= ~mask.any(-1)
    prob = torch.ones((N, A), device="cuda") if mask is None else mask.float()
    action = torch.multinomial(prob, 1, generator=g)[:, 0].to(torch.int32) if A < 1 << 24 else None
    x = logits.double()
    if mask is not None:
        x = x.masked_fill(~mask, -math.inf)
    lp = torch.log_softmax(x, -1).gather(-1, action.long()[:, None])[:, 0]
    kw = dict(old_log_prob=(lp + 0.3 * rnd(N)).float(), advantage=rnd(N), legal=mask,
              weight=torch.rand(N, generator=g, device="cuda") / N)
    if kl == "full":
        kw["reference_logits"] = (logits.float() + ref_spread * rnd(N, A)).to(DT[dtype])
    if kl == "sampled":
        kw["reference_log_prob"] = (lp + 0.2 * rnd(N)).float()
    return logits, action, kw


def _plain(logits, action, old_log_prob, advantage, legal=None, weight=None, reference_logits=None,
           reference_log_prob=None, clip_low=0.2, clip_high=0.2, kl_coefficient=0.0):
    """The definition in 64 bits, and what each output may be off by."""
    N, A = logits.shape
    x = logits.double()
    keep = x != -math.inf
    if legal is not None:
        keep = keep & legal.bool()
    x = torch.where(keep, x, -math.inf)
    k = action.long()
    at = k.clamp(0, A - 1)[:, None]
    w = torch.full((N,), 1.0 / N, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    counts = (w != 0) & (k >= 0) & (k < A) & keep.gather(-1, at)[:, 0]
    xs = torch.where(counts[:, None], x, 0.0)
    logp = torch.log_softmax(xs, -1)
    p = torch.where(keep, logp.exp(), 0.0)
    lp = logp.gather(-1, at)[:, 0]
    adv = advantage.double()
    ratio = torch.exp(lp - old_log_prob.double())
    lo, hi = 1 - clip_low, 1 + clip_high
    clipped = torch.where(adv >= 0, ratio > hi, ratio < lo)
    surrogate = -torch.where(adv == 0, 0.0, torch.minimum(ratio * adv, ratio.clamp(lo, hi) * adv))
    c = torch.where(clipped | (adv == 0), 0.0, -adv * ratio)
    c_tol = c.abs() * (2 * E)
    kl = kl_tol = torch.zeros_like(lp)
    d_term = torch.zeros_like(p)
    d_tol = torch.zeros_like(p)
    beta = kl_coefficient
    if reference_log_prob is not None:
        y = reference_log_prob.double() - lp
        kl = torch.expm1(y) - y
        kl_tol = torch.expm1(y).abs() * 2 * E + 16 * U * kl + 1e-30
        c = c - beta * torch.expm1(y)
        c_tol = c_tol + abs(beta) * (torch.exp(y) * 2 * E + 4 * U * torch.expm1(y).abs())
    if reference_logits is not None:
        r = torch.where(keep, reference_logits.double(), -math.inf)
        logq = torch.log_softmax(torch.where(counts[:, None], r, 0.0), -1)
        kl = (p * torch.where(p > 0, logp - logq, 0.0)).sum(-1)
        d = torch.where(keep, x - r, 0.0)
        d = torch.where(counts[:, None], d, 0.0)
        off = d - (p * d).sum(-1, keepdim=True)
        # d and its mean: 2^-24 of themselves and 2 E of the mean absolute d
        d_tol = U * d.abs() + (2 * E + 4 * U) * (p * d.abs()).sum(-1, keepdim=True)
        phi = torch.expm1(-off) + off
        kl_tol = (4 * E * (p * phi).sum(-1) + (p * torch.expm1(-off).abs() * d_tol).sum(-1)
                  + 16 * U * kl.abs() + 1e-30)
        d_term = off
    term = surrogate + beta * kl
    term_tol = ratio * adv.abs() * 2 * E + abs(beta) * kl_tol
    onehot = torch.zeros_like(p).scatter_(-1, at, 1.0)
    grad = w[:, None] * (c[:, None] * (onehot - p) + beta * p * d_term)
    # p is off by 2 E, the product of c and (delta - p) by that and c's own
    g_tol = w[:, None].abs() * ((c.abs() * (2 * E + 8 * U))[:, None] * (onehot + p)
                                + c_tol[:, None] * (onehot + p)
                                + abs(beta) * p * (d_term.abs() * (2 * E + 8 * U) + d_tol))
    grad = torch.where(counts[:, None] & keep, grad, 0.0)
    eps = torch.finfo(logits.dtype).eps / 2
    g_tol = (g_tol * (1 + eps) + grad.abs() * eps + torch.finfo(logits.dtype).smallest_normal
             * torch.finfo(logits.dtype).eps)
    zero = torch.zeros_like(lp)
    loss = torch.where(counts, w * term, zero).sum()
    loss_tol = torch.where(counts, w.abs() * (term_tol + 4 * U * term.abs()), zero).sum() + U * loss.abs() + 1e-30
    sel = lambda v: torch.where(counts, v, zero)
    return dict(loss=(loss, loss_tol), log_prob=(sel(lp), E + U * lp.abs()), kl=(sel(kl), kl_tol + 1e-30),
                grad_logits=(grad, g_tol)), counts & clipped


def _check(logits, action, kw, beta=0.05, gradient=True, **more):
    out = clipped_policy_loss(logits, action, kl_coefficient=beta, gradient=gradient, **kw, **more)
    flat = logits.reshape(-1, logits.shape[-1])
    torch.cuda.synchronize()
    want, clipped = _plain(flat, action.reshape(-1), kl_coefficient=beta, **{
        k: (v if v is None else v.reshape(-1, flat.shape[-1]) if v.dim() == logits.dim() and v.shape == logits.shape
            else v.reshape(-1)) for k, v in kw.items()}, **more)
    assert torch.equal(out.clipped.reshape(-1), clipped)
    for name, (value, tol) in want.items():
        got = getattr(out, name)
        if got is None:
            assert name == "kl" or not gradient
            continue
        err = (got.double().reshape(value.shape) - value).abs()
        over = err - tol
        assert torch.isfinite(err).all(), name
        assert float(over.max()) <= 0, f"{name}: off by {float(err.max()):.3g}, {float((err / tol).max()):.3g} x the bound"
    return out


# each width of vectors and each split of a row over lanes, warps and CTAs
SIZES = [(1, 1), (5, 1), (3, 2), (300, 3), (7, 10), (4000, 10), (65, 31), (64, 82), (1001, 82), (33, 83), (257, 122),
         (9, 127), (9, 129), (40, 362), (5, 512), (5, 513), (1, 1000), (300, 1024), (2, 4097), (70, 4672), (3, 16384),
         (200, 16385), (1, 32000), (160, 32000), (3, 50257), (2, 131071), (1, 131072), (1, 262144)]


@pytest.mark.parametrize("kl", ["none", "sampled", "full"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_matches_plain_form(cuda, size, dtype, kl):
    N, A = size
    legal = (N + A) % 2 == 1
    logits, action, kw = _inputs(N, A, dtype, legal, kl)
    _check(logits, action, kw, beta=0.0 if kl == "none" else 0.07, clip_high=0.28)
    if A in (82, 513, 32000):
        _check(logits, action, dict(kw, legal=None), beta=0.0 if kl == "none" else 0.07, gradient=False)


@pytest.mark.parametrize("kl", ["none", "sampled", "full"])
@pytest.mark.parametrize("A", [6, 82, 700])
def test_rows_that_do_not_count(cuda, A, kl):
    """Weight 0, actions out of range or illegal, rows without a legal
    action: zeros, whatever their logits hold."""
    N = 40
    logits, action, kw = _inputs(N, A, "fp32", True, kl)
    kw["weight"][:8] = 0.0
    logits[:4] = math.nan
    logits[4] = math.inf
    action[8], action[9], action[10] = -1, A, 2 ** 31 - 1
    kw["legal"][11] = False
    kw["legal"][12, action[12].long()] = False
    logits[13, action[13].long()] = -math.inf
    out = clipped_policy_loss(logits, action, kl_coefficient=0.0 if kl == "none" else 0.1, **kw)
    dead = slice(0, 14)
    for name in ("log_prob", "clipped", "kl", "grad_logits"):
        v = getattr(out, name)
        assert v is None or not v[dead].any(), name
    kw = {k: v if v is None else v[14:] for k, v in kw.items()}
    live = clipped_policy_loss(logits[14:], action[14:], kl_coefficient=0.0 if kl == "none" else 0.1, **kw)
    assert torch.equal(out.grad_logits[14:], live.grad_logits) and torch.equal(out.log_prob[14:], live.log_prob)
    assert abs(float(out.loss) - float(live.loss)) <= 4 * U * abs(float(live.loss))
    _check(logits[14:], action[14:], kw, beta=0.0 if kl == "none" else 0.1)


@pytest.mark.parametrize("fill", ["nan", "inf", "-inf", "lowest", "highest"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("A", [82, 515])
def test_illegal_places_may_hold_anything(cuda, A, dtype, fill):
    value = {"lowest": torch.finfo(DT[dtype]).min, "highest": torch.finfo(DT[dtype]).max}.get(fill)
    value = float(fill) if value is None else value
    logits, action, kw = _inputs(50, A, dtype, True, "full", seed=3)
    clean = clipped_policy_loss(logits, action, kl_coefficient=0.1, **kw)
    dirty_ref = kw["reference_logits"].masked_fill(~kw["legal"], value)
    dirty = clipped_policy_loss(logits.masked_fill(~kw["legal"], value), action, kl_coefficient=0.1,
                                **dict(kw, reference_logits=dirty_ref))
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    assert not clean.grad_logits[~kw["legal"]].any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_masks_written_into_the_logits(cuda, dtype):
    """-inf, or the type's lowest value, in place of a mask."""
    logits, action, kw = _inputs(64, 82, dtype, True, "sampled", seed=4)
    legal = kw.pop("legal")
    for fill in (-math.inf, torch.finfo(DT[dtype]).min):
        out = _check(logits.masked_fill(~legal, fill), action, dict(kw, legal=None))
        assert not out.grad_logits[~legal].any()


@pytest.mark.parametrize("A", [2, 82, 122, 600, 40000])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_either_side_of_a_clip_border(cuda, A, dtype):
    """Old log-probabilities one fp32 step apart around both borders: the
    side is the exact one's."""
    N = 512 if A < 1000 else 40
    logits, action, kw = _inputs(N, A, dtype, False, "none", seed=5)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, action.long()[:, None])[:, 0]
    for adv, border in ((1.0, math.log1p(0.2)), (-1.0, math.log1p(-0.2))):
        old = (lp - border).float()
        steps = torch.arange(N, device="cuda") % 7 - 3
        old = (old.view(torch.int32) + steps.to(torch.int32)).view(torch.float32)
        kw["old_log_prob"], kw["advantage"] = old, torch.full((N,), adv, device="cuda")
        out = _check(logits, action, kw, beta=0.0)
        assert 0 < int(out.clipped.sum()) < N


@pytest.mark.parametrize("A", [82, 2000])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 8.0, 60.0, 300.0])
def test_kl_of_near_and_far_policies(cuda, A, scale):
    logits, action, kw = _inputs(100, A, "fp32", True, "full", seed=6, spread=3.0, ref_spread=scale)
    kw["weight"] = None
    _check(logits, action, kw, beta=0.3)


@pytest.mark.parametrize("spread", [30.0, 1e4])
def test_large_logits(cuda, spread):
    """Rows whose mass is on one action, behaviour far off: finite results."""
    logits, action, kw = _inputs(200, 82, "fp32", True, "none", seed=7)
    logits = logits * spread / 2
    x = logits.double().masked_fill(~kw["legal"], -math.inf)
    kw["old_log_prob"] = torch.log_softmax(x, -1).gather(-1, action.long()[:, None])[:, 0].float()
    out = clipped_policy_loss(logits, action, **kw)
    want, _ = _plain(logits, action, **kw)
    # x - m itself rounds at 2^-24 of its size here: the log-probability is
    # held to that, the rest to being finite
    err = (out.log_prob.double() - want["log_prob"][0]).abs()
    assert float((err - (E + 2 * U * want["log_prob"][0].abs())).max()) <= 0
    assert torch.isfinite(out.loss) and torch.isfinite(out.grad_logits).all()


def test_zero_advantage_and_overflowing_ratio(cuda):
    logits, action, kw = _inputs(30, 82, "fp32", False, "none", seed=8)
    kw["old_log_prob"][:] = -500.0                      # the ratio overflows to infinity in 32 bits
    kw["advantage"][:15], kw["advantage"][15:] = 0.0, 2.0
    out = clipped_policy_loss(logits, action, **kw)
    assert not out.grad_logits.any() and bool(out.clipped.all())
    assert math.isclose(float(out.loss), float(-(kw["weight"][15:].double() * 2.0 * 1.2).sum()), rel_tol=1e-6)


def test_strided_rows_and_leading_shape(cuda):
    """A slice of a padded vocabulary, a transposed batch, an expanded row."""
    B, T, A = 6, 5, 82
    logits, action, kw = _inputs(B * T, A, "bf16", True, "full", seed=9)
    base = clipped_policy_loss(logits, action, kl_coefficient=0.1, **kw)
    for pad in (2, 5):
        wide = torch.full((B * T, A + pad), math.nan, dtype=torch.bfloat16, device="cuda")
        wide[:, :A] = logits
        ref = torch.full((B * T, A + 3 * pad), math.nan, dtype=torch.bfloat16, device="cuda")
        ref[:, :A] = kw["reference_logits"]
        got = clipped_policy_loss(wide[:, :A], action, kl_coefficient=0.1, **dict(kw, reference_logits=ref[:, :A]))
        for a, b in zip(base, got):
            assert torch.allclose(a.double(), b.double(), rtol=2e-5, atol=1e-6)
    shaped = {k: v if v is None else v.reshape(B, T, *v.shape[1:]).transpose(0, 1) for k, v in kw.items()}
    got = clipped_policy_loss(logits.reshape(B, T, A).transpose(0, 1), action.reshape(B, T).T, kl_coefficient=0.1,
                              **shaped)
    assert got.grad_logits.shape == (T, B, A) and got.log_prob.shape == (T, B)
    assert torch.equal(got.grad_logits.transpose(0, 1).reshape(B * T, A), base.grad_logits)
    assert torch.equal(got.clipped.T.reshape(-1), base.clipped)
    one = clipped_policy_loss(logits[:1].expand(4, A), action[:1].expand(4), kw["old_log_prob"][:1].expand(4),
                              kw["advantage"][:1].expand(4))
    assert torch.equal(one.grad_logits[0], one.grad_logits[3])
    scalar = clipped_policy_loss(logits[0], action[0].long(), kw["old_log_prob"][0], kw["advantage"][0])
    assert scalar.log_prob.shape == () and torch.equal(scalar.grad_logits, one.grad_logits[0] * 4)


def _moved(t, offset, pad):
    """`t` as rows `pad` elements further apart, from an odd place of a buffer of NaN (of ones, for a mask)."""
    N, A = t.shape
    fill = 1 if t.dtype == torch.bool else math.nan
    buf = torch.full((offset + N * (A + pad) + 64,), fill, dtype=t.dtype, device="cuda")
    view = buf[offset:offset + N * (A + pad)].view(N, A + pad)[:, :A]
    view.copy_(t)
    return view


@pytest.mark.parametrize("kl", ["none", "full"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("size", [(37, 82), (37, 81), (21, 600), (21, 601), (5, 20003), (2, 70001)], ids=str)
def test_rows_at_any_alignment(cuda, size, dtype, kl):
    """Bases and strides off every vector's alignment, together and each by
    itself, with masks likewise."""
    logits, action, kw = _inputs(*size, dtype, True, kl, seed=15)
    for x_at, r_at, m_at in (((1, 0), (1, 0), (1, 0)), ((0, 3), (0, 3), (0, 0)), ((3, 1), (2, 5), (7, 0)),
                             ((0, 0), (1, 0), (0, 0)), ((2, 8), (2, 8), (2, 0)), ((5, 0), (5, 0), (3, 0))):
        moved = dict(kw, legal=_moved(kw["legal"], *m_at))
        if kl == "full":
            moved["reference_logits"] = _moved(kw["reference_logits"], *r_at)
        _check(_moved(logits, *x_at), action, moved, beta=0.0 if kl == "none" else 0.1)


@pytest.mark.parametrize("A", [82, 3000])
def test_a_nan_stays_in_its_row(cuda, A):
    logits, action, kw = _inputs(12, A, "fp32", False, "full", seed=16)
    clean = clipped_policy_loss(logits, action, kl_coefficient=0.1, **kw)
    logits[5, (int(action[5]) + 1) % A] = math.nan
    out = clipped_policy_loss(logits, action, kl_coefficient=0.1, **kw)
    others = torch.arange(12, device="cuda") != 5
    assert math.isnan(float(out.loss)) and bool(torch.isnan(out.log_prob[5])) and bool(torch.isnan(out.grad_logits[5]).any())
    for name in ("log_prob", "kl", "grad_logits", "clipped"):
        assert torch.equal(getattr(out, name)[others], getattr(clean, name)[others]), name


def test_first_call_under_capture(cuda):
    """A process whose first calls are captured, not run."""
    code = """
import torch
from scacchi_b200.policy_loss import clipped_policy_loss
from scacchi_b200.muon import orthogonalize
g = torch.Generator(device="cuda").manual_seed(0)
x = [torch.randn(s, generator=g, device="cuda") for s in ((40, 82), (3, 5000), (90, 70), (300, 400))]
z = torch.zeros(40, device="cuda")
k = z.int()
torch.cuda.synchronize()
def work():
    a = clipped_policy_loss(x[0], k, z, z + 1)
    b = clipped_policy_loss(x[1], k[:3], z[:3], z[:3] + 1)
    return [a.grad_logits, b.grad_logits, orthogonalize(x[2]), orthogonalize(x[3])]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = work()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(held, work()):
    assert torch.equal(a, b) and bool(a.any())
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


def test_rows_past_32_bits(cuda):
    """Rows whose offset passes 2^31 elements."""
    N, stride, A = 70000, 32768, 82
    wide = torch.empty((N, stride), dtype=torch.bfloat16, device="cuda")
    logits, action, kw = _inputs(N, A, "bf16", False, "none", seed=10)
    wide[:, :A] = logits
    got = clipped_policy_loss(wide[:, :A], action, **kw)
    want = clipped_policy_loss(logits, action, **kw)
    for a, b in zip(got, want):
        assert a is b is None or torch.equal(a, b)


def test_no_rows(cuda):
    z = torch.zeros(0, device="cuda")
    out = clipped_policy_loss(torch.zeros((0, 82), device="cuda"), z.int(), z, z)
    assert float(out.loss) == 0.0 and out.grad_logits.shape == (0, 82) and out.log_prob.shape == (0,)


@pytest.mark.parametrize("size", [(5000, 82), (3, 40000)], ids=str)
def test_streams_graphs_and_repeats(cuda, size):
    """The same bits on another stream, from a captured graph (two of them,
    replayed at once) and from call to call."""
    a_in, b_in = _inputs(*size, "fp32", True, "full", seed=11), _inputs(*size, "fp32", True, "full", seed=12)
    call = lambda s: clipped_policy_loss(s[0], s[1], kl_coefficient=0.1, **s[2])
    want = [call(a_in), call(b_in)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = call(a_in)
    side.synchronize()
    for x, y in zip(want[0], other):
        assert torch.equal(x, y)
    graphs, outs = [], []
    for s in (a_in, b_in):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(s))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for x, y in zip(w, o):
            assert torch.equal(x, y)


def test_gradient_against_differences(cuda):
    """Central differences of the 64-bit loss at single logits."""
    logits, action, kw = _inputs(12, 20, "fp32", True, "full", seed=13)
    out = clipped_policy_loss(logits, action, kl_coefficient=0.2, **kw)
    rng = np.random.default_rng(0)
    h = 1e-5
    for i, a in zip(rng.integers(0, 12, 60), rng.integers(0, 20, 60)):
        x = logits.double()
        up, down = x.clone(), x.clone()
        up[i, a] += h
        down[i, a] -= h
        diff = (float(_loss64(up, action, kw)) - float(_loss64(down, action, kw))) / (2 * h)
        # the difference's own error: h^2 / 6 times a third derivative of at
        # most a few times the row's share, and 1e-16 / h of the loss
        assert abs(diff - float(out.grad_logits[i, a])) <= 1e-6 * float(kw["weight"][i]) * 12 + 1e-8


def _loss64(x, action, kw):
    want, _ = _plain(x, action, kl_coefficient=0.2, **kw)
    return want["loss"][0]


def test_refusals(cuda):
    x, k, kw = _inputs(4, 10, "fp32", True, "full", seed=14)
    old, adv = kw["old_log_prob"], kw["advantage"]
    bad = [
        dict(logits=x.double()), dict(logits=x.long()), dict(action=k.float()), dict(action=k[:3]),
        dict(action=k.cpu()), dict(old_log_prob=old[:2]), dict(old_log_prob=old.cpu()), dict(advantage=adv.long()),
        dict(weight=adv[None]), dict(legal=x), dict(legal=kw["legal"][:, :5]), dict(legal=kw["legal"].cpu()),
        dict(reference_logits=x.bfloat16()), dict(reference_logits=x[:, :5]),
        dict(reference_logits=x, reference_log_prob=old), dict(clip_low=1.0), dict(clip_low=-0.1),
        dict(clip_low=math.nan), dict(clip_high=math.inf), dict(kl_coefficient=math.nan), dict(kl_coefficient=0.1),
        dict(logits=torch.zeros((4, 0), device="cuda")), dict(logits=torch.zeros((1, 262145), device="cuda")),
    ]
    before = _lib.launch_count()
    for change in bad:
        args = dict(logits=x, action=k, old_log_prob=old, advantage=adv)
        args.update(change)
        with pytest.raises(ValueError):
            clipped_policy_loss(args.pop("logits"), args.pop("action"), args.pop("old_log_prob"),
                                args.pop("advantage"), **args)
    assert _lib.launch_count() == before


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("size", [(64, 82), (1, 5), (33, 511), (7, 520), (3, 70001), (4, 262144)], ids=str)
def test_few_rows_in_64_bits(cuda, size, dtype):
    """Few rows' terms may cancel: their sum is taken before any rounding to
    32 bits.  Exponentials to 1e-11 and 64-bit sums leave 1e-10 of each term;
    the results round once, by 2^-24."""
    for seed in range(4):
        logits, action, kw = _inputs(*size, dtype, size[1] < 1000, "none", seed=40 + seed)
        got = clipped_policy_loss(logits, action, **kw)
        x = logits.double()
        if kw["legal"] is not None:
            x = x.masked_fill(~kw["legal"], -math.inf)
        lp = torch.log_softmax(x, -1).gather(-1, action.long()[:, None])[:, 0]
        ratio, adv = torch.exp(lp - kw["old_log_prob"].double()), kw["advantage"].double()
        term = -torch.minimum(ratio * adv, ratio.clamp(1 - 0.2, 1 + 0.2) * adv) * kw["weight"].double()
        tol = U * abs(float(term.sum())) + 1e-10 * float(term.abs().sum())
        assert abs(float(got.loss) - float(term.sum())) <= tol
        assert bool(((got.log_prob.double() - lp).abs() <= U * lp.abs() + 1e-10).all())


@pytest.mark.parametrize("kl", ["none", "sampled", "full"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("size", [(3, 40000), (9, 131071), (74, 9001), (160, 60001)], ids=str)
def test_clusters_whose_first_rows_do_not_count(cuda, size, dtype, kl):
    """Rows in clusters of 2 to 16 CTAs: the first ones, every other one, or
    all of them without a part in the loss."""
    logits, action, kw = _inputs(*size, dtype, False, kl, seed=60)
    beta = 0.0 if kl == "none" else 0.1
    every = kw["weight"].clone()
    for off in (slice(0, 2), slice(0, None, 2), slice(0, None)):
        kw["weight"] = every.clone()
        kw["weight"][off] = 0.0
        out = _check(logits, action, kw, beta=beta)
        assert not out.grad_logits[off].any() and not out.log_prob[off].any()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("A", [2, 82, 301, 700, 40000])
def test_kl_of_actions_whose_logits_are_equal(cuda, A, masked):
    """Actions of p = e^-100 whose logits are the reference's (d = 0) carry
    the KL where the one of p = 1 has d = 120: log of the others' share of
    the reference, in 64 bits and rounded once."""
    N = 9
    x, r = torch.full((N, A), -100.0, device="cuda"), torch.full((N, A), -100.0, device="cuda")
    x[:, 0], r[:, 0] = 0.0, -120.0
    legal, others = None, A - 1
    if masked:
        legal = torch.ones((N, A), dtype=torch.bool, device="cuda")
        legal[:, 2::3] = False
        others = int(legal[0].sum()) - 1
    z = torch.zeros(N, device="cuda")
    out = clipped_policy_loss(x, z.int(), z, z, legal=legal, reference_logits=r, kl_coefficient=0.25)
    want = math.log1p(others * math.exp(20.0))
    assert float((out.kl.double() - want).abs().max()) <= 2 * U * want
    assert abs(float(out.loss) - 0.25 * want) <= 4 * U * want
    # p = 1 and d = mean there; p = 0 elsewhere
    assert not out.grad_logits.any()


@pytest.mark.parametrize("kl", ["none", "sampled", "full"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("A", [2, 82, 512])
def test_rows_of_the_lowest_value(cuda, A, dtype, kl):
    """A mask that leaves nothing, written as the type's lowest value: the
    uniform policy, the logits being equal."""
    _lowest_rows(A, dtype, kl)


def _lowest_rows(A, dtype, kl):
    logits, action, kw = _inputs(6, A, dtype, False, kl, seed=62)
    logits[::2] = torch.finfo(DT[dtype]).min
    kw["old_log_prob"][::2] = 0.1 - math.log(A)
    if kl == "full":
        kw["reference_logits"][::2] = torch.finfo(DT[dtype]).min
    if kl == "sampled":
        kw["reference_log_prob"][::2] = 0.2 - math.log(A)
    _check(logits, action, kw, beta=0.0 if kl == "none" else 0.07)


@pytest.mark.parametrize("kl", ["none", "sampled", "full"])
@pytest.mark.parametrize("m", [1e2, 1e3, 1e4, -6e4, 6e4])
@pytest.mark.parametrize("A", [82, 700, 5001, 33000])
def test_logits_around_a_large_value(cuda, A, m, kl):
    """A constant added to a row's logits changes p by nothing but what the
    logits' own type rounds: x - m is taken first, and is as exact as it was."""
    N = 100 if A < 5000 else 40
    logits, action, kw = _inputs(N, A, "fp32", True, kl, seed=61)
    logits = logits + m
    x = logits.double().masked_fill(~kw["legal"], -math.inf)
    lp = torch.log_softmax(x, -1).gather(-1, action.long()[:, None])[:, 0]
    kw["old_log_prob"] = lp.float() + 0.3 * torch.sin(torch.arange(N, device="cuda"))
    if kl == "sampled":
        kw["reference_log_prob"] = lp.float() + 0.2 * torch.cos(torch.arange(N, device="cuda"))
    if kl == "full":
        kw["reference_logits"] = kw["reference_logits"] + m
    _check(logits, action, kw, beta=0.0 if kl == "none" else 0.07)


@pytest.mark.parametrize("kl", ["none", "sampled"])
@pytest.mark.parametrize("dtype,m", [("bf16", 1e4), ("bf16", 1e30), ("fp16", 1e3), ("fp16", 6e4), ("fp16", -6e4)])
@pytest.mark.parametrize("A", [82, 700, 33000])
def test_ties_at_a_large_value(cuda, A, dtype, m, kl):
    """Half of a row's logits at m, the others one step of the type below
    (p of m is 2 / A, or a little less where the step is small)."""
    N = 40
    _, action, kw = _inputs(N, A, dtype, False, kl, seed=63)
    top = torch.tensor(m, dtype=DT[dtype], device="cuda")
    below = torch.nextafter(top, torch.full_like(top, -math.inf))
    logits = torch.where(torch.arange(A, device="cuda") % 2 == 0, top, below).expand(N, A).contiguous()
    action = action // 2 * 2
    lp = torch.log_softmax(logits.double(), -1).gather(-1, action.long()[:, None])[:, 0]
    kw["old_log_prob"] = lp.float() + 0.3 * torch.sin(torch.arange(N, device="cuda"))
    if kl == "sampled":
        kw["reference_log_prob"] = lp.float() + 0.2 * torch.cos(torch.arange(N, device="cuda"))
    # weights that the gradients stay normal numbers of the type with
    kw["weight"] = torch.full((N,), 256.0, device="cuda")
    _check(logits, action, kw, beta=0.0 if kl == "none" else 0.07)


@pytest.mark.parametrize("kl", ["none", "sampled", "full"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("A", [700, 40000])
def test_long_rows_of_the_lowest_value(cuda, A, dtype, kl):
    _lowest_rows(A, dtype, kl)


def _sliced(x, pad):
    """`x` as the first columns of rows `pad` elements longer."""
    wide = torch.full((x.shape[0], x.shape[1] + pad), math.nan, dtype=x.dtype, device="cuda")
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


@pytest.mark.parametrize("pad", [0, 1])
def test_borders_of_long_sums(cuda, pad):
    """Rows of one CTA, taken vector by vector or (rows an odd number of
    elements apart) one by one, whose sums round one way all along: each
    thread adds 222 terms of 0.57 steps to a first one of 1.  Log-probability
    and clipping as of any row."""
    N, A = 80, 57001
    x = torch.full((N, A), -16.5, dtype=torch.bfloat16, device="cuda")
    x[:, :256] = 0.0
    x = _sliced(x, pad)
    action = 3 * torch.arange(N, device="cuda", dtype=torch.int32)
    lp = torch.log_softmax(x.double(), -1).gather(-1, action.long()[:, None])[:, 0]
    steps = (torch.arange(N, device="cuda") % 7 - 3).to(torch.int32)
    for adv, border in ((1.0, math.log1p(0.2)), (-1.0, math.log1p(-0.2))):
        old = ((lp - border).float().view(torch.int32) + steps).view(torch.float32)
        out = _check(x, action, dict(old_log_prob=old, advantage=torch.full((N,), adv, device="cuda")), beta=0.0)
        assert 0 < int(out.clipped.sum()) < N


@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("span", [0.03, 0.3, 3.0, 30.0])
@pytest.mark.parametrize("dtype,A", [("fp32", 28000), ("bf16", 57000)])
def test_rows_that_ascend(cuda, dtype, A, span, pad):
    """Every element or vector is a new maximum: sums are rescaled all along."""
    N = 80
    end = span * (1 + torch.arange(N, device="cuda", dtype=torch.float64) / N)[:, None]
    x = _sliced((-end * (1 - torch.linspace(0, 1, A, device="cuda", dtype=torch.float64))).to(DT[dtype]), pad)
    action = (A - 1 - 5 * torch.arange(N, device="cuda")).to(torch.int32)
    lp = torch.log_softmax(x.double(), -1).gather(-1, action.long()[:, None])[:, 0]
    _check(x, action, dict(old_log_prob=lp.float() + 0.3 * torch.sin(torch.arange(N, device="cuda")),
                           advantage=torch.cos(torch.arange(N, device="cuda", dtype=torch.float32))), beta=0.0)


@pytest.mark.parametrize("A", [82, 2000])
def test_kl_without_a_coefficient_is_a_statistic(cuda, A):
    """References whose estimate overflows, or that exclude the action: the
    KL is infinite, and loss and gradient are those of a call without one."""
    logits, action, kw = _inputs(20, A, "fp32", True, "sampled", seed=66)
    reference = kw.pop("reference_log_prob")
    want = clipped_policy_loss(logits, action, **kw)
    reference[:5] += 300.0
    reference[5:9] = -math.inf
    got = clipped_policy_loss(logits, action, reference_log_prob=reference, **kw)
    assert torch.isposinf(got.kl[:9]).all() and torch.isfinite(got.kl[9:]).all()
    for name in ("loss", "log_prob", "clipped", "grad_logits"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("A", [82, 81, 2000, 2001, 40000])
def test_lowest_value_in_the_logits_alone(cuda, A, dtype):
    """Actions masked by the type's lowest value where the reference is not:
    their differences are of 1e38, their p and gradients 0.  A weight 2^12
    times larger gives 2^12 times the gradient, bit for bit."""
    logits, action, kw = _inputs(30, A, dtype, True, "full", seed=64)
    legal = kw.pop("legal")
    logits = logits.masked_fill(~legal, torch.finfo(DT[dtype]).min)
    grads = []
    for weight in (2.0 ** -6, 2.0 ** 6):
        kw["weight"] = torch.full((30,), weight, device="cuda")
        out = clipped_policy_loss(logits, action, kl_coefficient=4.0, **kw)
        assert torch.isfinite(out.loss) and torch.isfinite(out.kl).all() and not out.grad_logits[~legal].any()
        grads.append(out.grad_logits.float())
    # (the smallest normal number itself may be the rounding of a subnormal one, in coarser steps)
    normal = grads[0].abs() > torch.finfo(DT[dtype]).smallest_normal
    assert bool(normal.any()) and torch.equal((grads[0] * 2.0 ** 12)[normal], grads[1][normal])
    assert torch.isfinite(grads[1]).all()


@pytest.mark.parametrize("A", [82, 2000])
def test_a_nan_meets_an_advantage_of_zero(cuda, A):
    """0 times a ratio that overflows is 0, times one that is NaN is NaN: a
    check of the loss sees the row whose gradient is NaN."""
    logits, action, kw = _inputs(8, A, "fp32", False, "none", seed=65)
    kw["advantage"][3] = 0.0
    assert math.isfinite(float(clipped_policy_loss(logits, action, **kw).loss))
    bad = logits.clone()
    bad[3, 5] = math.nan
    out = clipped_policy_loss(bad, action, **kw)
    assert math.isnan(float(out.loss)) and bool(torch.isnan(out.grad_logits[3]).any())
    kw["old_log_prob"][3] = math.nan
    out = clipped_policy_loss(logits, action, **kw)
    assert math.isnan(float(out.loss)) and bool(torch.isnan(out.grad_logits[3]).any())


@pytest.mark.parametrize("kl", ["none", "sampled"])
@pytest.mark.parametrize("A", [82, 2000])
def test_a_ratio_beyond_32_bits_with_a_small_weight(cuda, A, kl):
    """e^90 leaves fp32, 1e-5 of it does not: the gradient is as finite as
    the loss."""
    logits, action, kw = _inputs(20, A, "fp32", True, kl, seed=67)
    kw["old_log_prob"] = kw["old_log_prob"] - 90.0
    kw["advantage"] = -1.0 - kw["advantage"].abs()
    kw["weight"] = torch.full((20,), 1e-5, device="cuda")
    _check(logits, action, kw, beta=0.0 if kl == "none" else 0.1)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("size", [(40, 3), (40, 82), (40, 81), (20, 512), (12, 700), (12, 701), (3, 40000), (90, 20003)],
                         ids=str)
def test_rows_of_the_lowest_value_against_a_reference_that_is_not(cuda, size, dtype):
    """The uniform policy again: loss and statistics as of rows of zeros (in
    fp16, where 2^-24 of the value is no more than 4e-3, as of rows of that
    value)."""
    N, A = size
    logits, action, kw = _inputs(N, A, dtype, True, "full", seed=68)
    logits[::2] = torch.finfo(torch.float16).min if dtype == "fp16" else 0.0
    kw["old_log_prob"][::2] = 0.1 - torch.log(kw["legal"][::2].sum(-1).float())
    kw["weight"] = torch.full((N,), 3.0, device="cuda")
    want, clipped = _plain(logits, action, kl_coefficient=0.7, **kw)
    logits[::2] = torch.finfo(DT[dtype]).min
    for pad in (0, 1):
        out = clipped_policy_loss(_sliced(logits, pad), action, kl_coefficient=0.7, **kw)
        assert torch.equal(out.clipped, clipped)
        for name in ("loss", "log_prob", "kl"):
            value, tol = want[name]
            err = (getattr(out, name).double() - value).abs()
            assert float((err - tol).max()) <= 0, f"{name}: off by {float(err.max()):.3g}"
        err = (out.grad_logits[1::2].double() - want["grad_logits"][0][1::2]).abs()
        assert float((err - want["grad_logits"][1][1::2]).max()) <= 0
