"""Log-probabilities, entropy, best actions and their gradient
(scacchi_log_probs, scacchi_log_probs_gradient) against the definition in 64
bits.

Tolerances, from the kernels' arithmetic (U = 2^-24 the largest rounding of a
32-bit operation, relative to its result).  An exponent v = u log2 e is off by
3 U |v| (difference, scale, product), its power by 2 U more, ex2.approx's
2^-22: e is off by (3 |u| + 6) U of itself.  With p = e / s the sum s is off
by the mean of that, 3 U sum p |u| + 6 U, and by its additions: at most 4 of
W = 8 elements, a thread's vectors (n / 256 / 4 for the longest rows a CTA
takes) and 9 levels of the tree, each U of the partial sum; call this E.

  log_sum  |log s| U + 2 U (logf) + E
  log_prob 3 U |u_a| + the above + U of each of the two terms
  entropy  the mean t / s: E + (3 |u| + 6) U, weighted by p |u|; and log_sum's
  gradient p off by (3 |u| + 8) U + log_sum's 64-bit rounding U |log s| + E,
           times |g + h (log p + H)|, whose own parts are off by U each and
           by 3 U (|u| + |log s|); then rounded once to its type.
"""

import math

import pytest
import torch

from scacchi_b200 import _lib
from scacchi_b200.log_probs import policy_log_probs, policy_log_probs_gradient

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _adds(n):
    return 8 + n / 1024 + 12


def _inputs(N, A, dtype, legal, seed=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + 7 * A + N)
    logits = (spread * torch.randn((N, A), generator=g, device="cuda")).to(DT[dtype])
    mask = None
    if legal:
        mask = torch.rand((N, A), generator=g, device="cuda") < 0.6
        mask[::5] = False  # rows without any legal action
    action = torch.randint(0, A, (N,), generator=g, device="cuda", dtype=torch.int32)
    action[1::7] = -1
    return logits, action, mask


def _definition(logits, action, legal, T):
    x = logits.double()
    keep = x != -math.inf
    if legal is not None:
        keep = keep & legal.bool()
    x = torch.where(keep, x, -math.inf)
    top = x.amax(-1)
    base = torch.where(top == -math.inf, 0.0, top)
    u = (x - base[:, None]) / T
    e = u.exp()
    s = e.sum(-1)
    p = torch.where(s[:, None] > 0, e / s[:, None], 0.0)
    au = torch.where(e > 0, u.abs(), 0.0)
    mean = (p * au).sum(-1)
    log_sum = s.log()
    logp = torch.where(keep, u - log_sum[:, None], -math.inf)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    E = (3 * mean + 8 + _adds(x.shape[1])) * U
    ls = torch.where(s > 0, log_sum, 0.0)
    sum_tol = ls.abs() * U + 2 * U + E
    k = action.long()
    inside = (k >= 0) & (k < x.shape[1])
    at = k.clamp(0, x.shape[1] - 1)[:, None]
    lp = torch.where(inside, logp.gather(-1, at)[:, 0], 0.0)
    lp_tol = 4 * U * torch.where(lp.isfinite(), u.gather(-1, at)[:, 0].abs(), 0.0) + sum_tol + U * torch.where(
        lp.isfinite(), lp.abs(), 0.0)
    h_tol = (p * au * ((3 * au + 6) * U + 2 * E[:, None])).sum(-1) + _adds(x.shape[1]) * U * mean + sum_tol + 3 * U * (
        mean + entropy)
    want = dict(log_prob=(lp, lp_tol), entropy=(entropy, h_tol), max_logit=(top, 0 * E), log_sum=(log_sum, sum_tol))
    return want, dict(x=x, keep=keep, u=u, au=au, p=p, logp=logp, entropy=entropy, E=E, ls=ls, sum_tol=sum_tol,
                      inside=inside, at=at)


def _near(got, want, tol, name):
    got = got.double()
    assert got.shape == want.shape, name
    fin = want.isfinite()
    assert torch.equal(got[~fin], want[~fin]), name
    assert bool(((got - want).abs() <= tol)[fin].all()), (name, float(((got - want).abs() - tol)[fin].max()))


def _check_top(out, d, top, T):
    x = d["x"]
    N, A = x.shape
    n = min(top, A)
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    found = order.values[:, :n] > -math.inf
    idx = torch.full((N, top), -1, dtype=torch.int32, device=x.device)
    idx[:, :n] = torch.where(found, order.indices[:, :n], -1).to(torch.int32)
    assert torch.equal(out.top_action, idx)
    value = torch.full((N, top), -math.inf, dtype=torch.float64, device=x.device)
    value[:, :n] = torch.where(found, d["logp"].gather(-1, order.indices[:, :n]), -math.inf)
    tol = torch.zeros_like(value)
    tol[:, :n] = (4 * U * d["u"].gather(-1, order.indices[:, :n]).abs() + d["sum_tol"][:, None]
                  + U * value[:, :n].abs())
    _near(out.top_log_prob, value, torch.where(value.isfinite(), tol, 0.0), "top_log_prob")


def _check(logits, action, legal, T, top, **kw):
    want, d = _definition(logits, action, legal, T)
    out = policy_log_probs(logits, action, legal=legal, temperature=T, top=top, **kw)
    for name, (value, tol) in want.items():
        _near(getattr(out, name), value, tol, name)
    if top:
        _check_top(out, d, top, T)
    else:
        assert out.top_action is None and out.top_log_prob is None
    return out, d


def _check_gradient(logits, action, legal, T, out, d, g, h):
    got = policy_log_probs_gradient(logits, action, out, grad_log_prob=g, grad_entropy=h, legal=legal, temperature=T)
    assert got.dtype == logits.dtype and got.shape == logits.shape
    zero = torch.zeros(logits.shape[0], dtype=torch.float64, device=logits.device)
    kept = d["inside"] & d["keep"].gather(-1, d["at"])[:, 0]
    G = zero if g is None else torch.where(kept, g.double(), 0.0)
    H = zero if h is None else h.double()
    p, logp = d["p"], torch.where(d["keep"], d["logp"], 0.0)
    # 2^-1e4 is where exponents end: p is 0 there, and so is p log p
    inner = G[:, None] + H[:, None] * torch.where(p > 0, logp + d["entropy"][:, None], 0.0)
    grad = -p * inner
    grad.scatter_add_(-1, d["at"], G[:, None])
    grad = torch.where(d["keep"], grad / T, 0.0)
    off = (3 * d["au"] + 3 * d["ls"].abs()[:, None] + 10) * U + d["sum_tol"][:, None]
    inner_tol = (4 * U * (G.abs()[:, None] + H.abs()[:, None] * (logp.abs() + d["entropy"][:, None]))
                 + H.abs()[:, None] * (off + 4 * d["sum_tol"][:, None] + 8 * U * d["entropy"][:, None]
                                       + 3 * U * _adds(p.shape[1]) * d["entropy"][:, None]))
    tol = (p * (inner.abs() * off + inner_tol) + 4 * U * grad.abs()) / T
    tol.scatter_add_(-1, d["at"], 4 * U * G.abs()[:, None] / T)
    f = torch.finfo(logits.dtype)
    tol = tol * (1 + f.eps) + grad.abs() * f.eps / 2 + f.smallest_normal * f.eps
    tol = tol + 2.0 ** -126 * (inner.abs() + 1) / T  # a p below the smallest normal number is 0
    _near(got, grad, tol, "gradient")


# (rows, actions): rows of one, two, odd and even lanes' worth, around the border between short and long ones, of one
# and of several CTAs, with heads and tails beside whole vectors
SHAPES = [(1, 1), (3, 2), (64, 82), (33, 83), (129, 122), (7, 255), (5, 512), (6, 513), (300, 1000), (9, 4099),
          (5, 20001), (3, 65536), (2, 131071), (1, 262144)]


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("legal", [False, True], ids=["all", "legal"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradient(cuda, shape, dtype, legal):
    N, A = shape
    logits, action, mask = _inputs(N, A, dtype, legal)
    gen = torch.Generator(device="cuda").manual_seed(A)
    g, h = torch.randn((2, N), generator=gen, device="cuda").unbind(0)
    for T, top in ((1.0, 0), (0.7, min(5, A + 1)), (1.3, 32)):
        out, d = _check(logits, action, mask, T, top)
        _check_gradient(logits, action, mask, T, out, d, g, h)
    _check_gradient(logits, action, mask, T, out, d, g, None)
    _check_gradient(logits, action, mask, T, out, d, None, h)


# many rows: a lane each, rows of whole 16-byte pieces, batches and groups that the last rows do not fill, rows between
# the short and the long ones
MANY = [(40001, 82), (38017, 64), (38000, 8), (40003, 5), (9001, 128), (5003, 361), (1193, 513), (1200, 1000), (1185, 1024),
        (1184, 1025), (1190, 2048), (1184, 2049)]


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_many_rows(cuda, shape, dtype):
    N, A = shape
    for legal in (False, True):
        logits, action, mask = _inputs(N, A, dtype, legal)
        out, d = _check(logits, action, mask, 0.9, 3)
        g, h = torch.linspace(-1, 1, N, device="cuda"), torch.linspace(1, -0.5, N, device="cuda")
        _check_gradient(logits, action, mask, 0.9, out, d, g, h)
    wide, action, _ = _inputs(N, A + 3, dtype, False, seed=1)
    logits = wide[:, 1:A + 1]
    out, d = _check(logits, action, mask, 1.0, 2)
    _check_gradient(logits, action, mask, 1.0, out, d, g, h)


@pytest.mark.parametrize("A", [64, 82])
def test_equal_logits_of_many_rows(cuda, A):
    logits = torch.randint(0, 3, (40000, A), device="cuda").bfloat16()
    logits[::3] = 1.0
    _check(logits, torch.zeros(40000, dtype=torch.int32, device="cuda"), None, 1.0, 32)


def test_plain_calls_and_the_python_way_agree(cuda, monkeypatch):
    """Every call through the extension module and without it."""
    class Nothing:
        @staticmethod
        def log_probs(*args):
            return None

        log_probs_gradient = log_probs

    cases = [_inputs(N, A, d, legal) for N, A in ((64, 82), (7, 5000)) for d in sorted(DT) for legal in (False, True)]

    def run():
        res = []
        for logits, action, mask in cases:
            for top in (0, 4):
                out = policy_log_probs(logits, action, legal=mask, temperature=0.7, top=top)
                ones = torch.ones_like(out.entropy)
                res += [*out, *(policy_log_probs_gradient(logits, action, out, grad_log_prob=g, grad_entropy=h,
                                                          legal=mask, temperature=0.7)
                                for g, h in ((ones, None), (None, ones), (ones, ones)))]
        return res

    fast = run()
    assert sum(v is not None for v in [_lib.host().log_probs(c[0], c[1], c[2], 1.0, 2) for c in cases]) == len(cases)
    monkeypatch.setattr(_lib, "host", lambda: Nothing)
    for a, b in zip(fast, run()):
        assert a is None and b is None or a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("shape", [(40, 82), (20, 700), (6, 30000)], ids=str)
def test_strided_rows_and_offsets(cuda, shape, dtype):
    N, A = shape
    for pad, begin in ((6, 0), (6, 1), (6, 3), (14, 2), (64, 8)):
        wide, action, mask = _inputs(N, A + pad, dtype, True, seed=pad)
        logits = wide[:, begin:begin + A]
        legal = mask[:, begin:begin + A]
        action = action.clamp(max=A)  # A itself is out of range
        out, d = _check(logits, action, legal, 1.0, 7)
        g = torch.linspace(-1, 1, N, device="cuda")
        _check_gradient(logits, action, legal, 1.0, out, d, g, -g)
    # a mask and rows off their boundaries, dense
    flat, action, _ = _inputs(1, N * A + 3, dtype, False, seed=9)
    bits = torch.rand(N * A + 3, device="cuda") < 0.5
    logits, legal = flat[0, 3:].view(N, A), bits[1:N * A + 1].view(N, A)
    action = torch.arange(N, device="cuda") % A
    out, d = _check(logits, action, legal, 1.0, 3)
    _check_gradient(logits, action, legal, 1.0, out, d, torch.ones(N, device="cuda"), None)


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("shape", [(40, 64), (1, 64), (3, 32), (38017, 64), (50, 512), (7, 8)], ids=str)
def test_rows_of_whole_pieces_strided(cuda, shape, dtype):
    """Rows of a multiple of 32 bytes, the first on a 16-byte boundary, others on none."""
    N, A = shape
    for pad in (1, 3, 8):
        wide, action, mask = _inputs(N, A + pad, dtype, True, seed=pad)
        logits, legal = wide[:, :A], mask[:, :A]
        out, d = _check(logits, action.clamp(max=A), legal, 1.0, 3)
        g = torch.linspace(-1, 1, N, device="cuda")
        _check_gradient(logits, action.clamp(max=A), legal, 1.0, out, d, g, g)


@pytest.mark.parametrize("A", [82, 700, 70000])
def test_far_apart_logits(cuda, A):
    """A maximum of 1e20 to 1e35 above ordinary logits: exponents of up to
    1e38, which float32 holds, at every temperature's end."""
    logits, action, _ = _inputs(8, A, "fp32", False)
    action[:4] = A // 2
    logits[:, A // 2] = torch.tensor([1e30, 1e35, 3e34, 1e20, -1e34, 6e29, 7e29, 2e32], device="cuda")
    logits[1, 3] = -3e34
    for T in (1e-3, 1.0, 1e3):
        out, d = _check(logits, action, None, T, 5)
        _check_gradient(logits, action, None, T, out, d, torch.ones(8, device="cuda"), torch.ones(8, device="cuda"))


def test_transposed_logits_are_copied(cuda):
    logits, action, _ = _inputs(82, 64, "fp32", False)
    out, _ = _check(logits, action, None, 1.0, 2)
    again = policy_log_probs(logits.t().contiguous().t(), action, top=2)
    for a, b in zip(out, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("A", [82, 512, 513, 5000, 40000])
@pytest.mark.parametrize("dtype", sorted(DT))
def test_equal_logits_go_by_index(cuda, A, dtype):
    """All equal, few values, the type's lowest value everywhere, and zeros of both signs."""
    g = torch.Generator(device="cuda").manual_seed(A)
    rows = torch.zeros((8, A), device="cuda")
    rows[1] = 3.0
    rows[2] = torch.randint(0, 3, (A,), generator=g, device="cuda").float()
    rows[3] = torch.finfo(DT[dtype]).min
    rows[4] = torch.where(torch.rand(A, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    rows[5] = -torch.arange(A, device="cuda") / A
    rows[6] = torch.arange(A, device="cuda") / A
    rows[7] = torch.finfo(DT[dtype]).min
    rows[7, A // 2] = 1.0
    logits = rows.to(DT[dtype])
    action = torch.full((8,), A // 2, device="cuda")
    legal = torch.rand((8, A), generator=g, device="cuda") < 0.9
    legal[:, A // 2] = True
    for mask in (None, legal):
        out, d = _check(logits, action, mask, 1.0, 32)
        _check_gradient(logits, action, mask, 1.0, out, d, torch.ones(8, device="cuda"), torch.ones(8, device="cuda"))


@pytest.mark.parametrize("A", [82, 700, 70000])
def test_masked_places_may_hold_anything(cuda, A):
    logits, action, _ = _inputs(16, A, "fp32", False)
    legal = torch.rand((16, A), device="cuda") < 0.5
    legal[3] = False
    legal[4] = False
    legal[4, A - 1] = True  # one action left
    legal[5] = True
    logits[5] = -math.inf
    logits[6, ::2] = -math.inf
    clean = logits.masked_fill(~legal, 0.0)
    for junk in (math.inf, math.nan, -math.inf, 3e38):
        dirty = logits.masked_fill(~legal, junk)
        a, d = _check(dirty, action, legal, 0.5, 6)
        b, _ = _check(clean, action, legal, 0.5, 6)
        for u, v in zip(a, b):
            assert torch.equal(u, v)
        one = torch.ones(16, device="cuda")
        _check_gradient(dirty, action, legal, 0.5, a, d, one, one)
    assert float(a.entropy[3]) == 0.0 and float(a.entropy[4]) == 0.0 and float(a.log_sum[3]) == -math.inf
    assert a.top_action[4].tolist() == [A - 1, -1, -1, -1, -1, -1]


@pytest.mark.parametrize("A", [82, 700, 70000])
@pytest.mark.parametrize("junk", [math.nan, math.inf])
def test_a_legal_nan_or_infinity_makes_its_row_nan(cuda, A, junk):
    logits, action, _ = _inputs(6, A, "fp32", False)
    action[:] = 0
    whole = policy_log_probs(logits, action, top=3)
    logits[2, A // 3] = junk
    out = policy_log_probs(logits, action, top=3)
    for name in ("log_prob", "entropy", "log_sum"):
        assert bool(getattr(out, name)[2].isnan())
    keep = [0, 1, 3, 4, 5]
    for a, b in zip(out, whole):
        assert torch.equal(a[keep], b[keep])
    grad = policy_log_probs_gradient(logits, action, out, grad_log_prob=torch.ones(6, device="cuda"))
    assert bool(grad[2].isnan().any()) and bool(grad[keep].isfinite().all())


@pytest.mark.parametrize("A", [82, 700, 70000])
def test_large_offsets_and_sharp_rows(cuda, A):
    """Rows far from zero, and nearly deterministic ones."""
    logits, action, _ = _inputs(8, A, "fp32", False)
    for shift, T in ((1e6, 1.0), (-1e6, 1.0), (0.0, 1e-3), (0.0, 1e3), (3e37, 2.0)):
        x = logits + shift
        out, d = _check(x, action, None, T, 4)
        _check_gradient(x, action, None, T, out, d, torch.ones(8, device="cuda"), None)


def test_gradient_against_differences(cuda):
    """Central differences of the 64-bit definition, whose second-order term
    is below h^2 max |f'''| / 6 < 2e-8 (derivatives of log p and entropy of
    bounded logits stay below 100) for h = 1e-5, plus 1e-16 / h of rounding;
    the kernel's own tolerance for |u| <= 12, |log s| <= 4 and 30 actions is
    below 70 U = 5e-6 a unit of p (|inner| + 1) / T < 1.25 x 4."""
    logits, action, mask = _inputs(10, 30, "fp32", True)
    action = action.clamp(min=0)
    action[mask.any(-1)] = mask[mask.any(-1)].int().argmax(-1).int()
    g = torch.linspace(-1, 1, 10, device="cuda")
    h = torch.linspace(0.5, -0.5, 10, device="cuda")
    out = policy_log_probs(logits, action, legal=mask, temperature=0.8)
    grad = policy_log_probs_gradient(logits, action, out, grad_log_prob=g, grad_entropy=h, legal=mask,
                                     temperature=0.8).double()

    def value(x):
        want, _ = _definition(x, action, mask, 0.8)
        lp = torch.where(want["log_prob"][0].isfinite(), want["log_prob"][0], 0.0)
        return g.double() * lp + h.double() * want["entropy"][0]

    for a in range(30):
        step = torch.zeros((10, 30), dtype=torch.float64, device="cuda")
        step[:, a] = 1e-5
        diff = (value(logits.double() + step) - value(logits.double() - step)) / 2e-5
        assert float((diff - grad[:, a]).abs().max()) < 2.5e-5


def test_shapes_types_and_empty_batches(cuda):
    logits, action, mask = _inputs(24, 82, "bf16", True)
    flat = policy_log_probs(logits, action, legal=mask, top=3)
    out = policy_log_probs(logits.view(2, 3, 4, 82), action.view(2, 3, 4).long(), legal=mask.view(2, 3, 4, 82), top=3)
    assert out.log_prob.shape == (2, 3, 4) and out.top_action.shape == (2, 3, 4, 3)
    for a, b in zip(flat, out):
        assert torch.equal(a, b.reshape(a.shape))
    one = policy_log_probs(logits[1], action[1], legal=mask[1], top=3)
    assert one.log_prob.shape == () and torch.equal(one.top_action, flat.top_action[1])
    assert torch.equal(policy_log_probs(logits, action, legal=mask.to(torch.uint8)).log_prob, flat.log_prob)
    far = action.long()
    far[0] = (1 << 32) + 3  # stays out of range
    assert float(policy_log_probs(logits, far).log_prob[0]) == 0.0
    none = policy_log_probs(logits[:0], action[:0], top=2)
    assert none.log_prob.shape == (0,) and none.top_action.shape == (0, 2)
    assert policy_log_probs_gradient(logits[:0], action[:0], none, grad_log_prob=none.log_prob).shape == (0, 82)
    grad = policy_log_probs_gradient(logits.view(2, 3, 4, 82), action.view(2, 3, 4), out, legal=mask.view(2, 3, 4, 82),
                                     grad_entropy=torch.ones((2, 3, 4), device="cuda", dtype=torch.bfloat16))
    assert grad.shape == (2, 3, 4, 82)
    tracked = logits.clone().requires_grad_(True)
    assert not policy_log_probs(tracked, action).log_prob.requires_grad
    assert not policy_log_probs_gradient(tracked, action, flat, grad_log_prob=flat.entropy).requires_grad


@pytest.mark.parametrize("shape", [(66001, 32768), (26_300_003, 82)], ids=str)
def test_offsets_past_32_bits(cuda, shape):
    """The last of more than 2^31 logits."""
    N, A = shape
    assert N * A > 1 << 31
    logits = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    action = torch.arange(N, device="cuda", dtype=torch.int32) % A
    legal = torch.ones(shape, dtype=torch.bool, device="cuda")
    legal[-2, ::3] = False
    out = policy_log_probs(logits, action, legal=legal, top=2)
    last = slice(-5, None)
    want, d = _definition(logits[last], action[last], legal[last], 1.0)
    for name, (value, tol) in want.items():
        _near(getattr(out, name)[last], value, tol, name)
    _check_top(type(out)(*(v[last] for v in out)), d, 2, 1.0)
    g = torch.ones(N, device="cuda")
    grad = policy_log_probs_gradient(logits, action, out, grad_log_prob=g, grad_entropy=g, legal=legal)
    few = policy_log_probs(logits[last], action[last], legal=legal[last])
    small = policy_log_probs_gradient(logits[last], action[last], few, grad_log_prob=g[last], grad_entropy=g[last],
                                      legal=legal[last])
    # the row's numbers of either call are off by less than 1e-5 each, and one step of bfloat16
    assert bool(((grad[last].float() - small.float()).abs() <= 1e-4 * small.float().abs() + 2.0 ** -8 * small.float().abs()
                 + 1e-7).all())


def test_repeats_bit_for_bit(cuda):
    for shape in ((4096, 82), (64, 20001), (2, 131071)):
        logits, action, mask = _inputs(*shape, "bf16", True)
        first = policy_log_probs(logits, action, legal=mask, top=20)
        for _ in range(3):
            for a, b in zip(first, policy_log_probs(logits, action, legal=mask, top=20)):
                assert torch.equal(a, b)


def test_captured_and_replayed(cuda):
    for shape in ((64, 82), (8, 131071)):
        logits, action, _ = _inputs(*shape, "fp32", False)
        g = torch.ones(shape[0], device="cuda")
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            policy_log_probs(logits, action, top=4)
            with torch.cuda.graph(graph, stream=side):
                out = policy_log_probs(logits, action, top=4)
                grad = policy_log_probs_gradient(logits, action, out, grad_log_prob=g)
        torch.cuda.synchronize()
        logits.copy_(_inputs(*shape, "fp32", False, seed=3)[0])
        graph.replay()
        torch.cuda.synchronize()
        again = policy_log_probs(logits, action, top=4)
        for a, b in zip(out, again):
            if a is not None:
                assert torch.equal(a, b)
        assert torch.equal(grad, policy_log_probs_gradient(logits, action, again, grad_log_prob=g))


def test_refusals(cuda):
    x, k = torch.zeros((3, 5), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    out = policy_log_probs(x, k)
    one = torch.ones(3, device="cuda")
    for bad in (dict(logits=x.double()), dict(logits=torch.zeros((3, 0), device="cuda")), dict(action=k[:2]),
                dict(action=k.float()), dict(action=k.cpu()), dict(legal=torch.ones((3, 4), dtype=torch.bool).cuda()),
                dict(legal=x), dict(temperature=0.0), dict(temperature=math.nan), dict(temperature=2e3)):
        kw = dict(logits=x, action=k)
        kw.update(bad)
        with pytest.raises(ValueError):
            policy_log_probs(**kw)
        with pytest.raises(ValueError):
            policy_log_probs_gradient(out=out, grad_log_prob=one, **kw)
    for top in (-1, 33):
        with pytest.raises(ValueError, match="top"):
            policy_log_probs(x, k, top=top)
    with pytest.raises(ValueError, match="both"):
        policy_log_probs_gradient(x, k, out)
    for bad in (one[:2], one.cpu(), one.int()):
        with pytest.raises(ValueError, match="grad_log_prob"):
            policy_log_probs_gradient(x, k, out, grad_log_prob=bad)
        with pytest.raises(ValueError, match="max_logit"):
            policy_log_probs_gradient(x, k, out._replace(max_logit=bad), grad_log_prob=one)


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("shape", [(6, 82), (40000, 82), (6, 700), (1200, 1000), (6, 70000)], ids=str)
@pytest.mark.parametrize("junk", [math.nan, math.inf])
def test_all_numbers_of_a_row_with_a_legal_nan_or_infinity_are_nan(cuda, shape, dtype, junk):
    """max_logit among them, beside other logits and where they are -inf; what
    is said of actions out of range and of illegal ones holds there too."""
    N, A = shape
    logits, action, _ = _inputs(N, A, dtype, False)
    legal = torch.ones((N, A), dtype=torch.bool, device="cuda")
    legal[:, 1] = False
    action[:5] = torch.tensor([0, A // 3, 0, -1, 1], dtype=torch.int32)
    whole = policy_log_probs(logits, action, legal=legal)
    logits[1] = -math.inf
    logits[[0, 1, 3, 4], A // 3] = junk
    for mask in (legal, None):
        out = policy_log_probs(logits, action, legal=mask, top=2)
        for name in ("entropy", "max_logit", "log_sum"):
            assert bool(getattr(out, name)[[0, 1, 3, 4]].isnan().all()), name
        assert out.log_prob[:2].isnan().all() and float(out.log_prob[3]) == 0.0
    # (the last row's action is illegal with the mask)
    out = policy_log_probs(logits, action, legal=legal)
    assert float(out.log_prob[4]) == -math.inf
    for a, b in zip(out[:4], whole[:4]):
        assert torch.equal(a[5:], b[5:]) and torch.equal(a[2], b[2])
    one = torch.ones(N, device="cuda")
    grad = policy_log_probs_gradient(logits, action, out, grad_log_prob=one, grad_entropy=one, legal=legal)
    assert bool(grad[[0, 1]].isnan().any(-1).all()) and bool(grad[2].isfinite().all())
    assert bool(grad[5:].isfinite().all())


@pytest.mark.parametrize("A", [200, 600, 9000])
@pytest.mark.parametrize("T", [1.0, 0.7, 3.0])
def test_log_probs_are_rounded_once(cuda, A, T):
    """n logits of 0, one u below them of e^-40 or less, the others -inf:
    the sum is n in any type (n + e^-40 rounds to n in 32 bits), so log n, u /
    T - log n and the entropy are off by their last rounding, 2^-24 of their
    value, by the logarithm's 1.2e-10 of its own (the series' next term, 2e-11
    twice, of at least 0.35) < 2^-32, and by 64-bit roundings and e^-40 (41 +
    log n) < 2^-50."""
    N = 180
    n = 1 + torch.arange(N, device="cuda") % (A - 2)
    logits = torch.where(torch.arange(A, device="cuda") < n[:, None], 0.0, -math.inf)
    u = -40.0 * T - torch.arange(N, device="cuda") * 0.37
    logits[:, A - 1] = u
    action = torch.full((N,), A - 1, dtype=torch.int32, device="cuda")
    action[::2] = 0
    offset = torch.linspace(-3, 3, 13, device="cuda").round()[torch.arange(N, device="cuda") % 13]  # (0 is exact)
    logits[:, :A - 1] += offset[:, None]
    logits[:, A - 1] += offset
    u = (logits[:, A - 1].double() - offset.double()) / T
    out = policy_log_probs(logits, action, temperature=T, top=1)
    log_n = n.double().log()
    for name, want in (("log_sum", log_n), ("entropy", log_n), ("log_prob", torch.where(action == 0, -log_n, u - log_n))):
        got = getattr(out, name).double()
        assert bool(((got - want).abs() <= U * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -50).all()), name
    assert bool(((out.top_log_prob[:, 0].double() + log_n).abs() <= U * (1 + 2.0 ** -8) * log_n + 2.0 ** -50).all())


@pytest.mark.parametrize("A", [82, 700, 20000])
def test_log_probs_of_differences_beyond_float32(cuda, A):
    """-3e38 below 3e38 at a temperature of 1000: 64 bits hold the difference,
    and float32 holds its thousandth."""
    logits = torch.zeros((4, A), device="cuda")
    logits[:, 5] = 3e38
    logits[:, 9] = -3e38
    out = policy_log_probs(logits, torch.tensor([5, 9, 0, 9], device="cuda"), temperature=1e3)
    want = [0.0, -6e35, -3e35, -6e35]
    for a, b in zip(out.log_prob.tolist(), want):
        assert abs(a - b) <= 4 * U * abs(b)
