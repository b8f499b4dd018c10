"""AdamW (scacchi_adamw_step) with moments in 32 and in 8 bits, and the norm
of gradients, against their definitions in 64 bits.

Tolerances (U = 2^-24, a 32-bit rounding).  b and 1 - b are rounded once,
their products and the sum once each:

  first    3 U (|b1 m| + |(1 - b1) g|)     (a clipped g: U more for the factor, U for its product)
  second   4 U of itself (all terms positive, g^2 one rounding more, clipping 4 more)
  root     second's half and U
  update   lr / bc1 first / (root inv + eps): relative 2 U (size) + U (product) + root's + U (inv) + 2 U
           (product and sum) + 4 U (a division to 2 ulp), and first's
  weight   2 U |w| (decay and its product), the update's, and U of the result; then its type's rounding

What rounds by random bits (8-bit codes, bfloat16 with a key) is the floor of
x / q + r on the grid of q: it must lie between the floors for x - tol and x +
tol.
"""

import math

import numpy as np
import pytest
import torch

from oracle import oracle as O
from scacchi_b200 import _lib
from scacchi_b200.adamw import BLOCK, AdamW, gradient_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
KEY = np.array([7, 1234567], np.uint32)
SIZES = [1, 3, 255, 256, 257, 0, 1000, 4096, 4097, 9001, (7, 13), (5, 3, 11)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tensors(sizes, dtype, seed, scale, shift=0):
    """Tensors by name; with a shift, that many elements off a 16-byte boundary."""
    g, out = _gen(seed), {}
    for i, s in enumerate(sizes):
        shape = s if isinstance(s, tuple) else (s,)
        n = math.prod(shape)
        flat = torch.empty((n + shift,), dtype=DT[dtype], device="cuda")
        rows = torch.exp(torch.randn((), generator=g, device="cuda"))
        flat[shift:] = (scale * rows * torch.randn((n,), generator=g, device="cuda")).to(DT[dtype])
        out[f"t{i}"] = flat[shift:].view(shape)
    return out


def _flat(opt, tensors):
    out = torch.zeros(opt.first.shape, dtype=torch.float64, device="cuda")
    for name, view in opt.views(out).items():
        if tensors.get(name) is not None:
            view.copy_(tensors[name])
    return out


def _held(opt):
    mask = torch.zeros(opt.first.shape, dtype=torch.bool, device="cuda")
    for view in opt.views(mask).values():
        view.fill_(True)
    return mask


def _random16(key, step, size):
    words = O.split(O.fold_in(key, step), size // 4).astype(np.int64)
    w = torch.from_numpy(words).cuda()
    return torch.stack((w[:, 0] & 0xffff, w[:, 0] >> 16, w[:, 1] & 0xffff, w[:, 1] >> 16), -1).reshape(-1)


def _value(code, exponent, fraction_bits):
    """What unsigned codes stand for."""
    field = code >> fraction_bits
    t = (code & ((1 << fraction_bits) - 1)).double() / (1 << fraction_bits)
    y = torch.where(field > 0, (1 + t) * torch.exp2(field.double() - 14), t * 2.0 ** -13)
    scale = torch.exp2(exponent.double() - 127)
    return y * torch.where(exponent == 255, math.nan, scale).repeat_interleave(BLOCK)


def _moments64(opt):
    """(first, second) in 64 bits."""
    if opt.state_bits == 32:
        return opt.first.double(), opt.second.double()
    c, r = opt.first.long(), opt.second.long()
    m = _value(c & 0x7f, opt.first_exponent.long(), 3) * torch.where(c >= 0x80, -1.0, 1.0)
    return m, _value(r, opt.second_exponent.long(), 4) ** 2


def _between(got, x, tol, q, random):
    """Whether got (>= 0) is x on the grid of q, up where the random part reaches."""
    low = torch.floor((x - tol) / q + random).clamp(min=0) * q
    high = torch.floor((x + tol) / q + random) * q
    return bool(((got >= low) & (got <= high)).all())


def _check_codes(codes, exponent, x, tol, fraction_bits, random, never_zero):
    got = _value(codes, exponent.long(), fraction_bits)
    most = x.view(-1, BLOCK).amax(-1).clamp(min=2.0 ** -100)
    e = exponent.long() - 127
    near = (most / torch.exp2(torch.round(torch.log2(most))) - 1).abs() < 2.0 ** -20
    assert bool(((torch.floor(torch.log2(most)).long() == e) | near).all())
    scale = torch.exp2(e.double()).repeat_interleave(BLOCK)
    q = torch.exp2(torch.floor(torch.log2((x / scale).clamp(min=2.0 ** -13))) - fraction_bits) * scale
    if never_zero:
        smallest = scale * 2.0 ** (-13 - fraction_bits)
        raised = (x > 0) & (got == smallest)
        assert bool((got[x > tol] > 0).all())
        x, got, q, tol, random = (t[~raised] for t in (x, got, q, tol, random))
    assert _between(got, x, tol, q, random)


def _step_and_check(opt, weights, grads, *, lr, b1, b2, eps, decay, clip=None, key=None, **kw):
    """One step, held to the definition from the state that it began with."""
    have = {k: v for k, v in grads.items() if v is not None}
    mask = torch.zeros(opt.first.shape, dtype=torch.bool, device="cuda")
    for name, view in opt.views(mask).items():
        view.fill_(name in have)
    w, g = _flat(opt, weights), _flat(opt, have)
    m, v = _moments64(opt)
    wd = torch.zeros_like(w)
    for name, view in opt.views(wd).items():
        view.fill_(decay[name] if isinstance(decay, dict) else decay)
    old = [t.clone() for t in (opt.first, opt.second)]
    t = opt.steps() + 1
    norm = opt.step(grads, **kw)
    assert opt.steps() == t
    if clip is not None:
        want = torch.linalg.vector_norm(g)
        if "norm" not in kw:
            assert abs(float(norm) - float(want)) <= U * float(want) + 1e-45
        g = g * min(1.0, clip / max(float(norm), 1e-300))
    extra = 4 if clip is not None else 0
    m_tol = (3 + extra) * U * ((b1 * m).abs() + ((1 - b1) * g).abs()) + 2.0 ** -148
    m = b1 * m + (1 - b1) * g
    v_tol = (4 + 2 * extra) * U
    v = b2 * v + (1 - b2) * g * g
    root = v.sqrt()
    size, inv = lr / (1 - b1 ** t), 1 / math.sqrt(1 - b2 ** t)
    den = root * inv + eps
    update = size * m / den
    u_tol = update.abs() * (10 * U + v_tol / 2) + abs(size) * m_tol / den
    u_tol = torch.where(den > 0, u_tol, 0.0)
    w_new = (1 - lr * wd) * w - torch.where(den > 0, update, math.nan)
    w_tol = 2 * U * w.abs() + u_tol + U * w_new.abs() + 2.0 ** -148
    random = None if key is None else _random16(key, t, w.numel())
    got = _flat(opt, weights)
    held = _held(opt)
    assert torch.equal(got[held & ~mask], w[held & ~mask])
    for view, (name, tensor) in zip(opt.views(mask).values(), weights.items()):
        if not view.numel() or not bool(view.all()):
            continue
        part = lambda flat: opt.views(flat)[name].reshape(-1)
        x, tol, out = part(w_new), part(w_tol), part(got)
        fin = x.isfinite()
        assert torch.equal(out.isfinite(), fin)
        x, tol, out = x[fin], tol[fin], out[fin]
        if tensor.dtype == torch.float32:
            assert bool(((out - x).abs() <= tol).all()), float(((out - x).abs() / tol).max())
        elif key is None:
            assert bool(((out - x).abs() <= tol + x.abs() * 2.0 ** -8 + 2.0 ** -134).all())
        else:
            r = (part(random) * 0x85eb & 0xffff)[fin]
            q = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -126))) - 7)
            assert _between((out * x.sign()).clamp(min=0), x.abs(), tol, q, r.double() / 65536)
    if opt.state_bits == 32:
        assert bool(((opt.first.double() - m).abs() <= m_tol)[mask].all())
        assert bool(((opt.second.double() - v).abs() <= v_tol * v + 2.0 ** -148)[mask].all())
        assert torch.equal(opt.first[~mask], old[0][~mask]) and torch.equal(opt.second[~mask], old[1][~mask])
        return
    c = opt.first.long()
    u = random
    m_abs = torch.where(mask, m.abs(), 0.0)
    sign = torch.where(c >= 0x80, -1.0, 1.0)
    nonzero = (c & 0x7f) > 0
    assert bool((sign * m >= -m_tol)[mask & nonzero].all())
    whole = mask.view(-1, BLOCK)[:, 0].repeat_interleave(BLOCK)  # blocks of tensors with a gradient
    blocks = whole.view(-1, BLOCK)[:, 0]
    for codes, exponent, x, tol, bits, r, raised in (
            (c & 0x7f, opt.first_exponent, m_abs, m_tol, 3, u, False),
            (opt.second.long(), opt.second_exponent, torch.where(mask, root, 0.0), root * (v_tol / 2 + U), 4,
             u * 0x9e37 & 0xffff, True)):
        _check_codes(codes[whole], exponent[blocks], x[whole], tol[whole], bits, (r[whole].double() + 0.5) / 65536,
                     raised)
    assert torch.equal(opt.first[~whole], old[0][~whole]) and torch.equal(opt.second[~whole], old[1][~whole])


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("gradient", sorted(DT))
@pytest.mark.parametrize("weight", ["fp32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps(cuda, bits, weight, gradient, shift):
    weights = _tensors(SIZES, weight, 1, 0.1, shift)
    decay = {k: 0.1 * (i % 3) for i, k in enumerate(weights)}
    keys = [KEY] if bits == 8 or weight == "fp32" else [None, KEY]
    for key in keys:
        opt = AdamW(weights, learning_rate=0.01, weight_decay=decay, state_bits=bits, key=key)
        for step in range(4):
            grads = _tensors(SIZES, gradient, 10 + step, 1e-2, shift)
            if step == 2:
                grads["t3"] = grads["t8"] = None
            if step == 3:
                del grads["t9"]
                for g in grads.values():
                    if g is not None:
                        g.zero_()
            _step_and_check(opt, weights, grads, lr=0.01, b1=0.9, b2=0.999, eps=1e-8, decay=decay, key=key)


@pytest.mark.parametrize("gradient", sorted(DT))
def test_moments_are_bit_for_bit_those_of_plain_operations(cuda, gradient):
    """Every product and sum rounded by itself, so that what is rounded to a
    code is the definition's: two fused sums in a million codes differ."""
    w = _tensors([1 << 20], "fp32", 1, 0.1)
    opt = AdamW(w, learning_rate=0.01, beta1=0.9, beta2=0.999)
    eight = AdamW({"t0": w["t0"].clone()}, learning_rate=0.01, beta1=0.9, beta2=0.999, state_bits=8, key=KEY)
    for step in range(3):
        g = _tensors([1 << 20], gradient, 5 + step, 1e-2)
        x = g["t0"].float()
        first, second = opt.first * 0.9 + x * (1 - 0.9), opt.second * 0.999 + x * x * (1 - 0.999)
        m0, v0 = _moments64(eight)
        m = m0.float() * 0.9 + x * (1 - 0.9)
        root = torch.sqrt(v0.float() * 0.999 + x * x * (1 - 0.999))
        opt.step(g)
        eight.step(g)
        assert torch.equal(opt.first, first) and torch.equal(opt.second, second)
        random = _random16(KEY, step + 1, 1 << 20)
        for y, u, codes, exponent, shift in ((m.abs(), random, eight.first & 0x7f, eight.first_exponent, 20),
                                             (root, random * 0x9e37 & 0xffff, eight.second, eight.second_exponent, 19)):
            most = (y.view(-1, BLOCK).amax(-1).view(torch.int32) >> 23).clamp(27, 253)
            assert torch.equal(exponent.int(), most)
            unit = torch.exp2(127.0 - most.float()).repeat_interleave(BLOCK)
            bits = (y * unit * 2.0 ** -113).view(torch.int32).long()
            want = (bits + (u << shift - 16) + (1 << shift - 17)) >> shift
            if shift == 19:
                want = torch.maximum(want, (y > 0).long())
            assert torch.equal(codes.long(), want)


@pytest.mark.parametrize("bits", [32, 8])
def test_settings(cuda, bits):
    """Other betas, eps and rates, among them a rate given per step, as a number and on the device."""
    for i, (b1, b2, eps, lr) in enumerate(((0.0, 0.0, 1e-3, 0.5), (0.0, 0.95, 0.0, 1e-3), (0.99, 0.9999, 1e-6, -0.1),
                                           (0.5, 0.5, 1e-8, 0.0))):
        weights = _tensors([300, 5000], "fp32", i, 1.0)
        opt = AdamW(weights, learning_rate=7.0, beta1=b1, beta2=b2, eps=eps, weight_decay=0.01, state_bits=bits, key=KEY)
        for step, rate in enumerate((lr, torch.tensor(lr, device="cuda"), lr)):
            grads = _tensors([300, 5000], "fp32", 20 + step, 1.0)
            value = float(rate)  # as the device holds it
            _step_and_check(opt, weights, grads, lr=value, b1=b1, b2=b2, eps=eps, decay=0.01, key=KEY,
                            learning_rate=rate)


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping(cuda, bits):
    weights = _tensors(SIZES, "fp32", 1, 0.1)
    opt = AdamW(weights, learning_rate=0.01, max_norm=0.5, state_bits=bits, key=KEY)
    args = dict(lr=0.01, b1=0.9, b2=0.999, eps=1e-8, decay=0.0, clip=0.5, key=KEY)
    _step_and_check(opt, weights, _tensors(SIZES, "bf16", 2, 1.0), **args)  # clipped
    _step_and_check(opt, weights, _tensors(SIZES, "fp32", 3, 1e-5), **args)  # below the limit
    _step_and_check(opt, weights, _tensors(SIZES, "fp16", 4, 1e-2), norm=torch.tensor(40.0, device="cuda"), **args)
    assert opt.step({"t0": torch.zeros(1, device="cuda")}) is not None
    # a norm that is not finite: nothing moves
    for bad in (math.inf, math.nan):
        state = [t.clone() for t in (*weights.values(), opt.first, opt.second)]
        taken = opt.steps()
        grads = _tensors(SIZES, "fp32", 5, 1.0)
        grads["t6"][17] = bad
        norm = opt.step(grads)
        assert not math.isfinite(float(norm)) and opt.steps() == taken
        for a, b in zip(state, (*weights.values(), opt.first, opt.second)):
            assert torch.equal(a, b)
    _step_and_check(opt, weights, _tensors(SIZES, "bf16", 6, 1.0), **args)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes(cuda, bits):
    sizes = [1 + (37 * i) % 250 for i in range(1100)]
    key = KEY if bits == 8 else None
    weights = _tensors(sizes, "fp32", 1, 0.1)
    opt = AdamW(weights, learning_rate=0.01, max_norm=1.0, state_bits=bits, key=key)
    launches = _lib.lib().scacchi_adamw_launch_count()
    _step_and_check(opt, weights, _tensors(sizes, "bf16", 2, 0.1), lr=0.01, b1=0.9, b2=0.999, eps=1e-8, decay=0.0,
                    clip=1.0, key=key)
    assert _lib.lib().scacchi_adamw_launch_count() - launches == 3 + 1 + 1 + 3


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("weight", ["fp32", "bf16"])
def test_alignment_and_company_change_no_bit(cuda, bits, weight):
    """The same tensors alone, shifted and split over two optimisers of other launch shapes."""
    grads = [_tensors([5000, 300], "bf16", s, 0.1) for s in (5, 6, 7)]
    results = []
    for shift in (0, 1, 3):
        weights = _tensors([5000, 300], weight, 1, 0.1, 0)
        moved = {}
        for k, v in weights.items():
            flat = torch.empty((v.numel() + shift,), dtype=v.dtype, device="cuda")
            moved[k] = flat[shift:]
            moved[k].copy_(v)
        opt = AdamW(moved, learning_rate=0.01, state_bits=bits, key=KEY)
        for g in grads:
            opt.step(g)
        results.append([*moved.values(), opt.first, opt.second, opt.first_exponent, opt.second_exponent])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert a is None and b is None or torch.equal(a, b)


def test_strided_gradients_are_copied(cuda):
    w = {"a": torch.zeros((30, 40), device="cuda")}
    v = {"a": torch.zeros((30, 40), device="cuda")}
    g = torch.randn((40, 30), device="cuda")
    AdamW(w, learning_rate=0.1).step({"a": g.t()})
    AdamW(v, learning_rate=0.1).step({"a": g.t().contiguous()})
    assert torch.equal(w["a"], v["a"]) and bool(w["a"].any())
    assert float(gradient_norm([g.t()])) == float(gradient_norm([g.t().contiguous()]))


def test_moments_are_the_values_of_the_codes(cuda):
    """Every code under several exponents, exact in bfloat16."""
    w = {"a": torch.zeros((4 * BLOCK,), device="cuda")}
    opt = AdamW(w, learning_rate=0.1, state_bits=8, key=KEY)
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(4)
    first = torch.where(codes & 0x7f == 0x7f, codes - 1, codes)
    exponents = torch.tensor([27, 100, 127, 253], dtype=torch.uint8, device="cuda")
    opt.load_state_dict(dict(step=5, first=first, second=codes, first_exponent=exponents, second_exponent=exponents))
    m, v = _moments64(opt)
    got = opt.moments()
    assert got[0].dtype == got[1].dtype == torch.bfloat16
    assert torch.equal(got[0].double(), m) and torch.equal(got[1].double() ** 2, v)
    exponents[1] = 255
    opt.load_state_dict(dict(step=5, first=first, second=codes, first_exponent=exponents, second_exponent=exponents))
    for t in opt.moments():
        bad = t.isnan().view(4, BLOCK)
        assert bool(bad[1].all()) and not bool(bad[[0, 2, 3]].any())


def test_what_is_not_finite_stays_in_its_block(cuda):
    for bad in (math.inf, -math.inf, math.nan):
        w = {"a": torch.ones((1000,), device="cuda"), "b": torch.ones((10,), device="cuda")}
        opt = AdamW(w, learning_rate=0.1, state_bits=8, key=KEY)
        g = {"a": torch.ones((1000,), device="cuda"), "b": torch.ones((10,), device="cuda")}
        g["a"][300] = bad
        opt.step(g)
        assert opt.first_exponent.tolist()[1] == 255 and 255 not in opt.first_exponent[[0, 2, 3, 4]].tolist()
        opt.step({k: torch.ones_like(v) for k, v in g.items()})
        nan = w["a"].isnan()
        assert bool(nan[256:512].all()) and not bool(nan[:256].any()) and not bool(nan[512:].any())
        assert not bool(w["b"].isnan().any())
        # in 32 bits the element alone
        w = {"a": torch.ones((1000,), device="cuda")}
        AdamW(w, learning_rate=0.1).step({"a": g["a"]})
        assert int((~w["a"].isfinite()).sum()) == 1


def test_zero_gradients_leave_zero(cuda):
    for bits in (32, 8):
        w = {"a": torch.ones((700,), device="cuda")}
        opt = AdamW(w, learning_rate=0.1, state_bits=bits, key=KEY)
        for _ in range(3):
            opt.step({"a": torch.zeros((700,), device="cuda")})
        assert torch.equal(w["a"], torch.ones_like(w["a"]))
        assert not any(bool(t.any()) for t in opt.moments())


def test_small_changes_add_up_in_8_bits(cuda):
    """Roots under b2 = 0.999 without gradients fall by sqrt(0.999) a step on
    average.  A step moves a root by 5e-4 of itself, f = 0.008 to 0.016 of its
    code's step q = r / 16 to r / 32: the variance f (1 - f) q^2 is at most 5e-4
    r q < 3.2e-5 r^2 a step, over 200 steps less than (0.08 r)^2, and the mean
    of 2^18 of them is off by less than 6 x 0.08 / 512 = 9.4e-4 of r."""
    n = 1 << 18
    w = {"a": torch.zeros((n,), device="cuda")}
    opt = AdamW(w, learning_rate=0.0, beta2=0.999, state_bits=8, key=KEY)
    opt.step({"a": 1.0 + torch.rand((n,), device="cuda", generator=_gen(1))})
    start = opt.moments()[1].double()
    zero = torch.zeros((n,), device="cuda")
    for _ in range(200):
        opt.step({"a": zero})
    ratio = float(opt.moments()[1].double().sum() / start.sum())
    assert abs(ratio - 0.999 ** 100) < 9.4e-4


def test_bfloat16_weights_add_up_with_a_key(cuda):
    """Steps of 1e-3 of a weight's 2^-8: 100 of them move 2^18 weights by 0.1
    on average (each rounding's variance is at most f q^2, f = 1e-3 / 2^-7 =
    0.128: 100 steps (0.028)^2, the mean 6 x 0.028 / 512 = 3.3e-4), or not at
    all to nearest."""
    for key, moved in ((KEY, 0.1), (None, 0.0)):
        w = {"a": torch.full((1 << 18,), 1.0, device="cuda", dtype=torch.bfloat16)}
        opt = AdamW(w, learning_rate=1e-3, eps=0.0, key=key)
        g = {"a": -torch.ones((1 << 18,), device="cuda")}
        for _ in range(100):
            opt.step(g)
        assert abs(float(w["a"].double().mean()) - 1.0 - moved) < 3.3e-4


@pytest.mark.parametrize("bits", [32, 8])
def test_state_is_carried_on(cuda, bits):
    def run(interrupt):
        weights = _tensors([1000, 7], "bf16", 1, 0.1)
        opt = AdamW(weights, learning_rate=0.01, state_bits=bits, key=KEY)
        for s in range(6):
            if interrupt and s == 3:
                saved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state_dict().items()}
                opt = AdamW(weights, learning_rate=0.01, state_bits=bits, key=KEY)
                opt.load_state_dict(saved)
            opt.step(_tensors([1000, 7], "fp32", 30 + s, 0.1))
        return [*weights.values(), opt.first, opt.second]

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(cuda, bits):
    """A captured step with its own norm and a rate on the device, replayed,
    gives what eager steps give; on a stream of its own."""
    grads = _tensors(SIZES, "bf16", 2, 0.1)
    results = []
    for captured in (False, True):
        weights = _tensors(SIZES, "fp32", 1, 0.1)
        opt = AdamW(weights, learning_rate=1.0, max_norm=0.5, state_bits=bits, key=KEY)
        rate = torch.tensor(0.0, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            if captured:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    norm = opt.step(grads, learning_rate=rate)
            for s in range(5):
                rate.fill_(0.01 * (s + 1))
                if captured:
                    graph.replay()
                else:
                    norm = opt.step(grads, learning_rate=rate)
        side.synchronize()
        assert opt.steps() == 5
        results.append([norm, *weights.values(), opt.first, opt.second])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_plain_calls_and_the_python_way_agree(cuda, monkeypatch):
    """Steps, norms and moments through the extension module and without it."""
    class Nothing:
        @staticmethod
        def adamw_step(*args):
            return None

        gradient_norm = adamw_moments = adamw_step

    def run():
        res = []
        for bits in (32, 8):
            for clip in (None, 0.5):
                weights = _tensors(SIZES, "bf16", 1, 0.1)
                opt = AdamW(weights, learning_rate=0.01, weight_decay=0.1, max_norm=clip, state_bits=bits, key=KEY)
                grads = _tensors(SIZES, "fp32", 2, 0.1)
                grads["t4"] = None
                norms = [opt.step(grads), opt.step(dict(list(grads.items())[3:]), learning_rate=0.1)]
                if clip:
                    norms.append(opt.step(grads, norm=torch.tensor(9.0, device="cuda")))
                opt.step(grads, learning_rate=torch.tensor(0.03, device="cuda"))
                res += [*norms, *weights.values(), *opt.moments(), opt.first, opt.second, torch.tensor(opt.steps())]
                res.append(gradient_norm([g for g in grads.values() if g is not None]))
        return res

    fast = run()
    host = _lib.host()
    assert host.gradient_norm([torch.ones((3,), device="cuda")]) is not None
    monkeypatch.setattr(_lib, "host", lambda: Nothing)
    slow = run()
    assert len(fast) == len(slow)
    for a, b in zip(fast, slow):
        assert a is None and b is None or a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def test_a_large_tensor(cuda):
    """Many CTAs, on either side of chunks' and blocks' ends."""
    for n in (1 << 18, 300_001):
        for bits, dtype in ((32, "fp32"), (8, "bf16"), (8, "fp32")):
            weights = _tensors([n], dtype, 1, 0.1)
            opt = AdamW(weights, learning_rate=0.01, state_bits=bits, max_norm=1.0, key=KEY)
            for step in range(2):
                _step_and_check(opt, weights, _tensors([n], "bf16", 2 + step, 1e-2), lr=0.01, b1=0.9, b2=0.999, eps=1e-8,
                                decay=0.0, clip=1.0, key=KEY)


def test_offsets_past_32_bits(cuda):
    """One step of gradients of 1 over more than 2^31 weights of 0: the first
    moment is 0.1, the root sqrt(0.001), each on one of the codes beside it
    (1/8 and 1/16 of their binades), the weight -0.01 to bfloat16."""
    n = (1 << 31) + 5003
    w = {"a": torch.zeros((n,), dtype=torch.bfloat16, device="cuda")}
    g = {"a": torch.ones((n,), dtype=torch.bfloat16, device="cuda")}
    opt = AdamW(w, learning_rate=0.01, state_bits=8, key=KEY)
    assert abs(float(gradient_norm(g)) - math.sqrt(n)) <= U * math.sqrt(n)
    opt.step(g)
    first, root = opt.moments()
    for part in (slice(0, 5000), slice(n - 5003, n)):
        assert float((w["a"][part].double() + 0.01).abs().max()) <= 0.01 * 2.0 ** -7
        assert float((first[part].double() / 0.1 - 1).abs().max()) <= 1 / 8
        assert float((root[part].double() / math.sqrt(0.001) - 1).abs().max()) <= 1 / 16
        assert abs(float(first[part].double().mean()) - 0.1) < 1e-3  # (5000 of at most 1/16 x 0.1 each: 6 sigma 5e-4)
    assert not bool(first[n:].any()) and not bool(root[n:].any())


def test_backward_through_a_stepped_weight_is_refused(cuda):
    w = torch.ones((8,), device="cuda", requires_grad=True)
    loss = (w * w).sum()
    opt = AdamW({"w": w.detach()}, learning_rate=0.1)
    opt.step({"w": torch.ones((8,), device="cuda")})
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_refusals(cuda):
    w = torch.zeros((10, 10), device="cuda")
    for bad in (w.double(), w.half(), w.t()[:5], w[:, ::2]):
        with pytest.raises(ValueError):
            AdamW({"a": bad}, learning_rate=0.1)
    with pytest.raises(ValueError, match="share memory"):
        AdamW({"a": w[:6], "b": w[5:]}, learning_rate=0.1)
    with pytest.raises(ValueError):
        AdamW({"a": w, "b": torch.zeros(3)}, learning_rate=0.1)
    opt = AdamW({"a": w}, learning_rate=0.1)
    good = torch.ones((10, 10), device="cuda")
    for bad in (good[:9], good.double(), good.cpu(), good.view(100)):
        with pytest.raises(ValueError, match="gradient of a"):
            opt.step({"a": bad})
    with pytest.raises(ValueError, match="no such weights"):
        opt.step({"b": good})
    for bad in (w, opt.first[:100].view(10, 10), opt.second[156:].view(10, 10)):
        with pytest.raises(ValueError, match="overlap"):
            opt.step({"a": bad})
    with pytest.raises(ValueError, match="max_norm"):
        opt.step({"a": good}, norm=torch.ones((), device="cuda"))
    for bad in (torch.ones((), device="cuda", dtype=torch.float64), torch.ones(()), torch.ones((2,), device="cuda")):
        with pytest.raises(ValueError, match="learning_rate"):
            opt.step({"a": good}, learning_rate=bad)
        with pytest.raises(ValueError, match="norm"):
            AdamW({"a": w}, learning_rate=0.1, max_norm=1.0).step({"a": good}, norm=bad)
    with pytest.raises(ValueError, match="learning_rate"):
        opt.step({"a": good}, learning_rate=math.nan)
    with pytest.raises(ValueError, match="overlap"):
        opt.step({"a": good}, learning_rate=w[0, 0])
    assert opt.steps() == 0 and not bool(w.any())
    state = opt.state_dict()
    for bad in (dict(state, step=-1), dict(state, first=state["first"][:-1]), dict(state, second=state["second"].double()),
                {"step": 1}, dict(state, more=1)):
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
    with pytest.raises(ValueError, match="buffer"):
        opt.views(w)


def _check_norm(grads):
    got = gradient_norm(grads)
    assert got.dtype == torch.float32 and got.shape == ()
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert abs(float(got) - want) <= U * want * 1.001 + 2.0 ** -149
    return got


def test_norms(cuda):
    every = [t for i, d in enumerate(sorted(DT)) for shift in (0, 1, 5)
             for t in _tensors(SIZES, d, 10 * i + shift, 0.1, shift).values()]
    first = _check_norm(every)
    assert torch.equal(first, gradient_norm(dict(enumerate(every))))
    for t in every:
        if t.numel():
            _check_norm([t])
    _check_norm([torch.randn((n,), device="cuda") for n in [1 + i % 50 for i in range(1300)]])
    _check_norm([torch.randn((3_000_001,), device="cuda"), torch.randn((5_000_000,), device="cuda").bfloat16()])
    assert float(gradient_norm([torch.zeros((0,), device="cuda")])) == 0.0
    assert float(gradient_norm([torch.zeros((100,), device="cuda")])) == 0.0


def test_norms_keep_the_range(cuda):
    """Squares beyond 32 bits either way."""
    for scale in (1e20, 1e-25, 1e30):
        _check_norm([scale * torch.randn((1000,), device="cuda"), torch.zeros((5,), device="cuda")])
    _check_norm([torch.full((100,), 65504.0, device="cuda", dtype=torch.float16)])
    assert math.isinf(float(gradient_norm([torch.full((100,), 3e38, device="cuda")])))
    for bad in (math.inf, -math.inf, math.nan):
        for d in DT.values():
            g = torch.ones((5000,), device="cuda", dtype=d)
            g[4999] = bad
            assert not math.isfinite(float(gradient_norm([torch.ones((3,), device="cuda"), g])))


def test_norm_refusals(cuda):
    good = torch.ones((3,), device="cuda")
    for bad in ([good, good.cpu()], [good.double()], [good, good.int()]):
        with pytest.raises(ValueError):
            gradient_norm(bad)


def test_weights_that_changed_are_refused(cuda):
    """Moved to the CPU, of another size, type or layout: nothing is written."""
    good = torch.ones((10, 10), device="cuda")
    for change in (lambda t: t.cpu(), lambda t: t[:5], lambda t: t.bfloat16(), lambda t: t.t()):
        w, other = torch.zeros((10, 10), device="cuda"), torch.zeros((3,), device="cuda")
        opt = AdamW({"a": w, "b": other}, learning_rate=0.1)
        w.data = change(w.data)
        for grads in ({"a": good, "b": torch.ones((3,), device="cuda")}, {"b": torch.ones((3,), device="cuda")}):
            with pytest.raises(ValueError, match="a has changed its device, size, type or layout|gradient of a"):
                opt.step(grads)
        assert opt.steps() == 0 and not bool(other.any()) and not bool(w.any())
    # another storage on the same device is taken up
    opt = AdamW({"a": w.data.t()}, learning_rate=0.1)
    opt.weights["a"].data = torch.ones((10, 10), device="cuda")
    opt.step({"a": good})
    assert float(opt.weights["a"].max()) < 0.95


@pytest.mark.parametrize("gradient", ["fp32", "bf16"])
@pytest.mark.parametrize("weight", ["fp32", "bf16"])
def test_a_square_beyond_float32_is_an_infinite_root(cuda, weight, gradient):
    """A finite gradient whose square is infinite: its weight rests (m / inf
    is 0) while the root is infinite, and in 8 bits its block of roots is NaN
    from the next step on, and so are its weights."""
    for bits in (32, 8):
        w = {"a": torch.ones((1000,), device="cuda", dtype=DT[weight]), "b": torch.ones((10,), device="cuda")}
        opt = AdamW(w, learning_rate=1e-3, state_bits=bits, key=KEY)
        g = {"a": torch.ones((1000,), device="cuda", dtype=DT[gradient]), "b": torch.ones((10,), device="cuda")}
        g["a"][300] = 3e38
        opt.step(g)
        assert float(w["a"][300]) == 1.0 and bool(w["a"].isfinite().all())
        assert bool((w["a"].double() < 1.0 + 2.0 ** -24).all())
        if bits == 8:
            assert opt.second_exponent.tolist()[1] == 255 and 255 not in opt.first_exponent.tolist()
        else:
            assert math.isinf(float(opt.second[300])) and math.isfinite(float(opt.first[300]))
        opt.step({k: torch.ones_like(v) for k, v in g.items()})
        nan = w["a"].isnan()
        if bits == 8:
            assert bool(nan[256:512].all()) and not bool(nan[:256].any()) and not bool(nan[512:].any())
        else:
            assert not bool(nan.any()) and float(w["a"][300]) == 1.0
        assert not bool(w["b"].isnan().any())


def test_a_second_moment_that_is_no_number_shows_in_the_weight(cuda):
    """A NaN that was loaded, and with beta2 = 0 one of infinity times 0."""
    w = {"a": torch.ones((1000,), device="cuda")}
    opt = AdamW(w, learning_rate=1e-3)
    second = opt.second.clone()
    second[7] = math.nan
    opt.load_state_dict(dict(step=3, first=opt.first.clone(), second=second))
    opt.step({"a": torch.ones((1000,), device="cuda")})
    assert w["a"].isnan().nonzero().flatten().tolist() == [7]
    w = {"a": torch.ones((1000,), device="cuda")}
    opt = AdamW(w, learning_rate=1e-3, beta2=0.0)
    g = torch.ones((1000,), device="cuda")
    g[5] = 1e25
    opt.step({"a": g})
    assert bool(w["a"].isfinite().all())
    opt.step({"a": torch.ones((1000,), device="cuda")})
    assert w["a"].isnan().nonzero().flatten().tolist() == [5]


def test_the_largest_codes_keep_their_sign(cuda):
    """First moments at the end of float32's range: 1.875 x 2^127 and above
    would round to a code beyond the seven bits, and stay at the largest."""
    n = 4 * BLOCK
    w = {"a": torch.zeros((n,), device="cuda")}
    opt = AdamW(w, learning_rate=0.0, beta1=0.0, state_bits=8, key=KEY)
    g = torch.full((n,), 3.3e38, device="cuda")
    g[BLOCK:2 * BLOCK] = torch.finfo(torch.float32).max
    g[2 * BLOCK:] = 1.75 * 2.0 ** 127
    g[::3] *= -1
    opt.step({"a": g})
    assert opt.first_exponent.tolist() == [253] * 4
    want = torch.where(g < 0, 0xfe, 0x7e).to(torch.uint8)
    assert torch.equal(opt.first, want)
    assert torch.equal(opt.moments()[0].double(), g.sign().double() * 1.75 * 2.0 ** 127)


def _order_shows(dtype):
    """Values whose squares' sum lies on a border of float32: 1 + 2^-23 +
    2^-48 is the square of the middle between 1 and the next number, and 24
    squares of 2^-54 count only where they meet each other before the 1."""
    x = torch.zeros((8192,), dtype=torch.float32)
    x[0], x[1001], x[2001], x[3001] = 1.0, 2.0 ** -12, 2.0 ** -12, 2.0 ** -24
    tiny = [i for i in range(256, 8192, 256) if i % (4096 // dtype.itemsize)]
    x[tiny] = 2.0 ** -27
    return x.to(dtype).cuda()


def _shifted(x, shift):
    flat = torch.empty((x.numel() + shift,), dtype=x.dtype, device="cuda")
    flat[shift:] = x
    return flat[shift:]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norms_do_not_depend_on_alignment(cuda, dtype):
    x = _order_shows(dtype)
    want = gradient_norm([x])
    for shift in range(1, 16 // x.element_size()):
        assert torch.equal(gradient_norm([_shifted(x, shift)]), want)
    # nor a step's own norm on where the weights lie
    for shift in (0, 1):
        w = _shifted(torch.zeros((8192,), device="cuda"), shift)
        assert torch.equal(AdamW({"w": w}, learning_rate=0.1, max_norm=1.0).step({"w": x}), want)


@pytest.mark.parametrize("plain", [True, False])
def test_backward_through_a_weight_that_was_not_stepped(cuda, plain):
    """A weight without a gradient stays as it is, and so does a graph that it is in."""
    a, b, c = (torch.ones((8,), device="cuda", requires_grad=True) for _ in range(3))
    loss, other = (b * b).sum() + (c * c).sum(), (a * a).sum()
    opt = AdamW({"a": a.detach(), "b": b.detach(), "c": c.detach()}, learning_rate=0.1)
    g = torch.ones((8,), device="cuda") if plain else torch.ones((16,), device="cuda")[::2]
    opt.step({"a": g, "c": None})
    loss.backward()
    assert torch.equal(b.grad, torch.full((8,), 2.0, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        other.backward()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("weight", ["fp32", "bf16"])
def test_launches_of_any_shape_change_no_bit(cuda, bits, weight):
    """Two tensors beside 0, 40 and 600 others (tables of each size, the last
    in two launches), stepped with them, each alone (the others without a
    gradient), and with gradients off their boundaries."""
    sizes = [5000, 300]
    grads = [_tensors(sizes, "bf16", s, 0.1) for s in (5, 6)]

    def run(more, alone=(None,), shift=0):
        others = {f"o{i}": torch.ones((1 + 7 * i % 500,), device="cuda") for i in range(more)}
        got = {}
        for name in alone:
            weights = {**_tensors(sizes, weight, 1, 0.1), **{k: v.clone() for k, v in others.items()}}
            opt = AdamW(weights, learning_rate=0.01, state_bits=bits, key=KEY)
            for g in grads:
                given = {k: _shifted(v.reshape(-1), shift) for k, v in g.items() if name in (None, k)}
                opt.step(given if name else {**given, **others})
            for k in [name] if name else ["t0", "t1"]:
                parts = [opt.views(opt.first)[k], opt.views(opt.second)[k], weights[k]]
                if bits == 8:
                    row = opt._table[opt._names.index(k)]
                    at = slice(int(row["offset"]) // BLOCK, -(-int(row["offset"] + row["count"]) // BLOCK))
                    parts += [opt.first_exponent[at], opt.second_exponent[at]]
                got[k] = [p.clone() for p in parts]
        return got

    want = run(0)
    for other in (run(40), run(600), run(0, ("t0", "t1")), run(600, ("t0", "t1")), run(0, shift=1), run(40, shift=5)):
        for k, parts in want.items():
            for a, b in zip(parts, other[k]):
                assert torch.equal(a, b)
