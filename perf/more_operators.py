"""Workloads of the operators around a policy step: log-probabilities of
played actions with entropy and best alternatives, their gradient in the
logits, the norm of a whole network's gradients, and an AdamW step over many
tensors with moments in 32 or in 8 bits.

``listed`` gives the fixed cases, ``draw`` more of the same ranges,
``prepare`` a case's inputs, ``run`` one pass (plain torch operations, or
the package's operators where ``own`` is set), ``exact`` the same outputs
in 64 bits and ``work`` what a pass cannot do without.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"

LEARNING_RATE, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
MAX_NORM = 1.0
BLOCK = 256  # elements that share an exponent where moments have 8 bits


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _rows(op, rows, actions, dtype, legal, temperature, top):
    return dict(op=op, rows=rows, actions=actions, dtype=dtype, legal=legal, temperature=temperature, top=top)


def _norm(layout, layers, rows, cols, gradient):
    return dict(op="norm", layout=layout, layers=layers, rows=rows, cols=cols, gradient=gradient)


def _adamw(layout, layers, rows, cols, weight, gradient, bits, clip):
    return dict(op="adamw", layout=layout, layers=layers, rows=rows, cols=cols, weight=weight, gradient=gradient,
                bits=bits, clip=clip)


def listed():
    return [
        # one frame of a small self-play batch (64 games of 9x9 Hex): latency
        dict(_rows("log_probs", 64, 82, "fp32", True, 1.0, 5), name="log_probs_frame64_hex9"),
        # 8192 lanes x 32 frames of 9x9 Hex: the behaviour policy's log-probs and the next best moves
        dict(_rows("log_probs", 8192 * 32, 82, "fp32", True, 1.0, 4), name="log_probs_frames8192x32_hex9"),
        # token rows over a generic vocabulary, twenty alternatives each
        dict(_rows("log_probs", 4096, 32000, "bf16", False, 1.0, 20), name="log_probs_vocab32000_bf16"),
        # a few rows over a large odd vocabulary, sampled at a temperature: one step of serving
        dict(_rows("log_probs", 8, 131071, "fp32", False, 0.7, 20), name="log_probs_vocab131071_rows8"),
        # the frames' gradient of a policy gradient with an entropy bonus
        dict(_rows("gradient", 8192 * 32, 82, "fp32", True, 1.0, 0), name="gradient_frames8192x32_hex9"),
        # the same over token rows in 16 bits
        dict(_rows("gradient", 4096, 32000, "bf16", False, 1.0, 0), name="gradient_vocab32000_bf16"),
        # every gradient of the 6x128 network (73 tensors): latency
        dict(_norm("network", 6, 128, 82, "fp32"), name="norm_network6x128"),
        # sixteen square layers' 16-bit gradients with their biases and scales
        dict(_norm("layers", 16, 2048, 2048, "bf16"), name="norm_layers16x2048_bf16"),
        # what orthogonalised updates leave of the 6x128 network (66 small tensors): latency
        dict(_adamw("network", 6, 128, 82, "fp32", "fp32", 32, False), name="adamw_network6x128"),
        # twelve wide layers in 32 bits throughout, gradients clipped by their norm
        dict(_adamw("layers", 12, 1024, 4096, "fp32", "fp32", 32, True), name="adamw_layers12x1024x4096"),
        # sixteen square layers of 16-bit weights and gradients, moments in 8 bits
        dict(_adamw("layers", 16, 2048, 2048, "bf16", "bf16", 8, True), name="adamw8_layers16x2048_bf16"),
        # a ragged stack: 32-bit weights, 16-bit gradients, moments in 8 bits
        dict(_adamw("layers", 3, 257, 1001, "fp32", "bf16", 8, False), name="adamw8_ragged3x257x1001"),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["log_probs", "log_probs", "gradient", "norm", "adamw", "adamw"])
    if op in ("log_probs", "gradient"):
        actions = _between(rng, 2, 131072)
        rows = _between(rng, 1, max(1, min(1 << 18, (1 << 26) // actions)))
        top = rng.choice([0, rng.randint(1, 32)]) if op == "log_probs" else 0
        return _rows(op, rows, actions, rng.choice(sorted(DTYPES)), rng.random() < 0.5,
                     rng.choice([1.0, round(rng.uniform(0.3, 2.0), 2)]), top)
    rows, cols = _between(rng, 1, 4096), _between(rng, 1, 4096)
    layers = _between(rng, 1, max(1, min(20, (1 << 25) // (rows * cols))))
    gradient = rng.choice(sorted(DTYPES))
    if op == "norm":
        return _norm("layers", layers, rows, cols, gradient)
    return _adamw("layers", layers, rows, cols, rng.choice(["fp32", "bf16"]), gradient, rng.choice([32, 8]),
                  rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(1000003 * (seed % (1 << 31)) + salt)
    return g


def _prepare_rows(case, seed):
    """Rows as self-play and sampling leave them: logits with a few strong
    actions, the legal ones, the action that the policy drew.  Where there is
    a mask one row in 64 has ended: no legal action, no action played."""
    N, A, T = case["rows"], case["actions"], case["temperature"]
    g = _gen(seed, 1)
    logits = torch.randn((N, A), generator=g, device=DEVICE).mul_(2.0).to(DTYPES[case["dtype"]])
    legal = ended = None
    if case["legal"]:
        legal = torch.rand((N, A), generator=g, device=DEVICE) < 0.7
        legal[:, 0] |= ~legal.any(-1)
        ended = torch.rand(N, generator=g, device=DEVICE) < 1 / 64
        legal &= ~ended[:, None]
    x = logits.float() / T
    if legal is not None:
        x.masked_fill_(~legal, -math.inf)
    noise = torch.rand((N, A), generator=g, device=DEVICE).clamp_(min=1e-12).log_().neg_().log_().neg_()
    action = (x + noise).argmax(-1).to(torch.int32)
    del noise, x
    if ended is not None:
        action.masked_fill_(ended, -1)
    state = dict(case=case, logits=logits, legal=legal, action=action)
    if case["op"] == "gradient":
        # what the forward pass left, and the gradients of a policy-gradient loss with an entropy bonus
        x = logits.double()
        if legal is not None:
            x.masked_fill_(~legal, -math.inf)
        top = x.amax(-1)
        u = torch.where(x > -math.inf, (x - top[:, None]) / T, -math.inf)
        e = u.exp()
        z = e.sum(-1)
        state["max_logit"], state["log_sum"] = top.float(), z.log().float()
        mean = torch.where(e > 0, e * u, 0.0).sum(-1) / z
        state["entropy"] = torch.where(z > 0, z.log() - mean, 0.0).float()
        state["grad_log_prob"] = torch.randn(N, generator=g, device=DEVICE) / N
        state["grad_entropy"] = torch.full((N,), -0.01 / N, device=DEVICE)
    return state


def _shapes(case):
    """The tensors' shapes by name, in order."""
    L, R, C = case["layers"], case["rows"], case["cols"]
    if case["layout"] == "layers":
        return {f"{i}.{k}": s for i in range(L)
                for k, s in (("matrix", (R, C)), ("bias", (C,)), ("scale", (R,)))}
    # the residual network of L blocks, R channels and C actions on an 81-point board
    bn = lambda name, n: {f"{name}.scale": (n,), f"{name}.bias": (n,)}  # noqa: E731
    out = {"conv_w": (3, 3, 4, R), "conv_b": (R,)}
    for i in range(L):
        for k in "12":
            out |= {**bn(f"{i}.bn{k}", R), f"{i}.conv{k}_b": (R,)}
    out |= bn("bn", R)
    for head, planes, hidden in (("policy", 2, C), ("value", 1, R), ("q_dir", 2, R), ("q_conc", 1, R)):
        out |= {f"{head}_conv_w": (1, 1, R, planes), f"{head}_conv_b": (planes,), **bn(f"{head}_bn", planes),
                f"{head}_b": (hidden,)}
    out |= {"value_dir_w": (R, 2), "value_dir_b": (2,), "value_conc_w": (R, 1), "value_conc_b": (1,),
            "q_dir_out_b": (2 * C,), "q_conc_out_b": (C,)}
    if case["op"] == "norm":
        out |= {"convs": (2 * L, 9 * R, R), "policy_w": (162, C), "value_w": (81, R), "q_dir_w": (162, R),
                "q_dir_out_w": (R, 2 * C), "q_conc_w": (81, R), "q_conc_out_w": (R, C)}
    return out


def _flat(case):
    """(name, shape, offset) of each tensor in a flat buffer whose tensors
    begin at whole blocks, and the buffer's size."""
    at, out = 0, []
    for name, shape in _shapes(case).items():
        out.append((name, shape, at))
        at += -(-math.prod(shape) // BLOCK) * BLOCK
    return out, at


def _views(case, flat):
    return {name: flat[at:at + math.prod(shape)].view(shape) for name, shape, at in _flat(case)[0]}


def _gradients(case, g):
    """A bucket of gradients: each tensor at a scale of its own, rows at theirs."""
    flat = torch.zeros(_flat(case)[1], device=DEVICE)
    for view in _views(case, flat).values():
        view.normal_(generator=g)
        scale = torch.randn(view.shape[:1] + (1,) * (view.dim() - 1), generator=g, device=DEVICE)
        view.mul_(scale.mul_(0.5).exp_()).mul_(3e-4)
    return flat.to(DTYPES[case["gradient"]])


def _prepare_adamw(case, seed):
    g = _gen(seed, 3)
    tensors, size = _flat(case)
    state = dict(case=case, gradient=_gradients(case, g), step=100, key=(seed & 0xffffffff, 0x5cacc41))
    state["gradients"] = _views(case, state["gradient"])
    weight = torch.zeros(size, device=DEVICE)
    inside = torch.zeros(size, dtype=torch.bool, device=DEVICE)
    decay = torch.ones(size, device=DEVICE)
    for name, shape, at in tensors:
        n = math.prod(shape)
        weight[at:at + n].normal_(generator=g).mul_(0.02)
        inside[at:at + n] = True
        if len(shape) > 1:  # matrices alone
            decay[at:at + n] = 1.0 - LEARNING_RATE * DECAY
    state["weight"] = weight.to(DTYPES[case["weight"]])
    state["weights"] = _views(case, state["weight"])
    state["decay"] = decay
    # moments after a hundred steps
    size_of = state["gradient"].abs().amax().float()
    first = torch.randn(size, generator=g, device=DEVICE) * (0.2 * size_of) * inside
    second = torch.rand(size, generator=g, device=DEVICE).square() * (0.1 * size_of) ** 2 * inside
    if case["bits"] == 32:
        moments = dict(first=first, second=second)
    else:
        exponents = []
        for x in (first, second.sqrt()):
            top = x.view(-1, BLOCK).abs().amax(-1)
            exponents.append(((top.view(torch.int32) >> 23).clamp(27, 253)).to(torch.uint8))
        codes = [torch.randint(0, 0x70, (size,), generator=g, device=DEVICE, dtype=torch.uint8) * inside,
                 torch.randint(1, 0xe0, (size,), generator=g, device=DEVICE, dtype=torch.uint8) * inside]
        codes[0] |= (torch.rand(size, generator=g, device=DEVICE) < 0.5).to(torch.uint8) * 0x80 * (codes[0] > 0)
        moments = dict(first=codes[0], second=codes[1], first_exponent=exponents[0], second_exponent=exponents[1])
    state["moments"] = moments
    if own:  # the handle that a training loop keeps from step to step
        from scacchi_b200.adamw import AdamW

        state["optimizer"] = AdamW(
            state["weights"], learning_rate=LEARNING_RATE, beta1=BETA1, beta2=BETA2, eps=EPS,
            weight_decay={name: DECAY if len(shape) > 1 else 0.0 for name, shape, _ in tensors},
            max_norm=MAX_NORM if case["clip"] else None, state_bits=case["bits"], key=state["key"])
        state["optimizer"].load_state_dict(dict(step=state["step"], **moments))
    return state


def prepare(case, seed):
    if case["op"] in ("log_probs", "gradient"):
        return _prepare_rows(case, seed)
    if case["op"] == "norm":
        flat = _gradients(case, _gen(seed, 2))
        return dict(case=case, gradient=flat, gradients=list(_views(case, flat).values()))
    return _prepare_adamw(case, seed)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _scaled(s):
    """(logits in 32 bits, which count, their largest, (x - largest) / T)."""
    x = s["logits"].float()
    keep = x != -math.inf
    if s["legal"] is not None:
        keep &= s["legal"]
    x = torch.where(keep, x, -math.inf)
    top = x.amax(-1)
    base = torch.where(top == -math.inf, 0.0, top)
    return x, keep, top, (x - base[:, None]) / s["case"]["temperature"]


def _plain_log_probs(s):
    A, k = s["logits"].shape[-1], s["case"]["top"]
    x, keep, largest, u = _scaled(s)
    e = torch.exp(u)
    z = e.sum(-1)
    log_z = torch.log(z.double())
    action = s["action"].long()
    inside = (action >= 0) & (action < A)
    chosen = u.gather(-1, action.clamp(0, A - 1)[:, None])[:, 0].double()
    log_prob = torch.where(chosen == -math.inf, chosen, chosen - log_z)
    mean = (e * torch.where(keep, u, 0.0)).sum(-1) / z
    out = dict(log_prob=torch.where(inside, log_prob, 0.0).float(),
               entropy=torch.where(z > 0, log_z - mean, 0.0).float(), max_logit=largest, log_sum=log_z.float())
    if k:
        # by value and, among equal ones, by the lower index: both in one whole number
        bits = (x + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7fffffff)).long()
        column = torch.arange(A, device=x.device)
        order = torch.where(keep, (order << 32) | (0x7fffffff - column), -(1 << 63))
        n = min(k, A)
        best = torch.topk(order, n, -1).values
        at = 0x7fffffff - (best & 0x7fffffff)
        found = best != -(1 << 63)
        value = (u.gather(-1, torch.where(found, at, 0)).double() - log_z[:, None]).float()
        out["top_action"] = torch.full((x.shape[0], k), -1, dtype=torch.int32, device=x.device)
        out["top_log_prob"] = torch.full((x.shape[0], k), -math.inf, device=x.device)
        out["top_action"][:, :n] = torch.where(found, at, -1).to(torch.int32)
        out["top_log_prob"][:, :n] = torch.where(found, value, -math.inf)
    return out


def _plain_gradient(s):
    A, T = s["logits"].shape[-1], s["case"]["temperature"]
    x, keep, _, u = _scaled(s)
    log_p = torch.where(keep, u - s["log_sum"][:, None], 0.0)
    p = torch.where(keep, torch.exp(log_p), 0.0)
    action = s["action"].long()
    at = action.clamp(0, A - 1)[:, None]
    counts = (action >= 0) & (action < A) & keep.gather(-1, at)[:, 0]
    slope = torch.where(counts, s["grad_log_prob"], 0.0)
    grad = -p * (slope[:, None] + s["grad_entropy"][:, None] * (log_p + s["entropy"][:, None]))
    grad.scatter_add_(-1, at, slope[:, None])
    return (grad / T).to(s["logits"].dtype)


def _plain_norm(flat):
    return torch.sqrt(flat.double().square().sum()).float()


M32 = 0xffffffff


def _mix(x0, x1, rotations):
    for r in rotations:
        x0 = (x0 + x1) & M32
        x1 = (((x1 << r) | (x1 >> (32 - r))) & M32) ^ x0
    return x0, x1


def _threefry(key, c0, c1):
    """Threefry-2x32 of 20 rounds on counters held in 64 bits."""
    a, b = (13, 15, 26, 6), (17, 29, 16, 24)
    k0, k1 = key
    k2 = k0 ^ k1 ^ 0x1BD11BDA
    x0, x1 = _mix((c0 + k0) & M32, (c1 + k1) & M32, a)
    x0, x1 = _mix((x0 + k1) & M32, (x1 + k2 + 1) & M32, b)
    x0, x1 = _mix((x0 + k2) & M32, (x1 + k0 + 2) & M32, a)
    x0, x1 = _mix((x0 + k0) & M32, (x1 + k1 + 3) & M32, b)
    x0, x1 = _mix((x0 + k1) & M32, (x1 + k2 + 4) & M32, a)
    return (x0 + k2) & M32, (x1 + k0 + 5) & M32


def _random16(key, step, size):
    """Sixteen random bits for each element: a group of four shares the two
    words of its counter, low half first, under the key folded with the step."""
    q = torch.arange(size // 4, device=DEVICE)
    w0, w1 = _threefry(_threefry(key, 0, step), q >> 32, q & M32)
    return torch.stack((w0 & 0xffff, w0 >> 16, w1 & 0xffff, w1 >> 16), -1).reshape(-1).to(torch.int32)


def _power(exponent, size):
    """2^exponent of each block, an element each."""
    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32).repeat_interleave(BLOCK)[:size]


def _decoded(moments):
    """The first moment and the second's root that 8-bit moments stand for:
    both unsigned floats below a block's exponent, of 3 and 4 fraction bits."""
    first, second = moments["first"].to(torch.int32), moments["second"].to(torch.int32)
    n = first.numel()
    mag = (((first & 0x7f) << 20).view(torch.float32) * 2.0 ** 113
           * _power(moments["first_exponent"].to(torch.int32) - 127, n))
    root = ((second << 19).view(torch.float32) * 2.0 ** 113
            * _power(moments["second_exponent"].to(torch.int32) - 127, n))
    return torch.where(first >= 0x80, -mag, mag), root


def _encode(x, random, shift):
    """(codes, exponents) of nonnegative values: the block's largest in the
    binade of exponent 14, dropped bits rounded up where the random ones reach."""
    exponent = (x.view(-1, BLOCK).amax(-1).view(torch.int32) >> 23).clamp(27, 253) - 127
    y = x * _power(-exponent, x.numel()) * 2.0 ** -113
    drop = shift - 16
    code = (y.view(torch.int32) + (random << drop) + (1 << (drop - 1))) >> shift
    return code, (exponent + 127).to(torch.uint8)


def _plain_adamw(s):
    case, moments = s["case"], s["moments"]
    s["step"] += 1
    g = s["gradient"].float()
    if case["clip"]:
        norm = _plain_norm(s["gradient"])
        g = g * (MAX_NORM / norm.double().clamp(min=MAX_NORM)).float()
    eight = case["bits"] == 8
    random = None
    if eight or case["weight"] == "bf16":
        random = _random16(s["key"], s["step"], g.numel())
    m, v = moments["first"], moments["second"]
    if eight:
        m, root = _decoded(moments)
        v = root * root
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    root = torch.sqrt(v)
    if eight:
        code, exponent = _encode(m.abs(), random, 20)
        moments["first"].copy_(code.clamp(max=0x7e) | torch.where(m < 0, 0x80, 0))
        moments["first_exponent"].copy_(exponent)
        code, exponent = _encode(root, random * 0x9e37 & 0xffff, 19)
        moments["second"].copy_(torch.maximum(code, (root > 0).to(torch.int32)).clamp(max=0xff))
        moments["second_exponent"].copy_(exponent)
    else:
        moments["first"].copy_(m)
        moments["second"].copy_(v)
    size = LEARNING_RATE / (1 - BETA1 ** s["step"])
    w = s["weight"].float() * s["decay"] - size * m / (root / math.sqrt(1 - BETA2 ** s["step"]) + EPS)
    if case["weight"] == "bf16":
        w = (w.view(torch.int32) + (random * 0x85eb & 0xffff) & -65536).view(torch.float32)
    s["weight"].copy_(w)
    out = dict(weight=s["weight"])
    if eight:  # as the 16-bit values that the codes stand for, without rounding
        m, root = _decoded(moments)
        return dict(out, first=m.to(torch.bfloat16), root=root.to(torch.bfloat16))
    return dict(out, first=moments["first"], second=moments["second"])


def _own_rows(s):
    from scacchi_b200.log_probs import LogProbs, policy_log_probs, policy_log_probs_gradient

    case = s["case"]
    if case["op"] == "log_probs":
        out = policy_log_probs(s["logits"], s["action"], legal=s["legal"], temperature=case["temperature"],
                               top=case["top"])
        return {k: v for k, v in out._asdict().items() if v is not None}
    out = LogProbs(None, s["entropy"], s["max_logit"], s["log_sum"])
    return policy_log_probs_gradient(s["logits"], s["action"], out, grad_log_prob=s["grad_log_prob"],
                                     grad_entropy=s["grad_entropy"], legal=s["legal"],
                                     temperature=case["temperature"])


def run(state):
    op = state["case"]["op"]
    if own:
        if op in ("log_probs", "gradient"):
            return _own_rows(state)
        if op == "norm":
            from scacchi_b200.adamw import gradient_norm

            return gradient_norm(state["gradients"])
        optimizer = state["optimizer"]
        optimizer.step(state["gradients"])
        out = dict(weight=state["weight"])
        if state["case"]["bits"] == 8:
            first, root = optimizer.moments()
            return dict(out, first=first, root=root)
        return dict(out, first=optimizer.first, second=optimizer.second)
    if op == "log_probs":
        return _plain_log_probs(state)
    if op == "gradient":
        return _plain_gradient(state)
    if op == "norm":
        return _plain_norm(state["gradient"])
    return _plain_adamw(state)


# ---------------------------------------------------------------------------
# work and the 64-bit values
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] in ("log_probs", "gradient"):
        N, A = case["rows"], case["actions"]
        size = DTYPES[case["dtype"]].itemsize
        if case["op"] == "log_probs":
            return {"bytes": N * (A * (size + case["legal"]) + 4 + 4 * 4 + 8 * case["top"]), "flops": 6 * N * A}
        return {"bytes": N * (A * (2 * size + case["legal"]) + 4 + 5 * 4), "flops": 7 * N * A}
    n = sum(math.prod(s) for s in _shapes(case).values())
    size = DTYPES[case["gradient"]].itemsize
    if case["op"] == "norm":
        return {"bytes": n * size + 4, "flops": 2 * n}
    cell = size + 2 * DTYPES[case["weight"]].itemsize
    # moments read and written; those of 8 bits come with an exponent a block, and are given back as 16-bit values
    cell += 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4
    return {"bytes": n * cell, "flops": 14 * n}


def _exact_rows(s):
    """From the log-softmax of the kept actions."""
    case = s["case"]
    N, A = s["logits"].shape
    T, k = case["temperature"], case["top"]
    x = s["logits"].double()
    if s["legal"] is not None:
        x = x.masked_fill(~s["legal"], -math.inf)
    empty = (x == -math.inf).all(-1)
    logp = torch.log_softmax(torch.where(empty[:, None], 0.0, x / T), -1)
    logp = torch.where(x == -math.inf, -math.inf, logp)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(-1)
    action = s["action"].long()
    played = (action >= 0) & (action < A)
    if case["op"] == "gradient":
        # d/dx of g log p_a + h H, by the chain over log p: (g_i - p_i sum g) / T
        h = s["grad_entropy"].double()[:, None]
        up = torch.where(p > 0, -h * (p + plogp), 0.0)
        up.scatter_add_(-1, action.clamp(0, A - 1)[:, None],
                        torch.where(played, s["grad_log_prob"].double(), 0.0)[:, None])
        return (up - p * up.sum(-1, keepdim=True)) / T
    lp = logp.gather(-1, action.clamp(0, A - 1)[:, None])[:, 0]
    top = x.amax(-1)
    lse = torch.logsumexp(torch.where(empty[:, None], 0.0, x / T), -1)
    out = dict(log_prob=torch.where(played, lp, 0.0), entropy=entropy, max_logit=top,
               log_sum=torch.where(empty, -math.inf, lse - top / T))
    if k:
        order = torch.sort(x, dim=-1, descending=True, stable=True)
        n = min(k, A)
        found = order.values[:, :n] > -math.inf
        out["top_action"] = torch.full((N, k), -1, dtype=torch.int32, device=x.device)
        out["top_log_prob"] = torch.full((N, k), -math.inf, dtype=torch.float64, device=x.device)
        out["top_action"][:, :n] = torch.where(found, order.indices[:, :n], -1).to(torch.int32)
        out["top_log_prob"][:, :n] = torch.where(found, logp.gather(-1, order.indices[:, :n]), -math.inf)
    return out


def _exact_value(code, exponent, fraction_bits):
    """An 8-bit code's value: fields of an exponent and a fraction, the
    exponent 14 of a block being the binade of its largest element."""
    field, fraction = code >> fraction_bits, (code & ((1 << fraction_bits) - 1)).double() / (1 << fraction_bits)
    unit = torch.where(field > 0, (1.0 + fraction) * torch.exp2(field.double() - 14), fraction * 2.0 ** -13)
    return unit * torch.exp2(exponent.double() - 127).repeat_interleave(BLOCK)


def _exact_rounded(x, random, fraction_bits):
    """x >= 0 on the grid of its block, up where the random bits say."""
    e = torch.floor(torch.log2(x.view(-1, BLOCK).amax(-1).clamp(min=2.0 ** -100)))
    scale = torch.exp2(e).repeat_interleave(BLOCK)
    y = x / scale
    quantum = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -13))) - fraction_bits)
    return torch.floor(y / quantum + (random.double() + 0.5) / 65536) * quantum * scale, scale * 2.0 ** -13


def _exact_adamw(s):
    case, moments = s["case"], s["moments"]
    t = s["step"] + 1
    g = s["gradient"].double()
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        g = g * torch.clamp(MAX_NORM / norm, max=1.0)
    eight = case["bits"] == 8
    if eight:
        first = moments["first"].to(torch.int32)
        m = _exact_value(first & 0x7f, moments["first_exponent"], 3) * torch.where(first >= 0x80, -1.0, 1.0)
        v = _exact_value(moments["second"].to(torch.int32), moments["second_exponent"], 4) ** 2
    else:
        m, v = moments["first"].double(), moments["second"].double()
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g ** 2 - v)
    m_hat, v_hat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    w = s["weight"].double()
    # the decoupled decay of matrices
    w = w - torch.where(s["decay"] < 1, LEARNING_RATE * DECAY, 0.0) * w
    w = w - LEARNING_RATE * m_hat / (v_hat.sqrt() + EPS)
    random = _random16(s["key"], t, g.numel()) if eight or case["weight"] == "bf16" else None
    if case["weight"] == "bf16":
        quantum = torch.exp2(torch.floor(torch.log2(w.abs().clamp(min=2.0 ** -126))) - 7)
        w = w.sign() * torch.floor(w.abs() / quantum + (random * 0x85eb & 0xffff).double() / 65536) * quantum
    if not eight:
        return dict(weight=w, first=m, second=v)
    size, _ = _exact_rounded(m.abs(), random, 3)
    root, smallest = _exact_rounded(v.sqrt(), random * 0x9e37 & 0xffff, 4)
    root = torch.where(v > 0, torch.maximum(root, smallest / 16), root)
    return dict(weight=w, first=size * m.sign(), root=root)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("log_probs", "gradient"):
        return _exact_rows(s)
    if case["op"] == "norm":
        return torch.linalg.vector_norm(s["gradient"].double())
    return _exact_adamw(s)
