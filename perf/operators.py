"""The training operators' workloads: the clipped policy loss with its
gradient, the orthogonalised update and Muon's step.

``listed`` gives the fixed cases, ``draw`` more of the same ranges,
``prepare`` a case's inputs, ``run`` one pass (plain torch operations, or
the package's operators where ``own`` is set), ``exact`` the same outputs
in 64 bits and ``work`` what a pass cannot do without.
"""

from __future__ import annotations

import math

import torch

own = False

STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-8
BETA = 0.95
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _policy(rows, actions, dtype, legal, kl, gradient):
    return dict(op="policy", rows=rows, actions=actions, dtype=dtype, legal=legal, kl=kl, gradient=gradient)


def _matrix(op, batch, rows, cols, dtype):
    return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=dtype)


def listed():
    return [
        # one frame of a small self-play batch (64 games of 9x9 Hex): latency
        dict(_policy(64, 82, "fp32", True, "sampled", True), name="policy_frame64_hex9"),
        # 8192 lanes x 32 frames of 9x9 Hex against an older network's logits
        dict(_policy(8192 * 32, 82, "fp32", True, "full", True), name="policy_frames8192x32_hex9"),
        # held-out frames of 11x11 Hex: the loss alone, 16-bit logits
        dict(_policy(4099 * 17, 122, "bf16", True, "full", False), name="policy_eval_hex11_bf16"),
        # token rows over a generic vocabulary, one behaviour and one reference log-prob each
        dict(_policy(4096, 32000, "bf16", False, "sampled", True), name="policy_vocab32000_bf16"),
        # a few rows over a large odd vocabulary with the reference's logits: the row is the work
        dict(_policy(8, 131071, "fp32", False, "full", True), name="policy_vocab131071_rows8"),
        # the policy head's kernel [162, 82]: the smallest matrix, latency
        dict(_matrix("orthogonalize", 1, 162, 82, "fp32"), name="orth_head162x82"),
        # a ragged stack of 16-bit momenta
        dict(_matrix("orthogonalize", 3, 257, 1001, "bf16"), name="orth_ragged3x257x1001_bf16"),
        # a square attention-sized projection in 32 bits
        dict(_matrix("orthogonalize", 1, 2048, 2048, "fp32"), name="orth_square2048"),
        # a tall feed-forward kernel in 16 bits
        dict(_matrix("orthogonalize", 1, 8192, 2048, "bf16"), name="orth_tall8192x2048_bf16"),
        # the twelve convolutions of the 6x128 tower, [9 * 128, 128] each
        dict(_matrix("muon", 12, 1152, 128, "fp32"), name="muon_tower12x1152x128"),
        # a wide dense kernel with 16-bit gradients
        dict(_matrix("muon", 1, 1024, 4096, "bf16"), name="muon_wide1024x4096_bf16"),
        # two large square kernels: the tensor cores' rate
        dict(_matrix("muon", 2, 4096, 4096, "fp32"), name="muon_square2x4096"),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["policy", "policy", "orthogonalize", "muon"])
    if op == "policy":
        actions = _between(rng, 2, 131072)
        rows = _between(rng, 1, max(1, min(1 << 18, (1 << 26) // actions)))
        return _policy(rows, actions, rng.choice(sorted(DTYPES)), rng.random() < 0.5,
                       rng.choice(["none", "sampled", "full"]), rng.random() < 0.7)
    rows, cols = _between(rng, 16, 4096), _between(rng, 16, 4096)
    batch = _between(rng, 1, max(1, min(24, (1 << 24) // (rows * cols))))
    return _matrix(op, batch, rows, cols, rng.choice(["fp32", "bf16"] if op == "muon" else sorted(DTYPES)))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(1000003 * (seed % (1 << 31)) + salt)
    return g


def _prepare_policy(case, seed):
    """Rows as self-play leaves them: logits, a behaviour policy and a
    reference a little apart from it, the action the behaviour policy drew,
    an advantage and the row's share of the loss (one in ten masked)."""
    N, A, dtype = case["rows"], case["actions"], DTYPES[case["dtype"]]
    g = _gen(seed, 1)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    logits = (2.0 * normal(N, A)).to(dtype)
    legal = None
    if case["legal"]:
        legal = torch.rand((N, A), generator=g, device=DEVICE) < 0.7
        legal[:, 0] |= ~legal.any(-1)
    behaviour = logits.float() + 0.1 * normal(N, A)
    if legal is not None:
        behaviour.masked_fill_(~legal, -math.inf)
    noise = torch.rand((N, A), generator=g, device=DEVICE).clamp_(min=1e-12).log_().neg_().log_().neg_()
    action = (behaviour + noise).argmax(-1).to(torch.int32)
    del noise
    top = behaviour.amax(-1)
    old = behaviour.gather(-1, action.long()[:, None])[:, 0] - top - (behaviour - top[:, None]).exp().sum(-1).log()
    del behaviour
    advantage = normal(N)
    counted = torch.rand(N, generator=g, device=DEVICE) < 0.9
    counted[0] = True
    state = dict(case=case, logits=logits, action=action, old_log_prob=old, advantage=advantage, legal=legal,
                 weight=counted.float() / counted.sum().float(), reference_logits=None, reference_log_prob=None)
    if case["kl"] == "full":
        state["reference_logits"] = (logits.float() + 0.3 * normal(N, A)).to(dtype)
    if case["kl"] == "sampled":
        state["reference_log_prob"] = old + 0.1 * normal(N)
    return state


def _update_like(g, batch, rows, cols):
    """A batch's gradient: a few strong directions over a bulk whose rows
    and columns have scales of their own."""
    r = max(1, min(rows, cols) // 16)
    left = torch.randn((batch, rows, r), generator=g, device=DEVICE)
    right = torch.randn((batch, r, cols), generator=g, device=DEVICE)
    bulk = torch.randn((batch, rows, cols), generator=g, device=DEVICE)
    row = torch.exp(0.5 * torch.randn((batch, rows, 1), generator=g, device=DEVICE))
    col = torch.exp(0.5 * torch.randn((batch, 1, cols), generator=g, device=DEVICE))
    return 1e-3 * (left.mul_(1.0 / math.sqrt(r)) @ right + bulk * row * col)


def _prepare_matrix(case, seed):
    B, R, C, dtype = case["batch"], case["rows"], case["cols"], DTYPES[case["dtype"]]
    g = _gen(seed, 2)
    if case["op"] == "orthogonalize":
        return dict(case=case, matrix=_update_like(g, B, R, C).to(dtype))
    return dict(case=case, weight=math.sqrt(2.0 / R) * torch.randn((B, R, C), generator=g, device=DEVICE),
                gradient=_update_like(g, B, R, C).to(dtype), momentum=0.3 * _update_like(g, B, R, C),
                learning_rate=0.02, weight_decay=0.01)


def prepare(case, seed):
    return _prepare_policy(case, seed) if case["op"] == "policy" else _prepare_matrix(case, seed)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _plain_policy(s):
    # 64 bits up to the log-probabilities: which side of a clip border a row
    # falls on and the KL of two near policies are lost in 32
    case, x = s["case"], s["logits"].double()
    A = x.shape[-1]
    keep = x > -math.inf
    if s["legal"] is not None:
        keep &= s["legal"]
    action = s["action"].long()
    at = action.clamp(0, A - 1)[:, None]
    counts = (s["weight"] != 0) & (action >= 0) & (action < A) & keep.gather(-1, at)[:, 0]
    x = torch.where(keep, x, -math.inf)
    top = torch.where(counts, x.amax(-1), 0.0)
    e = torch.exp(x - top[:, None])
    z = e.sum(-1)
    lse = top + torch.log(z)
    lp = torch.where(counts, x.gather(-1, at)[:, 0] - lse, 0.0)
    adv = s["advantage"].double()
    ratio = torch.exp(lp - s["old_log_prob"].double())
    clipped = counts & torch.where(adv >= 0, ratio > 1 + CLIP_HIGH, ratio < 1 - CLIP_LOW)
    bound = torch.where(adv >= 0, 1 + CLIP_HIGH, 1 - CLIP_LOW).double()
    term = -adv * torch.where(clipped, bound, ratio)
    slope = torch.where(clipped, 0.0, -adv * ratio)
    beta = 0.05 if case["kl"] != "none" else 0.0
    kl = mean = None
    if case["kl"] == "sampled":
        gap = s["reference_log_prob"].double() - lp
        kl = torch.where(counts, torch.exp(gap) - gap - 1, 0.0)
        slope = slope - beta * (torch.exp(gap) - 1)
    p = None
    if case["kl"] == "full":
        p = e / z[:, None]
        r = torch.where(keep, s["reference_logits"].double(), -math.inf)
        rtop = torch.where(counts, r.amax(-1), 0.0)
        rlse = rtop + torch.log(torch.exp(r - rtop[:, None]).sum(-1))
        d = torch.where(keep, x - r, 0.0)
        mean = (p * d).sum(-1)
        kl = torch.where(counts, mean - lse + rlse, 0.0)
    if kl is not None:
        term = term + beta * kl
    w = s["weight"].double()
    loss = torch.where(counts, w * term, 0.0).sum().float()
    out = dict(loss=loss, log_prob=lp.float(), clipped=clipped)
    if kl is not None:
        out["kl"] = kl.float()
    if case["gradient"]:
        p32 = (e / z[:, None]).float()
        grad = -slope.float()[:, None] * p32
        if mean is not None:
            grad += beta * p32 * (d - mean[:, None]).float()
        grad.scatter_add_(-1, at, slope.float()[:, None])
        grad = torch.where(counts[:, None] & keep, w.float()[:, None] * grad, 0.0)
        out["grad_logits"] = grad.to(s["logits"].dtype)
    return out


def _plain_orthogonalize(u):
    """Newton-Schulz steps of a stack of fp32 matrices."""
    a, b, c = COEFFICIENTS
    tall = u.shape[-2] > u.shape[-1]
    x = u.mT if tall else u
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + EPS)
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _plain_muon(s):
    g = s["gradient"].float()
    s["momentum"].mul_(BETA).add_(g, alpha=1 - BETA)
    o = _plain_orthogonalize((1 - BETA) * g + BETA * s["momentum"])
    R, C = g.shape[-2:]
    lr = s["learning_rate"]
    s["weight"].mul_(1 - lr * s["weight_decay"]).sub_(o, alpha=lr * math.sqrt(max(1.0, C / R)))
    return dict(weight=s["weight"], momentum=s["momentum"])


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "policy":
            from scacchi_b200.policy_loss import clipped_policy_loss

            out = clipped_policy_loss(
                state["logits"], state["action"], state["old_log_prob"], state["advantage"], legal=state["legal"],
                weight=state["weight"], reference_logits=state["reference_logits"],
                reference_log_prob=state["reference_log_prob"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                kl_coefficient=0.05 if state["case"]["kl"] != "none" else 0.0, gradient=state["case"]["gradient"])
            return {k: v for k, v in out._asdict().items() if v is not None}
        from scacchi_b200.muon import muon_update, orthogonalize

        if op == "orthogonalize":
            return orthogonalize(state["matrix"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        muon_update(state["weight"], state["gradient"], state["momentum"], learning_rate=state["learning_rate"],
                    beta=BETA, nesterov=True, weight_decay=state["weight_decay"], steps=STEPS,
                    coefficients=COEFFICIENTS, eps=EPS)
        return dict(weight=state["weight"], momentum=state["momentum"])
    if op == "policy":
        return _plain_policy(state)
    if op == "orthogonalize":
        return _plain_orthogonalize(state["matrix"].float()).to(state["matrix"].dtype)
    return _plain_muon(state)


# ---------------------------------------------------------------------------
# work and the 64-bit values
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "policy":
        N, A = case["rows"], case["actions"]
        size = DTYPES[case["dtype"]].itemsize
        full, sampled = case["kl"] == "full", case["kl"] == "sampled"
        row = 4 * 4 + 4 + 1 + (4 if sampled else 0) + (4 if full or sampled else 0)
        cell = size * (1 + full + case["gradient"]) + case["legal"]
        return {"bytes": N * (row + A * cell) + 4, "flops": N * A * (4 + 6 * full + 3 * case["gradient"])}
    B, R, C = case["batch"], case["rows"], case["cols"]
    m, n = min(R, C), max(R, C)
    size = DTYPES[case["dtype"]].itemsize
    # a step: X X^T and A A are symmetric (half of each), M X is whole
    flops = STEPS * B * (m * m * n + m * m * m + 2 * m * m * n)
    cell = 2 * size if case["op"] == "orthogonalize" else size + 4 * 4
    return {"bytes": B * R * C * cell, "flops": flops}


def _exact_policy(s):
    """Row-wise definition: log-softmax over the kept actions, the clipped
    objective as min(ratio A, clip(ratio) A), KL as sum p log(p / q)."""
    case = s["case"]
    A = s["logits"].shape[-1]
    x = s["logits"].double()
    if s["legal"] is not None:
        x = x.masked_fill(~s["legal"], -math.inf)
    counts = s["weight"] > 0
    idx = s["action"].long()[:, None]
    logp = torch.log_softmax(x, -1)
    lp = logp.gather(-1, idx).squeeze(-1)
    adv, w = s["advantage"].double(), s["weight"].double()
    ratio = torch.exp(lp - s["old_log_prob"].double())
    limited = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    objective = torch.minimum(ratio * adv, limited * adv)
    clipped = counts & (ratio != limited) & (limited * adv < ratio * adv)
    beta = 0.05
    per_row = -objective
    dlp = torch.where(clipped, 0.0, -(ratio * adv))
    kl = None
    p = logp.exp()
    grad = None
    if case["kl"] == "sampled":
        t = s["reference_log_prob"].double() - lp
        kl = torch.expm1(t) - t
        per_row = per_row + beta * kl
        dlp = dlp - beta * torch.expm1(t)
    if case["gradient"]:
        grad = -p * dlp[:, None]
        grad.scatter_add_(-1, idx, dlp[:, None])
    if case["kl"] == "full":
        logq = s["reference_logits"].double()
        if s["legal"] is not None:
            logq = logq.masked_fill(~s["legal"], -math.inf)
        logq = torch.log_softmax(logq, -1)
        apart = torch.where(p > 0, logp - logq, 0.0)
        kl = (p * apart).sum(-1)
        per_row = per_row + beta * kl
        if grad is not None:
            grad += beta * p * (apart - kl[:, None])
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    out = dict(loss=(w * torch.where(counts, per_row, zero)).sum(), log_prob=torch.where(counts, lp, zero),
               clipped=clipped)
    if kl is not None:
        out["kl"] = torch.where(counts, kl, zero)
    if grad is not None:
        out["grad_logits"] = grad * w[:, None]
    return out


def _exact_orthogonalize(u):
    """X (a I + G (b I + c G)) with G = X^T X on the narrow side."""
    a, b, c = COEFFICIENTS
    wide = u.shape[-1] > u.shape[-2]
    x = u.transpose(-1, -2) if wide else u
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + EPS)
    eye = torch.eye(x.shape[-1], dtype=x.dtype, device=x.device)
    for _ in range(STEPS):
        gram = x.transpose(-1, -2) @ x
        x = x @ (a * eye + gram @ (b * eye + c * gram))
    return x.transpose(-1, -2) if wide else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "policy":
        return _exact_policy(s)
    if case["op"] == "orthogonalize":
        return _exact_orthogonalize(s["matrix"].double())
    g = s["gradient"].double()
    m = BETA * s["momentum"].double() + (1 - BETA) * g
    o = _exact_orthogonalize((1 - BETA) * g + BETA * m)
    R, C = g.shape[-2:]
    lr = s["learning_rate"]
    w = (1 - lr * s["weight_decay"]) * s["weight"].double() - lr * math.sqrt(max(1.0, C / R)) * o
    return dict(weight=w, momentum=m)
