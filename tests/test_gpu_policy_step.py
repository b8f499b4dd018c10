"""The operators around a policy step in a row, as a training loop uses
them: the behaviour policy's log-probs -> clipped policy loss -> an entropy
bonus's gradient beside the loss's -> the head's weight and bias gradients ->
their norm -> Muon for the weight, AdamW for the bias and everything else ->
the network with the new parameters.

Each link is held to its definition in 64 bits on what the link before it
gave."""

import math

import numpy as np
import pytest
import torch

from oracle import network_ref as NR
from scacchi_b200 import _lib
from scacchi_b200.adamw import NetworkAdamW, gradient_norm
from scacchi_b200.log_probs import policy_log_probs, policy_log_probs_gradient
from scacchi_b200.loss_input import TrainingLossConfig, make_compute_input_for_lossfn
from scacchi_b200.muon import NetworkMuon
from scacchi_b200.network import AZDirichletNet, init_params
from scacchi_b200.policy_loss import clipped_policy_loss
from scacchi_b200.random import PRNGKey
from tests.test_gpu_adamw import _step_and_check
from tests.test_gpu_log_probs import _check, _check_gradient
from tests.test_gpu_targets import _random_frames, _to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_frames_to_new_parameters(cuda, bits):
    B, T, A = 24, 17, 82
    frames = _to(_random_frames(np.random.default_rng(3), B, T, A, True, True), "cuda")
    sample = make_compute_input_for_lossfn(TrainingLossConfig())(frames)
    params = init_params(1)
    key = PRNGKey(5)
    muon = NetworkMuon(params, learning_rate=0.02)
    adam = NetworkAdamW(params, learning_rate=1e-2, weight_decay=0.1, max_norm=0.25, state_bits=bits, key=key)
    g = torch.Generator(device="cuda").manual_seed(0)
    features = torch.randn((B * T, 162), generator=g, device="cuda")
    advantage = torch.randn((B * T,), generator=g, device="cuda")
    action, legal = sample.played_action.reshape(-1), sample.policy_mask.reshape(-1, A)
    mask = sample.policy_loss_mask.reshape(-1)
    weight = mask.float() / mask.sum()
    decay = {k: 0.1 if w.dim() > 1 else 0.0 for k, w in adam.weights.items()}
    assert decay["policy_conv_w"] == 0.1 and decay["policy_b"] == 0.0

    def logits_of():
        return features @ muon.matrices["policy_w"] + adam.weights["policy_b"]

    old, _ = _check(logits_of(), action, legal, 1.0, 5)
    old_log_prob = old.log_prob.masked_fill(~old.log_prob.isfinite(), 0.0)
    for _ in range(3):
        logits = logits_of()
        loss = clipped_policy_loss(logits, action, old_log_prob, advantage, legal=legal, weight=weight)
        now, d = _check(logits, action, legal, 1.0, 0)
        counted = mask & now.log_prob.isfinite()
        assert float((now.log_prob - loss.log_prob)[counted].abs().max()) < 1e-5
        bonus = -0.01 * weight
        _check_gradient(logits, action, legal, 1.0, now, d, None, bonus)
        grad = loss.grad_logits + policy_log_probs_gradient(logits, action, now, grad_entropy=bonus, legal=legal)
        assert not bool(grad[~legal].any())
        grads = {"policy_b": grad.sum(0)}
        for k, w in adam.weights.items():
            if k != "policy_b" and k != "value_b":  # one weight without a gradient
                grads[k] = 1e-3 * torch.randn(w.shape, generator=g, device="cuda")
        dense = {"policy_w": features.t() @ grad}
        norm = gradient_norm([*grads.values(), *dense.values()])
        want = math.sqrt(sum(float(t.double().square().sum()) for t in (*grads.values(), *dense.values())))
        assert abs(float(norm) - want) <= 2.0 ** -23 * want
        muon.step(dense)
        _step_and_check(adam, adam.weights, grads, lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, decay=decay, clip=0.25, key=key,
                        norm=norm)
    new = adam.params(muon.params())
    assert np.array_equal(new.policy_b, adam.weights["policy_b"].cpu().numpy())
    assert np.array_equal(new.blocks[2]["bn1"].scale, adam.weights["blocks.2.bn1.scale"].cpu().numpy())
    assert np.array_equal(new.policy_w, muon.matrices["policy_w"].cpu().numpy())
    assert not np.array_equal(new.policy_b, params.policy_b) and not np.array_equal(new.conv_w, params.conv_w)
    assert np.array_equal(new.value_b, params.value_b) and np.array_equal(new.bn.mean, params.bn.mean)
    assert np.array_equal(new.blocks[0]["conv1_w"], params.blocks[0]["conv1_w"])
    obs = NR.observations(16, seed=2)
    got, _, _ = AZDirichletNet(new)(torch.from_numpy(obs).cuda())
    assert float(np.abs(got.cpu().numpy() - NR.forward(new, obs)[0]).max()) < 2e-2
    assert _lib.tower_error() == 0 and _lib.muon_error() == 0
