"""The training operators in a row, as a training loop uses them: self-play
frames -> loss input -> clipped policy loss and its gradient -> the policy
head's weight gradient -> Muon -> the network with the new weights.

Each link is held to its own definition in 64 bits on what the link before
it gave (the bounds of test_gpu_policy_loss.py and test_gpu_muon.py)."""

import math

import numpy as np
import pytest
import torch

from oracle import network_ref as NR
from scacchi_b200 import _lib
from scacchi_b200.loss_input import TrainingLossConfig, make_compute_input_for_lossfn
from scacchi_b200.muon import DENSE, NetworkMuon
from scacchi_b200.network import AZDirichletNet, init_params
from scacchi_b200.policy_loss import clipped_policy_loss
from tests.test_gpu_muon import _bound, _exact, _muon64
from tests.test_gpu_policy_loss import _plain
from tests.test_gpu_targets import _random_frames, _to

pytestmark = pytest.mark.gpu


def test_frames_to_new_weights(cuda):
    B, T, A = 24, 17, 82
    frames = _to(_random_frames(np.random.default_rng(3), B, T, A, True, True), "cuda")
    sample = make_compute_input_for_lossfn(TrainingLossConfig())(frames)
    params = init_params(1)
    opt = NetworkMuon(params, learning_rate=0.02, weight_decay=0.01)
    g = torch.Generator(device="cuda").manual_seed(0)
    features = torch.randn((B, T, 162), generator=g, device="cuda")
    advantage = torch.randn((B, T), generator=g, device="cuda")
    mask = sample.policy_loss_mask
    weight = mask.float() / mask.sum()
    assert 0 < int(mask.sum()) < B * T
    with torch.no_grad():
        start = features @ opt.matrices["policy_w"]
        legal_start = start.masked_fill(~sample.policy_mask, -math.inf)
        old = torch.log_softmax(legal_start, -1).gather(-1, sample.played_action.long()[..., None])[..., 0]
        old = old.masked_fill(~torch.isfinite(old), 0.0)
    kw = dict(legal=sample.policy_mask, weight=weight, reference_logits=start)
    losses = []
    for _ in range(3):
        w = opt.matrices["policy_w"].clone().requires_grad_(True)
        logits = features @ w
        out = clipped_policy_loss(logits, sample.played_action, old, advantage, kl_coefficient=0.1, **kw)
        want, clipped = _plain(logits.detach().reshape(-1, A), sample.played_action.reshape(-1), old.reshape(-1),
                               advantage.reshape(-1), kl_coefficient=0.1, legal=sample.policy_mask.reshape(-1, A),
                               weight=weight.reshape(-1), reference_logits=start.reshape(-1, A))
        assert torch.equal(out.clipped.reshape(-1), clipped)
        for name, (value, tol) in want.items():
            assert float(((getattr(out, name).double().reshape(value.shape) - value).abs() - tol).max()) <= 0, name
        assert not out.grad_logits[~mask].any()
        logits.backward(out.grad_logits)
        before = opt.matrices["policy_w"].clone()
        new_w, new_m, u = _muon64(before, w.grad, opt.momentum["policy_w"], 0.02, 0.95, True, 0.01, 1.0)
        opt.step({"policy_w": w.grad})
        norm = torch.linalg.vector_norm
        o_tol = float(_bound(u.float(), _exact(u)) + 2.0 ** -20 * norm(_exact(u)))
        assert float(norm(opt.matrices["policy_w"].double() - new_w)) <= 0.02 * o_tol + 3 * 2.0 ** -24 * float(norm(new_w))
        losses.append(float(out.loss))
    assert all(math.isfinite(v) for v in losses) and _lib.muon_error() == 0
    # the network evaluates the new head; nothing else moved
    new = opt.params()
    assert not np.array_equal(new.policy_w, params.policy_w)
    for name in DENSE[1:]:
        assert np.array_equal(getattr(new, name), getattr(params, name))
    obs = NR.observations(16, seed=2)
    got, _, _ = AZDirichletNet(new)(torch.from_numpy(obs).cuda())
    ref = NR.forward(new, obs)[0]
    assert float(np.abs(got.cpu().numpy() - ref).max()) < 2e-2
    assert float(np.abs(ref - NR.forward(params, obs)[0]).max()) > 0


def test_network_muon_steps_every_matrix(cuda):
    params = init_params(2, random_batchnorm=True)
    opt = NetworkMuon(params, learning_rate=0.05, nesterov=False)
    g = torch.Generator(device="cuda").manual_seed(1)
    grads = {k: torch.randn(v.shape, generator=g, device="cuda") for k, v in opt.matrices.items()}
    assert grads["convs"].shape == (12, 1152, 128)
    before = {k: v.clone() for k, v in opt.matrices.items()}
    opt.step(grads)
    new = opt.params()
    for k, w in before.items():
        scale = math.sqrt(max(1.0, w.shape[-1] / w.shape[-2]))
        want, _, u = _muon64(w, grads[k], torch.zeros_like(w), 0.05, 0.95, False, 0.0, scale)
        err = torch.linalg.vector_norm(opt.matrices[k].double() - want, dim=(-2, -1))
        tol = (0.05 * scale * (_bound(u.float(), _exact(u))
                               + 2.0 ** -20 * torch.linalg.vector_norm(_exact(u), dim=(-2, -1)))
               + 3 * 2.0 ** -24 * torch.linalg.vector_norm(want, dim=(-2, -1)))
        assert bool((err <= tol).all()), k
    convs = opt.matrices["convs"].cpu().numpy()
    for i, blk in enumerate(new.blocks):
        assert blk["conv1_w"].shape == (3, 3, 128, 128)
        assert np.array_equal(blk["conv1_w"].reshape(1152, 128), convs[2 * i])
        assert np.array_equal(blk["conv2_w"].reshape(1152, 128), convs[2 * i + 1])
        assert np.array_equal(blk["bn1"].scale, params.blocks[i]["bn1"].scale)
    with pytest.raises(ValueError, match="no such matrices"):
        opt.step({"conv_w": grads["convs"]})
