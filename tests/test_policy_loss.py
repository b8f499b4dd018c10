"""The clipped policy loss refuses what it cannot compute, before any
launch (no GPU needed)."""

import ctypes as C
from pathlib import Path

import pytest
import torch

from scacchi_b200 import _lib
from scacchi_b200.policy_loss import MAX_ACTIONS, clipped_policy_loss


def test_rejects_cpu_tensors():
    x = torch.zeros((2, 5))
    with pytest.raises(ValueError, match="CUDA device"):
        clipped_policy_loss(x, torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.zeros(2))


def _call(rows_kw=None, out_kw=None, n=4, actions=82, dtype=0, low=0.2, high=0.2, kl=0.0, workspace=1 << 20):
    """scacchi_policy_loss with made-up addresses: a refused call reads none."""
    rows = dict(logits=1 << 20, reference_logits=None, legal=None, action=1 << 20, old_log_prob=1 << 20,
                advantage=1 << 20, weight=None, reference_log_prob=None, logits_stride=actions,
                reference_stride=actions)
    out = dict(loss=1 << 20, log_prob=1 << 20, kl=None, clipped=1 << 20, grad_logits=None)
    rows.update(rows_kw or {})
    out.update(out_kw or {})
    r, o = _lib.PolicyRows(**rows), _lib.PolicyOut(**out)
    return _lib.lib().scacchi_policy_loss(C.byref(r), C.byref(o), n, actions, dtype, low, high, kl, workspace, None)


@pytest.mark.parametrize("kw", [
    dict(n=-1), dict(actions=0), dict(actions=MAX_ACTIONS + 1), dict(dtype=3), dict(dtype=-1), dict(low=1.0),
    dict(low=-0.1), dict(low=float("nan")), dict(high=-0.5), dict(high=float("inf")), dict(high=float("nan")),
    dict(kl=float("nan")), dict(workspace=None), dict(workspace=(1 << 20) + 4),
    dict(rows_kw=dict(logits=None)), dict(rows_kw=dict(action=None)), dict(rows_kw=dict(old_log_prob=None)),
    dict(rows_kw=dict(advantage=None)), dict(rows_kw=dict(logits_stride=81)),
    dict(rows_kw=dict(logits=(1 << 20) + 2)), dict(rows_kw=dict(action=(1 << 20) + 1)),
    dict(rows_kw=dict(logits=(1 << 20) + 1), dtype=1),
    dict(rows_kw=dict(reference_logits=1 << 20, reference_log_prob=1 << 20), out_kw=dict(kl=1 << 20)),
    dict(rows_kw=dict(reference_logits=1 << 20)), dict(rows_kw=dict(reference_log_prob=1 << 20)),
    dict(rows_kw=dict(reference_logits=1 << 20, reference_stride=10), out_kw=dict(kl=1 << 20)),
    dict(out_kw=dict(loss=None)), dict(out_kw=dict(log_prob=None)), dict(out_kw=dict(clipped=None)),
    dict(out_kw=dict(grad_logits=(1 << 20) + 1)),
], ids=str)
def test_library_rejects_without_launching(kw):
    before = _lib.lib().scacchi_policy_loss_launch_count()
    assert _call(**kw) == _lib.EINVAL
    assert _lib.lib().scacchi_policy_loss_launch_count() == before


def test_null_structs_are_rejected():
    out = _lib.PolicyOut(*[1 << 20] * 5)
    assert _lib.lib().scacchi_policy_loss(None, C.byref(out), 1, 2, 0, 0.2, 0.2, 0.0, 8, None) == _lib.EINVAL


def test_clusters_meet_before_the_first_remote_write():
    """A CTA may write another's shared memory only once that one runs: the
    long rows' kernel arrives on the cluster's barrier before its first row
    and waits for it before the first reduction across CTAs, also where the
    first row does not count.  Read from the source: on a GPU the row's
    latency hides a missing barrier."""
    source = (Path(__file__).parents[1] / "scacchi_b200" / "csrc" / "policy_loss.cu").read_text()
    kernel = source[source.index("policy_loss_long_kernel(const"):]
    kernel = kernel[:kernel.index("\n}\n")]
    rows = kernel.index("for (int64_t row = first")
    arrive, wait = kernel.find("barrier_arrive()"), kernel.find("barrier_wait()")
    assert 0 <= arrive < rows < wait
    assert "row == first" in kernel[kernel.rindex("\n", 0, wait):wait]  # once, by every thread
    for later in ("grp.stats(", "grp.reduce<", "finish_row<", "continue;", "map_shared_rank"):
        assert kernel.find(later) == -1 or wait < kernel.index(later), later
