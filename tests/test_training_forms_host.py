"""What the trained layer's further entry points refuse before any device call: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from crosspool_amd import _native
from crosspool_amd.muon import MuonPlan
from test_training_host import BAD, BF16, F32, SILU, backward, dense

CONCATENATED = _native.XP_GATE_UP_CONCATENATED


def kept_activation(**changes):
    call = dict(projected=0x100000, activated=0x200000, rows=8, width=40, dtype=BF16, order=CONCATENATED, act=SILU)
    call.update(changes)
    return _native.library().xp_kept_activation(*call.values(), None)


@pytest.mark.parametrize("changes", [
    dict(act=None), dict(rows=-1), dict(width=-1), dict(dtype=F32), dict(dtype=0), dict(order=0), dict(order=3), dict(projected=None),
    dict(activated=None), dict(projected=0x100001), dict(activated=0x200001), dict(activated=0x100000), dict(activated=0x100002),
    dict(act=ctypes.byref(_native.ActivationDesc(function=7, gated=1, alpha=1.0))),
])
def test_kept_activation_refusals(changes):
    assert kept_activation(**changes) == BAD, changes
    assert _native.last_error()


def test_kept_activation_of_nothing():
    assert kept_activation(rows=0, projected=None, activated=None) == 0


def test_inputs_are_needed_by_their_weights_gradient_alone():
    """Without it a missing input is not what is refused."""

    assert backward(x=None) == BAD and dense(x=None) == BAD
    assert backward(x=None, gw=None, ws_bytes=64) == BAD and "workspace" in _native.last_error()
    assert dense(x=None, gi=None, ws_bytes=100) == BAD and "workspace" in _native.last_error()


def test_rows_too_far_apart():
    for changes in (dict(ld_x=(1 << 20) + 8), dict(ld_grad=(1 << 20) + 8), dict(ld_gx=(1 << 20) + 8)):
        assert backward(**changes) == BAD and "2^20" in _native.last_error()


def test_batches_past_their_extents():
    with pytest.raises(ValueError, match="2\\^36"):
        MuonPlan.prepare(matrices=2, rows=1 << 16, columns=1 << 20, dtype=torch.bfloat16)
    # many tiles are no reason to refuse: they run in several launches
    assert MuonPlan.prepare(matrices=4096, rows=1, columns=1 << 20, dtype=torch.bfloat16).workspace.nbytes >= 2 * 4096 << 21
