"""What the entry points of projection gradients, the Dense layer's training and orthogonal updates refuse before any
device call, and the sizes they ask for: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from crosspool_amd import _native
from crosspool_amd.ffn import GateTransform, GateUpOrder, SiluActivation
from crosspool_amd.muon import MuonPlan, gate_up_matrices
from crosspool_amd.operators import (
    Activation,
    DenseAdapterLayout,
    DenseExecutionPlan,
    DenseGradients,
    DenseSignature,
    GemmPlan,
    ProjectionLayout,
    TensorLayout,
)

BAD = _native.XP_ERROR_INVALID_ARGUMENT
BF16, F16, F32 = _native.XP_DTYPE_BF16, _native.XP_DTYPE_F16, _native.XP_DTYPE_F32
SILU = ctypes.byref(_native.ActivationDesc(function=_native.XP_ACTIVATION_SILU, gated=1, alpha=1.0))
BIG = 1 << 40


def backward(**changes):
    call = dict(x=0x100000, ld_x=64, rows=8, k=64, w=0x200000, n=48, grad=0x300000, ld_grad=48, dtype=BF16, gx=0x400000, ld_gx=64,
                gw=0x500000, gw_dtype=BF16, gb=0x600000, accumulate=0, capacity=8, ws=0x10000000, ws_bytes=BIG)
    call.update(changes)
    return _native.library().xp_projection_backward(*call.values(), None)


def keep(**changes):
    call = dict(x=0x100000, ld_x=64, rows=8, k=64, w=0x200000, n=48, bias=None, projected=0x300000, ld_p=48, activated=0x400000,
                dtype=BF16, order=_native.XP_GATE_UP_INTERLEAVED, act=SILU, capacity=8, ws=0x10000000, ws_bytes=BIG)
    call.update(changes)
    return _native.library().xp_projection_keep(*call.values(), None)


def dense(**changes):
    call = dict(x=0x100000, ld_x=64, rows=8, hidden=64, w_in=0x200000, w_out=0x300000, width=40, projected=0x400000, ld_p=80,
                grad=0x500000, ld_grad=64, dtype=BF16, order=_native.XP_GATE_UP_INTERLEAVED, act=SILU, gx=0x600000, ld_gx=64,
                gi=0x700000, go=0x800000, kept=BF16, bi=0x900000, bo=0xA00000, accumulate=0, capacity=8, ws=0x10000000, ws_bytes=BIG)
    call.update(changes)
    return _native.library().xp_dense_backward(*call.values(), None)


def matrices(data, matrix=4096, row=64):
    return ctypes.byref(_native.Matrices(data, matrix, row))


def orthogonalize(updates=None, output=None, **changes):
    call = dict(matrices=2, rows=48, columns=64, dtype=BF16, steps=5, eps=1e-7)
    call.update({key: value for key, value in changes.items() if key in call})
    return _native.library().xp_muon_orthogonalize(
        updates or matrices(0x100000), *call.values(), output or matrices(0x200000), changes.get("ws", 0x10000000),
        changes.get("ws_bytes", BIG), None)


def step(**changes):
    call = dict(weights=matrices(0x100000), gradients=matrices(0x200000), momentum=matrices(0x300000),
                new_weights=matrices(0x100000), new_momentum=matrices(0x300000), matrices=2, rows=48, columns=64, dtype=BF16,
                weights_dtype=BF16, steps=5, eps=1e-7, rate=0.02, decay=0.1, factor=0.95, nesterov=1, scale=1.0, ws=0x10000000,
                ws_bytes=BIG)
    call.update(changes)
    return _native.library().xp_muon_step(*call.values(), None)


@pytest.mark.parametrize("changes", [
    dict(dtype=0), dict(dtype=4), dict(rows=-1), dict(rows=9), dict(k=0), dict(n=0), dict(k=(1 << 20) + 8), dict(capacity=1 << 25),
    dict(w=None), dict(w=0x200008), dict(grad=None), dict(x=None), dict(x=0x100002), dict(ld_x=60), dict(ld_x=63), dict(ld_x=68),
    dict(ld_grad=(1 << 20) + 8), dict(grad=0x300008), dict(gx=0x400001), dict(ld_gx=32), dict(gw_dtype=F16), dict(gw=0x500001),
    dict(gb=0x600002), dict(ws=None), dict(ws=0x10000008), dict(ws_bytes=64),
    dict(gx=0x100000), dict(gx=0x2FFFF0), dict(gw=0x200000), dict(gw=0x400100), dict(gb=0x300010), dict(ws=0x2FFFF0),
])
def test_projection_gradient_refusals(changes):
    assert backward(**changes) == BAD, changes
    assert _native.last_error()


@pytest.mark.parametrize("changes", [
    dict(dtype=9), dict(rows=9), dict(k=0), dict(n=47), dict(w=None), dict(x=None), dict(x=0x100008), dict(projected=None), dict(ld_p=40),
    dict(act=None), dict(bias=0x700002), dict(activated=0x400001), dict(ws=0x1000000C, k=61), dict(ws_bytes=16, k=61), dict(projected=0x400010), dict(activated=0x100000),
    dict(projected=0x200000), dict(act=ctypes.byref(_native.ActivationDesc(function=7))),
    dict(order=0), dict(order=3), dict(order=_native.XP_GATE_UP_CONCATENATED, n=1 << 20, k=1 << 10, ld_x=1 << 10, ld_p=1 << 20),
])
def test_kept_projection_refusals(changes):
    assert keep(**changes) == BAD, changes


@pytest.mark.parametrize("changes", [
    dict(dtype=0), dict(act=None), dict(order=0), dict(width=0), dict(hidden=0), dict(width=1 << 20), dict(rows=9), dict(w_in=None),
    dict(w_out=0x300004), dict(projected=None), dict(ld_p=79), dict(grad=0x500002), dict(x=None), dict(ld_x=65), dict(gx=0x600001),
    dict(kept=F16), dict(gi=0x700001), dict(bi=0x900001), dict(ws=None), dict(ws_bytes=100), dict(gi=0x200000), dict(go=0x700040),
    dict(gx=0x500000), dict(bo=0x900004), dict(gi=0x10000100),
])
def test_dense_backward_refusals(changes):
    assert dense(**changes) == BAD, changes


@pytest.mark.parametrize("changes", [
    dict(matrices=0), dict(matrices=4097), dict(rows=0), dict(columns=0), dict(rows=(1 << 16) + 1, columns=(1 << 16) + 1),
    dict(columns=(1 << 20) + 1), dict(dtype=7), dict(steps=0), dict(steps=17), dict(eps=0.0), dict(eps=float("nan")), dict(ws=None),
    dict(ws=0x10000008), dict(ws_bytes=1000), dict(ws=0x1FFFF0), dict(updates=matrices(None)), dict(updates=matrices(0x100001)),
    dict(updates=matrices(0x100000, 4096, 63)), dict(updates=matrices(0x100000, 64, 127)), dict(output=matrices(0x100002)),
    dict(output=matrices(0x100000, 4096, 80)), dict(output=matrices(0x200000, 0, 64)),
])
def test_orthogonal_update_refusals(changes):
    assert orthogonalize(**changes) == BAD, changes


@pytest.mark.parametrize("changes", [
    dict(weights_dtype=F16), dict(rate=float("inf")), dict(decay=float("nan")), dict(factor=1.0), dict(factor=-0.1),
    dict(scale=float("nan")), dict(momentum=matrices(0x300002)), dict(new_momentum=matrices(0x300100)),
    dict(new_weights=matrices(0x100020)), dict(new_weights=matrices(0x200000)), dict(new_momentum=matrices(0x100000)),
    dict(new_weights=matrices(0x300000)), dict(gradients=None), dict(ws_bytes=10),
])
def test_optimiser_step_refusals(changes):
    assert step(**changes) == BAD, changes


def test_workspace_sizes():
    lib = _native.library()
    for query, sizes in ((lib.xp_projection_backward_workspace_bytes, (64, 48, 40)), (lib.xp_projection_keep_workspace_bytes, (64, 48, 41)),
                         (lib.xp_dense_backward_workspace_bytes, (64, 48, 40, 1)), (lib.xp_muon_workspace_bytes, (2, 48, 40))):
        assert query(*sizes, BF16) > 0 and query(*sizes, F32) > 0
        assert query(*sizes, 0) == 0 and query(*sizes, 5) == 0
        assert query(0, *sizes[1:], BF16) == 0 and query(sizes[0], 0, *sizes[2:], BF16) == 0
    # a larger capacity needs no less
    last = 0
    for rows in (1, 5, 64, 65, 500, 4096):
        size = lib.xp_dense_backward_workspace_bytes(rows, 1030, 2053, 1, F16)
        assert size >= last
        last = size


def layouts(dtype=torch.bfloat16, rows=8, k=64, n=48):
    return dict(input_layout=TensorLayout((rows, k), dtype), weight_layout=ProjectionLayout(TensorLayout((n, k), dtype)),
                result_layout=TensorLayout((rows, n), dtype))


def test_plan_refusals():
    GemmPlan.prepare(**layouts(), activation=None, backward=True)
    with pytest.raises(ValueError, match="activation"):
        GemmPlan.prepare(**layouts(), activation=Activation(SiluActivation(), None), backward=True)
    gated = Activation(SiluActivation(), GateTransform())

    def signature(dtype, order):
        return DenseSignature(payload_dtype=dtype, payload_row_capacity=8, hidden_size=64, local_intermediate_size=40, activation=gated,
                              i_proj=ProjectionLayout(TensorLayout((80, 64), dtype), gate_up_order=order),
                              o_proj=ProjectionLayout(TensorLayout((64, 40), dtype)))

    plan = DenseExecutionPlan.prepare(signature(torch.bfloat16, GateUpOrder.CONCATENATED), backward=True)
    assert plan.backward and plan.workspace.nbytes > DenseExecutionPlan.prepare(signature(torch.bfloat16, GateUpOrder.CONCATENATED)).workspace.nbytes
    with pytest.raises(ValueError, match="adapters"):
        DenseExecutionPlan.prepare(signature(torch.bfloat16, GateUpOrder.INTERLEAVED), adapters=DenseAdapterLayout(2, 4), backward=True)
    with pytest.raises(ValueError, match="INTERLEAVED"):
        DenseExecutionPlan.prepare(signature(torch.float32, GateUpOrder.CONCATENATED), backward=True)
    with pytest.raises(ValueError, match="share one dtype"):
        DenseGradients(i_values=torch.zeros(2, 2), o_values=torch.zeros(2, 2, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="bf16"):
        MuonPlan.prepare(rows=4, columns=4, dtype=torch.float64)
    with pytest.raises(ValueError, match="matrices"):
        MuonPlan.prepare(rows=4, columns=0, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="even"):
        gate_up_matrices(torch.zeros(3, 2))
    view = gate_up_matrices(torch.arange(12.0).view(4, 3))
    assert view.shape == (2, 2, 3) and view[1, 0].tolist() == [3.0, 4.0, 5.0] and view.data_ptr() != 0
