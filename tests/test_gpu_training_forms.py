"""The training operators' further forms on the GPU: values past a limit, gradients asked for singly or kept in another
dtype, layers below their capacity, strided operands, and extents at the borders between kernels.  Tolerances are those of
test_gpu_training, whose operators and 64-bit formulas these tests use."""

from __future__ import annotations

import pytest
import torch

from test_gpu_training import BF16, CONCATENATED, FP16, FP32, INTERLEAVED, Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,order", [(BF16, INTERLEAVED), (BF16, CONCATENATED), (FP16, INTERLEAVED), (FP16, CONCATENATED),
                                         (FP32, INTERLEAVED)])
@pytest.mark.parametrize("function", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("rows,hidden,width", [(6, 64, 40), (70, 136, 201), (300, 1032, 520)])
def test_forward_pass_does_not_clip_nan(device, rows, hidden, width, function, order, dtype):
    """A NaN Gate or Up past a limit makes its row of the output NaN, as the backward pass has it, and no other."""

    def layer_and_row():
        layer = Layer(device, rows, hidden, width, dtype, function=function, order=order, limit=1.0, offset=0.5, bias=True)
        return layer, rows // 2

    layer, row = layer_and_row()
    layer.x[row, hidden - 1] = float("nan")
    projected, out = layer.forward()
    others = torch.arange(rows, device=device) != row
    assert bool(projected[row].isnan().all()) and bool(out[row].isnan().all())
    assert bool(projected[others].isfinite().all()) and bool(out[others].isfinite().all())
    for side in (0, 1):  # a NaN Gate beside a finite Up, and the other way round
        layer, row = layer_and_row()
        gate_up = layer.split(layer.weights.i_proj.bias.unsqueeze(0))
        gate_up[side][0, width - 1] = float("nan")
        projected, out = layer.forward()
        kept = layer.split(projected)
        assert bool(kept[side][:, width - 1].isnan().all()) and bool(kept[side][:, :width - 1].isfinite().all())
        assert bool(kept[1 - side].isfinite().all()) and bool(out.isnan().all())


def test_forward_pass_of_large_halves_does_not_clip_nan(device):
    """CONCATENATED weights of 2 GiB, whose activation is a launch of its own."""

    layer = Layer(device, 3, 16384, 32768, BF16, order=CONCATENATED, limit=1.0, offset=0.5, bias=True)
    layer.x[1, 5] = float("nan")
    projected, out = layer.forward()
    assert bool(projected[1].isnan().all()) and bool(out[1].isnan().all()) and bool(out[0::2].isfinite().all())
    layer.x[1, 5] = 0.0
    for side in (0, 1):
        gate_up = layer.split(layer.weights.i_proj.bias.unsqueeze(0))
        gate_up[side][0, 7] = float("nan")
        _, out = layer.forward()
        assert bool(out.isnan().all())
        gate_up[side][0, 7] = 0.0
    projected, out = layer.forward()
    layer.check_forward(projected, out)
