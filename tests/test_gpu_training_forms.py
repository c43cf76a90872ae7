"""The training operators' further forms on the GPU: values past a limit, gradients asked for singly or kept in another
dtype, layers below their capacity, strided operands, and extents at the borders between kernels.  Tolerances are those of
test_gpu_training, whose operators and 64-bit formulas these tests use."""

from __future__ import annotations

import pytest
import torch

from test_gpu_training import BF16, CONCATENATED, FP16, FP32, INTERLEAVED, Layer, Projection, near, product

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


def test_padded_copies_of_more_chunks_than_a_launch_has_threads(device):
    """2^24 rows of 257 chunks, the last cut: their padded copy is past 2^32 chunks."""

    rows, k, n = 1 << 24, 8, 2049
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(device)[0] < 160 << 30:
        pytest.skip("64 GiB of gradients and their copy do not fit the free memory")
    case = Projection(device, 8, k, n, BF16, capacity=rows)
    case.grad = torch.empty((rows, n), dtype=BF16, device=device).normal_(generator=torch.Generator(device=device).manual_seed(3))
    case.x = torch.zeros((rows, k), dtype=BF16, device=device)
    grad_x = torch.full((rows, k), float("nan"), dtype=BF16, device=device)
    case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=grad_x)
    for first in range(0, rows, 1 << 18):
        some = slice(first, first + (1 << 18))
        exact, magnitude = product(case.grad[some], case.weights.values)
        near(grad_x[some], exact, n * 2.0**-23 * magnitude, f"input gradient from row {first}")
    del case, grad_x, exact, magnitude
    torch.cuda.empty_cache()
