"""The training operators' further forms on the GPU: values past a limit, gradients asked for singly or kept in another
dtype, layers below their capacity, strided operands, and extents at the borders between kernels.  Tolerances are those of
test_gpu_training, whose operators and 64-bit formulas these tests use."""

from __future__ import annotations

import pytest
import torch

from crosspool_amd.operators import DenseGradients

from test_gpu_training import ACT, BF16, CONCATENATED, FP16, FP32, INTERLEAVED, Layer, Projection, half_step, near, product, rows_of, tiny

pytestmark = pytest.mark.gpu


def check_forward(layer, projected, out):
    """The forward pass against the formula of its inputs, not of the kept values: the activation is that of the unrounded sums.

    Those are off by what n fp32 products may be off by; no activation's slope passes 1.13, and a limit none at all, so
    f(g) h is off by 1.13 of g's error times |h| and |f(g)| times h's, then by its own 2^-14 (fp32 2^-20) and half a step.
    """

    bias_in, bias_out = layer.weights.i_proj.bias, layer.weights.o_proj.bias
    exact, magnitude = product(layer.x, layer.weights.i_proj.values.T.contiguous())
    if bias_in is not None:
        exact, magnitude = exact + bias_in.double(), magnitude + bias_in.double().abs()
    off = (layer.hidden + 1) * 2.0**-23 * magnitude
    near(projected, exact, off, "projected")
    f, _, _, factor, _, _ = layer.terms(exact)
    gate_off, up_off = layer.split(off)
    if factor is None:
        activated, activated_off = f, 1.13 * gate_off
    else:
        activated, activated_off = f * factor, 1.13 * gate_off * (factor.abs() + up_off) + f.abs() * up_off
    activated_off = activated_off + (half_step(layer.dtype) + ACT[layer.dtype]) * (activated.abs() + activated_off) + tiny(layer.dtype)
    w_out = layer.weights.o_proj.values.T.contiguous().double()
    exact, magnitude = product(activated, w_out)
    slack = activated_off @ w_out.abs()
    slack = slack + (layer.width + 1) * 2.0**-23 * (magnitude + slack)
    if bias_out is not None:
        exact, slack = exact + bias_out.double(), slack + (layer.width + 1) * 2.0**-23 * bias_out.double().abs()
    near(out, exact, slack, "output")


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


KINDS = [(BF16, INTERLEAVED), (BF16, CONCATENATED), (BF16, None), (FP16, CONCATENATED), (FP32, INTERLEAVED), (FP32, None)]
ROWS = [1, 5, 9, 17, 70, 300, 1100]
NAMES = ("i_values", "o_values", "i_bias", "o_bias")


@pytest.mark.parametrize("dtype,order", KINDS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("hidden,width", [(136, 72), (61, 131)])
def test_fp32_gradients_of_any_layer(device, rows, hidden, width, dtype, order):
    """Weights' gradients kept in fp32, written and then added to."""

    layer = Layer(device, rows, hidden, width, dtype, function="gelu", order=order, bias=True)
    projected, _ = layer.forward()
    into = layer.gradients(kept=FP32)
    grad_x = layer.backward(projected, into)
    layer.check_backward(projected, grad_x, into)
    before = {name: getattr(into, name).clone() for name in NAMES}
    grad_x = layer.backward(projected, into, accumulate=True)
    layer.check_backward(projected, grad_x, into, before)


@pytest.mark.parametrize("dtype,order", KINDS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("hidden,width", [(136, 72), (61, 131)])
def test_gradients_asked_for_singly(device, rows, hidden, width, dtype, order):
    """None of the gradients, each by itself, and pairs of them."""

    layer = Layer(device, rows, hidden, width, dtype, order=order, limit=1.5 if order else None, bias=True)
    projected, _ = layer.forward()
    layer.dense.backward_into(hidden_states=layer.x, layer_weights=layer.weights, projected=projected, grad_output=layer.grad)
    layer.check_backward(projected, layer.backward(projected, None), DenseGradients())
    for wanted in [(name,) for name in NAMES] + [("i_values", "o_bias"), ("o_values", "i_bias"), ("i_bias", "o_bias")]:
        full = layer.gradients()
        into = DenseGradients(**{name: getattr(full, name) for name in wanted})
        layer.dense.training_scratch.fill_(0xFF)
        layer.dense.backward_into(hidden_states=layer.x, layer_weights=layer.weights, projected=projected, grad_output=layer.grad,
                                  gradients=into)
        layer.check_backward(projected, None, into)


@pytest.mark.parametrize("dtype,order", KINDS)
@pytest.mark.parametrize("hidden,width", [(136, 72), (61, 131)])
def test_layers_below_their_capacity(device, hidden, width, dtype, order):
    """One plan and workspace serve every number of rows, whatever the workspace held."""

    big = Layer(device, 1100, hidden, width, dtype, function="relu", order=order, bias=True)
    x, grad = big.x, big.grad
    for rows in (1, 2, 8, 9, 16, 17, 63, 65, 129, 300, 1023, 1024, 1025, 1099):
        big.rows, big.x, big.grad = rows, x[:rows], grad[:rows]
        found = []
        for fill in (0xFF, 0x00):
            big.dense.training_scratch.fill_(fill)
            projected, out = big.forward()
            into = big.gradients()
            found.append((projected, out, big.backward(projected, into), into.i_values, into.o_values, into.i_bias, into.o_bias))
        assert all(torch.equal(a, b) for a, b in zip(*found))
        check_forward(big, projected, out)
        big.check_backward(projected, found[0][2], into)


@pytest.mark.parametrize("dtype,order", KINDS)
@pytest.mark.parametrize("rows", [1, 5, 17, 150])
@pytest.mark.parametrize("hidden,width,strides", [(64, 40, (72, 160, 96, 80)), (61, 131, (64, 300, 61, 75)), (136, 8, (1000, 88, 136, 136))])
def test_layers_of_rows_any_stride_apart(device, rows, hidden, width, strides, dtype, order):
    """Hidden states, kept values, the output's gradient and the hidden states' gradient as columns of wider tensors."""

    layer = Layer(device, rows, hidden, width, dtype, order=order, bias=True)
    x, grad = layer.x, layer.grad
    layer.x = rows_of(x, strides[0])
    projected, out = layer.forward()
    layer.x = x
    check_forward(layer, projected, out)
    held = torch.full((rows, strides[3]), 7.0, dtype=dtype, device=device)
    grad_x, into = held[:, :hidden], layer.gradients()
    layer.dense.backward_into(
        hidden_states=rows_of(x, strides[0]), layer_weights=layer.weights, projected=rows_of(projected, strides[1]),
        grad_output=rows_of(grad, strides[2]), grad_hidden_states=grad_x, gradients=into)
    assert bool((held[:, hidden:] == 7.0).all())
    layer.check_backward(projected, grad_x, into)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [1022, 1023, 1024, 1025, 1026])
def test_sums_over_rows_at_once_and_in_bands(device, rows, dtype):
    """The biases' gradients where their kernel changes: of a projection, and of a layer whose two share their bands' place."""

    for k, n in ((264, 136), (61, 131)):
        case = Projection(device, rows, k, n, dtype, bias=True)
        grad_b = torch.full((n,), float("nan"), device=device)
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_bias=grad_b)
        case.check(None, None, grad_b)
        before = None, grad_b.clone()
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_bias=grad_b, accumulate=True)
        case.check(None, None, grad_b, before)
        for order in (INTERLEAVED, CONCATENATED):
            if dtype is FP32 and order is CONCATENATED:
                continue
            layer = Layer(device, rows, k, n, dtype, order=order, bias=True)
            projected, _ = layer.forward()
            into = layer.gradients()
            grad_x = layer.backward(projected, into)
            layer.check_backward(projected, grad_x, into)
            before = {name: getattr(into, name).clone() for name in NAMES}
            layer.backward(projected, into, accumulate=True)
            layer.check_backward(projected, None, into, before)


@pytest.mark.parametrize("rows", [5, 300])
def test_a_frozen_layer_in_a_graph(device, rows):
    """Hidden states' gradient alone, captured and replayed on other data with eager work between."""

    layer = Layer(device, rows, 264, 200, BF16, function="gelu_tanh", offset=0.5, bias=True)
    projected, _ = layer.forward()
    grad_x = torch.empty_like(layer.x)

    def run():
        layer.dense.backward_into(hidden_states=layer.x, layer_weights=layer.weights, projected=projected, grad_output=layer.grad,
                                  grad_hidden_states=grad_x)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in (1, 2, 3):
        layer.grad.copy_(Layer(device, rows, 264, 200, BF16, bias=True, seed=seed).grad)
        grad_x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = grad_x.clone()
        layer.check_backward(projected, grad_x, DenseGradients())
        run()
        assert torch.equal(replayed, grad_x)


@pytest.mark.parametrize("rows,dtype", [(511, FP32), (512, FP32), (512, BF16), (1279, BF16), (1280, BF16), (1279, FP16), (1280, FP16)])
def test_output_projections_of_odd_widths(device, rows, dtype):
    """Row counts where the output projection of a trained layer changes its kernel."""

    for hidden, width in ((136, 131), (61, 77)):
        layer = Layer(device, rows, hidden, width, dtype, function="gelu", order=INTERLEAVED, bias=True)
        projected, out = layer.forward()
        check_forward(layer, projected, out)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows", [0, 5, 150])
def test_frozen_weights_need_no_inputs(device, rows, dtype):
    """Without the gradient of a projection's values its inputs are not kept."""

    case = Projection(device, rows, 61, 131, dtype, bias=True)
    grad_x, grad_b = torch.full((rows, 61), float("nan"), dtype=dtype, device=device), torch.full((131,), float("nan"), device=device)
    case.gemm.backward_into(None, case.grad, case.weights, grad_inputs=grad_x, grad_bias=grad_b)
    case.check(grad_x, None, grad_b)
    with pytest.raises(ValueError, match="inputs"):
        case.gemm.backward_into(None, case.grad, case.weights, grad_values=torch.empty((131, 61), dtype=dtype, device=device))
    layer = Layer(device, rows, 136, 72, dtype, bias=True)
    projected, _ = layer.forward()
    full = layer.gradients()
    into, grad_x = DenseGradients(o_values=full.o_values, i_bias=full.i_bias, o_bias=full.o_bias), torch.empty_like(layer.x)
    layer.dense.backward_into(layer_weights=layer.weights, projected=projected, grad_output=layer.grad, grad_hidden_states=grad_x,
                              gradients=into)
    layer.check_backward(projected, grad_x, into)
    with pytest.raises(ValueError, match="hidden states"):
        layer.dense.backward_into(layer_weights=layer.weights, projected=projected, grad_output=layer.grad, gradients=full)
