"""The gradient of the standalone activation, against torch's own in 64 bits.

Tolerance: the kernel evaluates sigmoids with the hardware's exp and reciprocal, relative error at most
2^-16 for any argument a 16-bit payload leads to (|x| 2^-23 of the exponent up to 88, 2^-22 besides), and
1 - sigmoid to 2^-22; every factor is a product of values of those, so the error is at most 2^-15 of
|dout| (|h| + 1) (1 + |alpha v|) times the sigmoid's magnitude, taken as 1 for v > 0 and through the tails
as f's own size; erff adds 2^-22 absolutely.  A sigmoid below fp32's smallest normal number becomes 0: it
was at most 2^-126, which stands beside the tail's own size (v = -88: sigmoid 6e-39, f' 88 times that).  The
store rounds once.
"""

from __future__ import annotations

import pytest
import torch

from crosspool_amd.ffn import GateTransform, GateUpOrder, GeluActivation, ReluActivation, SiluActivation
from crosspool_amd.operators import Activation

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTIVATIONS = {
    "silu": SiluActivation(), "silu_1.7": SiluActivation(1.7), "relu": ReluActivation(), "gelu": GeluActivation(),
    "gelu_tanh": GeluActivation("tanh"),
}


def evaluate(function, v):
    if isinstance(function, SiluActivation):
        return v * torch.sigmoid(function.alpha * v)
    if isinstance(function, GeluActivation):
        return torch.nn.functional.gelu(v, approximate=function.approximate)
    return torch.relu(v)


def split(values, order, width):
    if order is GateUpOrder.INTERLEAVED:
        return values[..., 0::2], values[..., 1::2]
    return values[..., :width], values[..., width:]


def expected_gradient(activation, inputs, grad, order):
    """(gradient in 64 bits, the magnitude its error is relative to)."""

    values = inputs.double().requires_grad_(True)
    width = grad.shape[-1]
    function, gate_transform = activation.function, activation.gate
    if gate_transform is None:
        out = evaluate(function, values)
        gate, factor = values.detach(), torch.ones_like(grad.double())
    else:
        gate, up = split(values, order, width)
        if gate_transform.limit is not None:
            gate, up = gate.clamp(max=gate_transform.limit), up.clamp(-gate_transform.limit, gate_transform.limit)
        factor = up + gate_transform.up_offset
        out = evaluate(function, gate) * factor
        gate, factor = gate.detach(), factor.detach()
    (found,) = torch.autograd.grad(out, values, grad.double())
    alpha = getattr(function, "alpha", 1.0)
    # The size of f and f' at v: at most 1 + |alpha v| above zero, that times the tail below.
    tail = torch.where(gate < 0, torch.sigmoid(alpha * gate), 1.0)
    if isinstance(function, GeluActivation):
        tail = torch.where(gate < 0, torch.special.ndtr(gate).clamp_min(2.0**-7), 1.0)  # erff: absolute
    size = grad.double().abs() * (1 + alpha * gate.abs()) * (tail + 2.0**-111)  # 2^-15 of it: 2^-126
    if gate_transform is None:
        return found, size
    magnitude = torch.zeros_like(found)
    for target, amount in zip(split(magnitude, order, width), (size * factor.abs(), size)):
        target.copy_(amount)
    return found, magnitude


def check(activation, inputs, grad, order, device):
    got = torch.full(inputs.shape, float("nan"), dtype=inputs.dtype, device=device)
    activation.backward_into(inputs=inputs.to(device), grad_output=grad.to(device), grad_inputs=got, order=order)
    value, size = expected_gradient(activation, inputs, grad, order)
    bound = size * 2.0**-15
    smallest = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}[inputs.dtype]
    allowed = bound + (value.abs() + bound) * torch.finfo(inputs.dtype).eps / 2 + smallest
    excess = (got.cpu().double() - value).abs() - allowed
    assert bool((excess <= 0).all()), f"{int((~(excess <= 0)).sum())} beyond the bound, worst by {float(excess.max()):.3e}"
    return got


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("name", list(ACTIVATIONS))
@pytest.mark.parametrize("order", [GateUpOrder.INTERLEAVED, GateUpOrder.CONCATENATED, None], ids=["pairs", "halves", "ungated"])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 7), (3, 8), (2, 13), (5, 129), (33, 1000), (257, 2053)])
def test_gradient_matches_the_definition(device, rows, width, order, name, dtype):
    g = torch.Generator().manual_seed(rows * width)
    wide = width if order is None else 2 * width
    inputs = (torch.randn((rows, wide), generator=g) * 3).to(DTYPES[dtype])
    grad = torch.randn((rows, width), generator=g).to(DTYPES[dtype])
    for gate in (None,) if order is None else (GateTransform(), GateTransform(2.0, 1.0)):
        check(Activation(ACTIVATIONS[name], gate), inputs, grad, order, device)


@pytest.mark.parametrize("name", list(ACTIVATIONS))
def test_every_finite_bf16_value(device, name):
    """All finite bf16 values as gate (up to where v^2 overflows in 64-bit-free formulas none is NaN)."""

    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    values = bits[bits.isfinite()]
    values = values[: values.numel() // 8 * 8].reshape(-1, 8)
    got = check(Activation(ACTIVATIONS[name], None), values, torch.ones_like(values), None, device)
    assert bool(got.isfinite().all())


def test_clipped_values_get_nothing_and_values_at_the_limit_do(device):
    inputs = torch.tensor([[2.0, 2.0], [2.015625, 1.0], [1.0, -2.0], [1.0, -2.015625]], dtype=torch.bfloat16, device=device)
    grad = torch.ones((4, 1), dtype=torch.bfloat16, device=device)
    out = torch.empty_like(inputs)
    activation = Activation(ReluActivation(), GateTransform(2.0))
    activation.backward_into(inputs=inputs, grad_output=grad, grad_inputs=out, order=GateUpOrder.INTERLEAVED)
    assert out.tolist() == [[2.0, 2.0], [0.0, 2.0], [-2.0, 1.0], [-2.0, 0.0]]


def test_gradient_matches_differences(device):
    """Differences of the framework's forward: fp16 outputs of size 1 rounded to 2^-11, halved steps of 1/8
    give 2^-11 / (1/4) = 2^-9 each way; the third derivative (below 1) leaves h^2 / 6."""

    activation = Activation(SiluActivation(), GateTransform())
    inputs = torch.tensor([[0.5, 1.0, -1.0, 0.75, 0.25, -0.5]], dtype=torch.float16, device=device)
    grad = torch.ones((1, 3), dtype=torch.float16, device=device)
    out = torch.empty_like(inputs)
    activation.backward_into(inputs=inputs, grad_output=grad, grad_inputs=out, order=GateUpOrder.CONCATENATED)

    def total(values):
        result = torch.empty((1, 3), dtype=torch.float16, device=device)
        activation.apply_into(inputs=values, output=result, order=GateUpOrder.CONCATENATED)
        return result.double().sum().item()

    h = 0.125
    for column in range(6):
        above, below = inputs.clone(), inputs.clone()
        above[0, column] += h
        below[0, column] -= h
        difference = (total(above) - total(below)) / (2 * h)
        assert abs(difference - out[0, column].item()) <= 2.0**-9 * 2 + h * h / 6 + 2.0**-11


def test_in_place_and_graph(device):
    g = torch.Generator().manual_seed(1)
    inputs = torch.randn((40, 66), generator=g).to(torch.bfloat16).to(device)
    grad = torch.randn((40, 33), generator=g).to(torch.bfloat16).to(device)
    for order in GateUpOrder:
        activation = Activation(SiluActivation(), GateTransform())
        expected = torch.empty_like(inputs)
        activation.backward_into(inputs=inputs, grad_output=grad, grad_inputs=expected, order=order)
        inplace = inputs.clone()
        activation.backward_into(inputs=inplace, grad_output=grad, grad_inputs=inplace, order=order)
        assert torch.equal(inplace, expected)
    flat = Activation(GeluActivation(), None)
    expected, over_grad = torch.empty_like(grad), grad.clone()
    flat.backward_into(inputs=inputs[:, :33].contiguous(), grad_output=grad, grad_inputs=expected, order=None)
    flat.backward_into(inputs=inputs[:, :33].contiguous(), grad_output=over_grad, grad_inputs=over_grad, order=None)
    assert torch.equal(over_grad, expected)
    activation = Activation(SiluActivation(), GateTransform())
    out = torch.empty_like(inputs)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        activation.backward_into(inputs=inputs, grad_output=grad, grad_inputs=out, order=GateUpOrder.INTERLEAVED)
    for seed in (2, 3):
        inputs.copy_(torch.randn((40, 66), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(inputs)
        activation.backward_into(inputs=inputs, grad_output=grad, grad_inputs=eager, order=GateUpOrder.INTERLEAVED)
        assert torch.equal(out, eager)


@pytest.mark.parametrize("order", [GateUpOrder.INTERLEAVED, GateUpOrder.CONCATENATED, None])
def test_as_many_values_as_a_call_takes(device, order):
    """2^31 outputs: the rows at both ends and in the middle are those of calls of their own."""

    rows, width = 1 << 16, 1 << 15
    wide = width if order is None else 2 * width
    activation = Activation(SiluActivation(), None if order is None else GateTransform())
    inputs = torch.zeros((rows, wide), dtype=torch.bfloat16, device=device)
    grad = torch.zeros((rows, width), dtype=torch.bfloat16, device=device)
    out = torch.full_like(inputs, 1.0)
    parts = [slice(0, 3), slice((1 << 15) - 2, (1 << 15) + 2), slice(rows - 3, rows)]
    for part in parts:
        inputs[part].normal_()
        grad[part].normal_()
    activation.backward_into(inputs=inputs, grad_output=grad, grad_inputs=out, order=order)
    for part in parts:
        own = torch.empty_like(inputs[part])
        activation.backward_into(inputs=inputs[part], grad_output=grad[part], grad_inputs=own, order=order)
        assert torch.equal(out[part], own) and bool(own.any())
    assert not bool(out[100:200].any())


def test_refusals(device):
    activation = Activation(SiluActivation(), GateTransform())
    inputs = torch.zeros((4, 16), dtype=torch.bfloat16, device=device)
    grad = torch.zeros((4, 8), dtype=torch.bfloat16, device=device)
    good = dict(inputs=inputs, grad_output=grad, grad_inputs=torch.empty_like(inputs), order=GateUpOrder.INTERLEAVED)
    for bad in (
        dict(good, order=None), dict(good, grad_output=grad.half()), dict(good, inputs=inputs.float()),
        dict(good, grad_inputs=torch.empty((4, 8), dtype=torch.bfloat16, device=device)),
        dict(good, grad_output=grad.t().contiguous().t()), dict(good, inputs=inputs.cpu()),
    ):
        with pytest.raises(ValueError):
            activation.backward_into(**bad)
    flat = torch.zeros(200, dtype=torch.bfloat16, device=device)
    with pytest.raises(RuntimeError, match="whole"):
        activation.backward_into(inputs=flat[:64].view(4, 16), grad_output=grad, grad_inputs=flat[8:72].view(4, 16),
                                 order=GateUpOrder.INTERLEAVED)
    empty = torch.empty((0, 16), dtype=torch.bfloat16, device=device)
    activation.backward_into(inputs=empty, grad_output=empty[:, :8].contiguous(), grad_inputs=empty, order=GateUpOrder.INTERLEAVED)


NAN, INFINITY = float("nan"), float("inf")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("name", list(ACTIVATIONS))
@pytest.mark.parametrize("order", [GateUpOrder.INTERLEAVED, GateUpOrder.CONCATENATED], ids=["pairs", "halves"])
@pytest.mark.parametrize("limit", [None, 2.0])
def test_nan_reaches_the_gradients_of_its_pair(device, limit, order, name, dtype):
    """A NaN Gate gives NaN for both, a NaN Up for the Gate's (its factor) while Up's own is dout f(g); a NaN in
    the output's gradient gives NaN for both.  A limit clips infinities, not NaN."""

    gate = torch.tensor([[1.0, NAN, 0.5, 1.0, NAN, INFINITY, 1.0, 0.5]])
    up = torch.tensor([[1.0, 1.0, NAN, -0.5, NAN, 1.0, -INFINITY, 0.5]])
    grad = torch.tensor([[1.0, 1.0, 1.0, NAN, 1.0, 1.0, 1.0, 2.0]]).to(DTYPES[dtype])
    inputs = torch.stack((gate, up), dim=2).flatten(1) if order is GateUpOrder.INTERLEAVED else torch.cat((gate, up), dim=1)
    got = torch.zeros(inputs.shape, dtype=DTYPES[dtype], device=device)
    Activation(ACTIVATIONS[name], GateTransform(limit, 1.0)).backward_into(
        inputs=inputs.to(DTYPES[dtype]).to(device), grad_output=grad.to(device), grad_inputs=got, order=order)
    grad_gate, grad_up = split(got.cpu().float(), order, 8)
    assert grad_gate.isnan().tolist() == [[False, True, True, True, True, False, False, False]]
    assert grad_up.isnan().tolist() == [[False, True, False, True, True, False, False, False]]
    # A finite Gate beside a NaN Up: dout f(g), as beside any other Up.
    assert torch.equal(grad_up[0, 2], grad_up[0, 7] / 2)
    if limit is None:
        # f(inf) = inf, f'(inf) = 1 and h = 2; an infinite Up makes the Gate's gradient infinite.
        assert grad_up[0, 5] == INFINITY and grad_gate[0, 5] == 2.0
        assert grad_gate[0, 6] == -INFINITY
    else:
        # Clipped: the Gate's gradient and the Up's are zero, the other factors those at the limit.
        assert grad_gate[0, 5] == 0.0 and grad_up[0, 6] == 0.0
        assert bool(grad_up[0, 5].isfinite()) and grad_up[0, 5] > 0 and bool(grad_gate[0, 6].isfinite())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("name", list(ACTIVATIONS))
def test_nan_and_infinity_of_ungated_values(device, name, dtype):
    values = torch.tensor([[NAN, INFINITY, 1.0, 0.0]], dtype=DTYPES[dtype], device=device)
    grad = torch.tensor([[1.0, 1.0, NAN, 1.0]], dtype=DTYPES[dtype], device=device)
    out = torch.zeros_like(values)
    Activation(ACTIVATIONS[name], None).backward_into(inputs=values, grad_output=grad, grad_inputs=out, order=None)
    assert out.isnan().tolist() == [[True, False, True, False]]
    assert out[0, 1] == 1.0 and out[0, 3] == (0.0 if name == "relu" else 0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("order", [GateUpOrder.INTERLEAVED, GateUpOrder.CONCATENATED], ids=["pairs", "halves"])
def test_tails_keep_their_relative_accuracy(device, order, name, dtype):
    """Gates from -8 to -3, where f and f' are down to 1e-14, relative to the sizes of their own terms.

    erf form: the argument v / sqrt 2 is off by 2^-23 relatively, and (v^2 + 2) is how much more its
    complementary error function is; exp(-v^2 / 2) likewise, with the exponent's product by log2 e rounded
    once more: (v^2 + 2) 2^-22 covers both.  tanh form: sigmoid(2 y) with 2 y off by four roundings and the exponent's
    product: (|2 y| + 2) 2^-21.  SiLU: (|v| + 2) 2^-21 the same way.  The library's complementary error
    function and the hardware's exp and reciprocal add units in the last place: 2^-20.
    """

    g = torch.Generator().manual_seed(3)
    rows, width = 64, 129
    gate = (torch.rand((rows, width), generator=g) * -5 - 3).to(DTYPES[dtype])
    up = torch.randn((rows, width), generator=g).to(DTYPES[dtype])
    # fp16 outputs of 1e-14 would round to zero: gradients as large as a loss scale makes them.
    grad = (torch.rand((rows, width), generator=g) + 0.5).mul(1.0 if dtype == "bf16" else 2.0**14).to(DTYPES[dtype])
    inputs = torch.stack((gate, up), dim=2).flatten(1) if order is GateUpOrder.INTERLEAVED else torch.cat((gate, up), dim=1)
    got = torch.full(inputs.shape, NAN, dtype=DTYPES[dtype], device=device)
    Activation(ACTIVATIONS[name], GateTransform()).backward_into(
        inputs=inputs.to(device), grad_output=grad.to(device), grad_inputs=got, order=order)
    v, u, d = gate.double(), up.double(), grad.double()
    if name == "gelu":
        share, density = 0.5 * torch.special.erfc(-v * 2**-0.5), torch.exp(-v * v / 2) * (2 * torch.pi) ** -0.5
        terms, relative = (share, v * density), (v * v + 2) * 2.0**-22 + 2.0**-20
    elif name == "gelu_tanh":
        c = (2 / torch.pi) ** 0.5
        twice = 2 * c * (v + 0.044715 * v**3)
        share = torch.sigmoid(twice)
        terms = (share, v * share * torch.sigmoid(-twice) * 2 * c * (1 + 3 * 0.044715 * v * v))
        relative = (twice.abs() + 2) * 2.0**-21 + 2.0**-20
    else:
        share = torch.sigmoid(v)
        terms, relative = (share, v * share * torch.sigmoid(-v)), (v.abs() + 2) * 2.0**-21 + 2.0**-20
    smallest = {"bf16": 2.0**-134, "fp16": 2.0**-25}[dtype]
    for actual, value, size in zip(
        split(got.cpu().double(), order, width), (d * u * (terms[0] + terms[1]), d * v * share),
        ((d * u).abs() * (terms[0].abs() + terms[1].abs()), (d * v * share).abs()),
    ):
        bound = size * relative
        allowed = bound + (value.abs() + bound) * torch.finfo(DTYPES[dtype]).eps / 2 + smallest
        excess = (actual - value).abs() - allowed
        assert bool((excess <= 0).all()), f"{int((~(excess <= 0)).sum())} beyond the bound"
