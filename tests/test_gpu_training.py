"""Gradients of projections and of a Dense layer on the GPU, against the formulas in 64 bits.

Tolerances, derived before the first run.  A sum of n products in fp32 is off by at most n 2^-23 of the sum of their
magnitudes (2^-24 for every addition, twice that for accumulators that truncate), and a result rounded to its dtype by
half a step of its value, ``finfo.eps / 2`` (and half a subnormal step).  What is rounded between two products (the gradient
of the projected values, the activated values) carries half a step of itself into the next sum, and the
16-bit activations' values and slopes are within 2^-14 of their terms.  Every check is element by element.
"""

from __future__ import annotations

import pytest
import torch

from crosspool_amd.ffn import GateTransform, GateUpOrder, GeluActivation, ReluActivation, SiluActivation
from crosspool_amd.operators import (
    Activation,
    Dense,
    DenseExecutionPlan,
    DenseGradients,
    DenseSignature,
    Gemm,
    GemmPlan,
    ProjectionLayout,
    TensorLayout,
)
from crosspool_amd.weights import DenseFfnWeights, ProjectionWeights

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ACT = {BF16: 2.0**-14, FP16: 2.0**-14, FP32: 2.0**-20}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def near(actual, expected, slack, what):
    """|actual - expected| <= half a step of the result + what its inputs and sums may be off by (64 bits)."""

    assert actual.shape == expected.shape, what
    allowed = half_step(actual.dtype) * (expected.abs() + slack) + tiny(actual.dtype) + slack
    error = (actual.double() - expected).abs()
    over = error > allowed
    over |= ~torch.isfinite(actual.double())
    assert not bool(over.any()), (
        f"{what}: {int(over.sum())} of {over.numel()} values off, first at {torch.nonzero(over)[0].tolist()}, "
        f"worst {float((error / allowed.clamp(min=1e-300)).max()):.2f} of the tolerance"
    )


def product(a, b):
    """a @ b in 64 bits, and the magnitudes' sum."""

    a, b = a.double(), b.double()
    return a @ b, a.abs() @ b.abs()


def rows_of(tensor, stride, fill=float("nan")):
    """The same rows `stride` elements apart, something else between them."""

    if stride is None:
        return tensor
    wide = torch.full((tensor.shape[0], stride), fill, dtype=tensor.dtype, device=tensor.device)
    wide[:, :tensor.shape[1]] = tensor
    return wide[:, :tensor.shape[1]]


class Projection:
    def __init__(self, device, rows, k, n, dtype, *, bias=False, capacity=None, seed=0):
        g = torch.Generator(device=device).manual_seed(seed + rows * 7 + k * 3 + n)
        self.x = torch.randn((rows, k), generator=g, device=device).to(dtype)
        self.grad = (torch.randn((rows, n), generator=g, device=device) * 0.05).to(dtype)
        values = (torch.randn((n, k), generator=g, device=device) * k**-0.5).to(dtype)
        self.weights = ProjectionWeights(values, bias=torch.randn(n, generator=g, device=device) if bias else None)
        plan = GemmPlan.prepare(
            input_layout=TensorLayout((capacity or max(rows, 1), k), dtype), weight_layout=ProjectionLayout.of(self.weights),
            result_layout=TensorLayout((capacity or max(rows, 1), n), dtype), activation=None, backward=True)
        self.gemm = Gemm(plan, torch.full((plan.workspace.nbytes,), 0xFF, dtype=torch.uint8, device=device))

    def check(self, grad_x, grad_w, grad_bias, before=None):
        rows, n = self.grad.shape
        if grad_x is not None:
            exact, magnitude = product(self.grad, self.weights.values)
            near(grad_x, exact, n * 2.0**-23 * magnitude, "input gradient")
        if grad_w is not None:
            exact, magnitude = product(self.grad.T.contiguous(), self.x)
            if before is not None:
                exact, magnitude = exact + before[0].double(), magnitude + before[0].double().abs()
            near(grad_w, exact, (rows + 1) * 2.0**-23 * magnitude, "weight gradient")
        if grad_bias is not None:
            exact, magnitude = self.grad.double().sum(0), self.grad.double().abs().sum(0)
            if before is not None:
                exact, magnitude = exact + before[1].double(), magnitude + before[1].double().abs()
            near(grad_bias, exact, (rows + 1) * 2.0**-23 * magnitude, "bias gradient")


SIZES = [(1, 8, 8), (1, 1, 1), (2, 3, 5), (7, 64, 64), (33, 72, 136), (64, 128, 256), (65, 257, 129), (130, 264, 520),
         (300, 1030, 517), (257, 512, 768), (700, 1536, 1536), (1000, 136, 2056), (5, 6144, 2048), (2100, 320, 192)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_projection_gradients(device, rows, k, n, dtype):
    case = Projection(device, rows, k, n, dtype, bias=True)
    for kept in {dtype, FP32}:
        grad_x = torch.full((rows, k), float("nan"), dtype=dtype, device=device)
        grad_w = torch.full((n, k), float("nan"), dtype=kept, device=device)
        grad_b = torch.full((n,), float("nan"), device=device)
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=grad_x, grad_values=grad_w, grad_bias=grad_b)
        case.check(grad_x, grad_w, grad_b)
        before = grad_w.clone(), grad_b.clone()
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_values=grad_w, grad_bias=grad_b, accumulate=True)
        case.check(None, grad_w, grad_b, before)


class Layer:
    FUNCTIONS = {"silu": SiluActivation(), "gelu": GeluActivation(), "gelu_tanh": GeluActivation("tanh"), "relu": ReluActivation()}

    def __init__(self, device, rows, hidden, width, dtype, *, function="silu", order=GateUpOrder.INTERLEAVED, limit=None,
                 offset=0.0, bias=False, capacity=None, seed=0):
        g = torch.Generator(device=device).manual_seed(seed + rows * 7 + hidden * 3 + width)

        def normal(*shape, std=1.0):
            return (torch.randn(shape, generator=g, device=device) * std).to(dtype)

        self.gated = order is not None
        self.order, self.function, self.limit, self.offset = order, function, limit, offset
        self.rows, self.hidden, self.width, self.wide = rows, hidden, width, width * (2 if self.gated else 1)
        self.dtype, self.device = dtype, device
        self.x, self.grad = normal(rows, hidden), normal(rows, hidden, std=0.05)
        biases = [torch.randn(size, generator=g, device=device) * 0.1 if bias else None for size in (self.wide, hidden)]
        self.weights = DenseFfnWeights(
            ProjectionWeights(normal(self.wide, hidden, std=hidden**-0.5), bias=biases[0]),
            ProjectionWeights(normal(hidden, width, std=width**-0.5), bias=biases[1]))
        activation = Activation(self.FUNCTIONS[function], GateTransform(limit, offset) if self.gated else None)
        self.signature = DenseSignature(
            payload_dtype=dtype, payload_row_capacity=capacity or max(rows, 1), hidden_size=hidden, local_intermediate_size=width,
            activation=activation, i_proj=ProjectionLayout.of(self.weights.i_proj, order=order),
            o_proj=ProjectionLayout.of(self.weights.o_proj))
        self.plan = DenseExecutionPlan.prepare(self.signature, backward=True)
        self.dense = Dense(self.plan, torch.full((self.plan.workspace.nbytes,), 0xFF, dtype=torch.uint8, device=device))

    def split(self, values):
        if self.order is GateUpOrder.INTERLEAVED:
            return values[:, 0::2], values[:, 1::2]
        return (values[:, :self.width], values[:, self.width:]) if self.gated else (values, None)

    def join(self, gate, up):
        if not self.gated:
            return gate
        return torch.stack((gate, up), 2).flatten(1) if self.order is GateUpOrder.INTERLEAVED else torch.cat((gate, up), 1)

    def terms(self, values):
        """f, f' and their terms' magnitudes, and the up factor, of kept values in 64 bits."""

        gate, up = self.split(values.double())
        v = gate.clamp(max=self.limit) if self.limit else gate
        if self.function == "silu":
            s = torch.sigmoid(v)
            f, slope, size = v * s, s * (1 + v * (1 - s)), s * (1 + (v * (1 - s)).abs())
        elif self.function == "relu":
            f, slope = v.clamp(min=0), (v > 0).double()
            size = slope
        elif self.function == "gelu":
            s = torch.special.ndtr(v)
            d = v * torch.exp(-0.5 * v * v) * 0.3989422804014327
            f, slope, size = v * s, s + d, s + d.abs()
        else:
            s = torch.sigmoid(2 * 0.7978845608028654 * (v + 0.044715 * v**3))
            d = v * s * (1 - s) * 2 * 0.7978845608028654 * (1 + 3 * 0.044715 * v * v)
            f, slope, size = v * s, s + d, s + d.abs()
        if up is None:
            return f, slope, size, None, None, None
        factor = (up.clamp(-self.limit, self.limit) if self.limit else up) + self.offset
        gate_on = (gate <= self.limit) if self.limit else torch.ones_like(gate, dtype=torch.bool)
        up_on = (up.abs() <= self.limit) if self.limit else torch.ones_like(gate, dtype=torch.bool)
        return f, slope, size, factor, gate_on, up_on

    def check_forward(self, projected, out):
        bias_in, bias_out = self.weights.i_proj.bias, self.weights.o_proj.bias
        exact, magnitude = product(self.x, self.weights.i_proj.values.T.contiguous())
        if bias_in is not None:
            exact, magnitude = exact + bias_in.double(), magnitude + bias_in.double().abs()
        near(projected, exact, (self.hidden + 1) * 2.0**-23 * magnitude, "projected")
        f, _, _, factor, _, _ = self.terms(projected)  # of the values that were kept
        activated = f if factor is None else f * factor
        off = activated.abs() * (half_step(self.dtype) + 2.0**-20)
        exact, magnitude = product(activated, self.weights.o_proj.values.T.contiguous())
        slack = off @ self.weights.o_proj.values.T.contiguous().double().abs() + (self.width + 1) * 2.0**-23 * magnitude
        slack += tiny(self.dtype) * self.weights.o_proj.values.double().abs().sum(1)
        if bias_out is not None:
            exact, slack = exact + bias_out.double(), slack + (self.width + 1) * 2.0**-23 * bias_out.double().abs()
        near(out, exact, slack, "output")

    def check_backward(self, projected, grad_x, into, before=None):
        h, act = half_step(self.dtype), ACT[self.dtype]
        w_in, w_out = self.weights.i_proj.values.double(), self.weights.o_proj.values.double()
        grad, x = self.grad.double(), self.x.double()
        d, d_size = product(grad, w_out)
        d_off = self.hidden * 2.0**-23 * d_size
        f, slope, size, factor, gate_on, up_on = self.terms(projected)
        if factor is None:
            through, off = d * slope, d_off * slope.abs() + (d.abs() + d_off) * size * act
            activated = f
        else:
            gate, up = d * slope * factor, d * f
            gate_off = (d_off * slope.abs() + (d.abs() + d_off) * size * act) * factor.abs()
            up_off = (d_off + (d.abs() + d_off) * act) * f.abs()
            through = self.join(gate * gate_on, up * up_on)
            off = self.join(gate_off * gate_on, up_off * up_on)
            activated = f * factor
        rounded = off + h * (through.abs() + off) + tiny(self.dtype)  # how far the stored gradient may be off
        activated_off = activated.abs() * (h + act) + tiny(self.dtype)
        fp32 = lambda count, a, b: count * 2.0**-23 * (a.abs() @ b.abs())  # noqa: E731
        if grad_x is not None:
            near(grad_x, through @ w_in, rounded @ w_in.abs() + fp32(self.wide, through.abs() + rounded, w_in), "hidden gradient")
        names = ("i_values", "o_values", "i_bias", "o_bias")
        held = {name: (0.0 if before is None or getattr(into, name) is None else before[name].double()) for name in names}
        if into.i_values is not None:
            t = through.T.contiguous()
            slack = rounded.T.contiguous() @ x.abs() + fp32(self.rows + 1, t.abs() + rounded.T, x)
            near(into.i_values, t @ x + held["i_values"], slack + 2.0**-23 * abs(held["i_values"]), "i_proj gradient")
        if into.o_values is not None:
            t = grad.T.contiguous()
            slack = t.abs() @ activated_off + fp32(self.rows + 1, t, activated.abs() + activated_off)
            near(into.o_values, t @ activated + held["o_values"], slack + 2.0**-23 * abs(held["o_values"]), "o_proj gradient")
        if into.i_bias is not None:
            slack = off.sum(0) + (self.rows + 1) * 2.0**-23 * (through.abs() + off).sum(0)
            near(into.i_bias, through.sum(0) + held["i_bias"], slack + 2.0**-23 * abs(held["i_bias"]), "i_proj bias gradient")
        if into.o_bias is not None:
            slack = (self.rows + 1) * 2.0**-23 * grad.abs().sum(0)
            near(into.o_bias, grad.sum(0) + held["o_bias"], slack + 2.0**-23 * abs(held["o_bias"]), "o_proj bias gradient")

    def gradients(self, kept=None, bias=True):
        kept = kept or self.dtype
        empty = lambda shape, dtype: torch.full(shape, float("nan"), dtype=dtype, device=self.device)  # noqa: E731
        bias = bias and self.weights.i_proj.bias is not None
        return DenseGradients(empty((self.wide, self.hidden), kept), empty((self.hidden, self.width), kept),
                              empty((self.wide,), FP32) if bias else None, empty((self.hidden,), FP32) if bias else None)

    def forward(self):
        projected = torch.full((self.rows, self.wide), float("nan"), dtype=self.dtype, device=self.device)
        out = torch.full((self.rows, self.hidden), float("nan"), dtype=self.dtype, device=self.device)
        self.dense.run_into(hidden_states=self.x, layer_weights=self.weights, output=out, projected=projected)
        return projected, out

    def backward(self, projected, into, accumulate=False):
        grad_x = torch.full((self.rows, self.hidden), float("nan"), dtype=self.dtype, device=self.device)
        self.dense.backward_into(hidden_states=self.x, layer_weights=self.weights, projected=projected, grad_output=self.grad,
                                 grad_hidden_states=grad_x, gradients=into, accumulate=accumulate)
        return grad_x


INTERLEAVED, CONCATENATED = GateUpOrder.INTERLEAVED, GateUpOrder.CONCATENATED
LAYERS = [
    ("silu", INTERLEAVED, None, 0.0), ("silu", CONCATENATED, 1.0, 1.0), ("gelu", INTERLEAVED, 1.5, 0.0),
    ("gelu_tanh", CONCATENATED, None, 0.0), ("relu", INTERLEAVED, None, 0.5), ("silu", None, None, 0.0),
    ("gelu", None, None, 0.0), ("relu", None, None, 0.0),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("function,order,limit,offset", LAYERS)
@pytest.mark.parametrize("rows,hidden,width", [(1, 64, 64), (3, 5, 3), (70, 136, 200), (150, 257, 131), (260, 512, 384)])
def test_dense_training(device, rows, hidden, width, function, order, limit, offset, dtype):
    if dtype is FP32 and order is CONCATENATED:
        pytest.skip("gated fp32 layers are INTERLEAVED")
    layer = Layer(device, rows, hidden, width, dtype, function=function, order=order, limit=limit, offset=offset, bias=True)
    projected, out = layer.forward()
    layer.check_forward(projected, out)
    into = layer.gradients()
    grad_x = layer.backward(projected, into)
    layer.check_backward(projected, grad_x, into)
    before = {name: getattr(into, name).clone() for name in ("i_values", "o_values", "i_bias", "o_bias")}
    grad_x = layer.backward(projected, into, accumulate=True)
    layer.check_backward(projected, grad_x, into, before)
