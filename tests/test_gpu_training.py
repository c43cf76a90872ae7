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


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,k,n,strides", [
    (33, 72, 136, (80, 200, 96)), (64, 61, 35, (64, 37, 100)), (40, 128, 64, (4096, 64, 128)), (5, 30, 50, (31, 51, 33)),
    (1, 64, 48, (640, 480, 64)), (100, 257, 130, (300, 131, 257))])
def test_projection_gradients_of_rows_any_stride_apart(device, rows, k, n, strides, dtype):
    case = Projection(device, rows, k, n, dtype, bias=True)
    plain_x = case.x
    case.x, case.grad = rows_of(case.x, strides[0]), rows_of(case.grad, strides[1])
    held = torch.full((rows, strides[2]), 7.0, dtype=dtype, device=device)
    grad_x = held[:, :k]
    grad_w, grad_b = torch.empty((n, k), dtype=dtype, device=device), torch.empty(n, device=device)
    case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=grad_x, grad_values=grad_w, grad_bias=grad_b)
    assert bool((held[:, k:] == 7.0).all())  # what lies between the rows stays
    case.x, case.grad = plain_x, case.grad.contiguous()
    case.check(grad_x, grad_w, grad_b)


def test_gradients_are_written_alone_and_behind_nothing(device):
    """Each gradient by itself, in the middle of guarded memory."""

    rows, k, n = 45, 130, 70
    case = Projection(device, rows, k, n, BF16, bias=True, capacity=100)
    for name, shape, dtype in (("grad_inputs", (rows, k), BF16), ("grad_values", (n, k), BF16), ("grad_bias", (n,), FP32)):
        size = shape[0] if len(shape) == 1 else shape[0] * shape[1]
        flat = torch.full((size + 64,), 3.0, dtype=dtype, device=device)
        target = flat[32:32 + size].view(shape)
        case.gemm.backward_into(case.x, case.grad, case.weights, **{name: target})
        assert bool((flat[:32] == 3.0).all()) and bool((flat[32 + size:] == 3.0).all())
        case.check(*(target if name == each else None for each in ("grad_inputs", "grad_values", "grad_bias")))
    case.gemm.backward_into(case.x, case.grad, case.weights)  # nothing asked for


def test_every_row_count_below_the_capacity(device):
    """One workspace serves every number of rows, and a row's gradient does not depend on the workspace's contents."""

    k, n = 264, 200
    big = Projection(device, 300, k, n, BF16, bias=True)
    x, grad = big.x, big.grad
    for rows in (1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 299):
        big.x, big.grad = x[:rows], grad[:rows]
        results = []
        for fill in (0xFF, 0x00):
            big.gemm.scratch.fill_(fill)
            grad_x = torch.empty((rows, k), dtype=BF16, device=device)
            grad_w, grad_b = torch.empty((n, k), device=device), torch.empty(n, device=device)
            big.gemm.backward_into(big.x, big.grad, big.weights, grad_inputs=grad_x, grad_values=grad_w, grad_bias=grad_b)
            results.append((grad_x, grad_w, grad_b))
        assert all(torch.equal(a, b) for a, b in zip(*results))
        big.check(*results[0])


def test_no_rows(device):
    case = Projection(device, 8, 64, 48, BF16, bias=True)
    empty_x, empty_grad = case.x[:0], case.grad[:0]
    grad_w, grad_b = torch.ones((48, 64), dtype=BF16, device=device), torch.ones(48, device=device)
    case.gemm.backward_into(empty_x, empty_grad, case.weights, grad_inputs=torch.empty((0, 64), dtype=BF16, device=device),
                            grad_values=grad_w, grad_bias=grad_b, accumulate=True)
    assert bool((grad_w == 1).all()) and bool((grad_b == 1).all())
    case.gemm.backward_into(empty_x, empty_grad, case.weights, grad_values=grad_w, grad_bias=grad_b)
    assert bool((grad_w == 0).all()) and bool((grad_b == 0).all())
    layer = Layer(device, 8, 64, 40, BF16, bias=True)
    layer.rows, layer.x, layer.grad = 0, layer.x[:0], layer.grad[:0]
    projected, out = layer.forward()
    assert projected.shape == (0, 80) and out.shape == (0, 64)
    into = layer.gradients()
    layer.backward(projected, into)
    assert all(bool((t == 0).all()) for t in (into.i_values, into.o_values, into.i_bias, into.o_bias))


def test_bad_values_stay_in_their_rows_and_columns(device):
    """A NaN or infinity reaches what depends on it and nothing else, in tiles and beside ragged edges."""

    for rows, k, n in ((70, 72, 136), (70, 61, 131), (9, 72, 40)):
        case = Projection(device, rows, k, n, BF16, bias=True)
        case.grad[3, 5] = float("nan")
        case.x[rows - 1, k - 1] = float("inf")
        grad_x = torch.empty((rows, k), dtype=BF16, device=device)
        grad_w, grad_b = torch.empty((n, k), dtype=BF16, device=device), torch.empty(n, device=device)
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=grad_x, grad_values=grad_w, grad_bias=grad_b)
        assert bool(grad_x[3].isnan().all()) and not bool(grad_x[torch.arange(rows) != 3].isnan().any())
        assert bool(grad_w[5].isnan().all()) and not bool(grad_w[torch.arange(n) != 5, :k - 1].isnan().any())
        assert not bool(grad_w[torch.arange(n) != 5, k - 1].isfinite().any())
        assert bool(grad_b[5].isnan()) and not bool(grad_b[torch.arange(n) != 5].isnan().any())


@pytest.mark.parametrize("order", [INTERLEAVED, CONCATENATED], ids=["pairs", "halves"])
def test_clipped_and_bad_gates(device, order):
    """At the limit a value has its gradient, past it none; NaN is past no limit; an infinite gate is what it is in the
    activation and in its own gradient (-inf 0: NaN)."""

    layer = Layer(device, 6, 64, 40, BF16, function="silu", order=order, limit=1.0, bias=True)
    projected, _ = layer.forward()
    gate, up = layer.split(projected)
    gate[0], up[0] = 1.0, -1.0
    gate[1], up[1] = 1.5, 0.5
    gate[2], up[2] = 0.5, -1.5
    gate[3, 7], up[4, 9] = float("nan"), float("nan")
    gate[5], up[5] = float("-inf"), 0.25
    into = layer.gradients()
    grad_x = layer.backward(projected, into)
    assert bool(grad_x[3].isnan().all())
    # a NaN Up is in its Gate's gradient, which a clipped Gate does not have
    assert bool(grad_x[4].isnan().all()) == bool(gate[4, 9] <= 1.0) and bool(grad_x[:3].isfinite().all())
    apart = torch.empty((1, layer.wide), dtype=BF16, device=device)
    layer.signature.activation.backward_into(inputs=projected[5:6], grad_output=torch.ones((1, 40), dtype=BF16, device=device),
                                             grad_inputs=apart, order=order)
    assert bool(grad_x[5].isnan().all()) == bool(apart.isnan().any())
    layer.x, layer.grad, layer.rows = layer.x[:3].contiguous(), layer.grad[:3].contiguous(), 3
    kept = projected[:3].contiguous()
    grad_x = layer.backward(kept, into)
    layer.check_backward(kept, grad_x, into)


def test_offsets_past_32_bits(device):
    """Rows of operands and outputs beyond 2^31 elements from their begin."""

    rows, k, n = 2200, 64, 72
    stride = 1 << 20
    case = Projection(device, rows, k, n, BF16)
    base = torch.zeros(rows * stride, dtype=BF16, device=device)
    x = base.view(rows, stride)[:, 64:64 + k]
    x.copy_(case.x)
    grad = base.view(rows, stride)[:, 4096:4096 + n]
    grad.copy_(case.grad)
    grad_x = base.view(rows, stride)[:, 8192:8192 + k]
    grad_w = torch.empty((n, k), dtype=BF16, device=device)
    case.gemm.backward_into(x, grad, case.weights, grad_inputs=grad_x, grad_values=grad_w)
    case.check(grad_x, grad_w, None)
    del base


@pytest.mark.parametrize("rows", [12, 200])
def test_training_pass_in_a_graph(device, rows):
    """Forward and backward captured once and replayed on other data, with eager work between the replays."""

    layer = Layer(device, rows, 264, 200, BF16, function="gelu", bias=True)
    projected = torch.empty((rows, layer.wide), dtype=BF16, device=device)
    out = torch.empty((rows, layer.hidden), dtype=BF16, device=device)
    grad_x = torch.empty((rows, layer.hidden), dtype=BF16, device=device)
    into = layer.gradients()

    def run():
        layer.dense.run_into(hidden_states=layer.x, layer_weights=layer.weights, output=out, projected=projected)
        layer.dense.backward_into(hidden_states=layer.x, layer_weights=layer.weights, projected=projected, grad_output=layer.grad,
                                  grad_hidden_states=grad_x, gradients=into)

    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    run()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before  # no call allocates
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    targets = (projected, out, grad_x, into.i_values, into.o_values, into.i_bias, into.o_bias)
    for seed in (1, 2, 3):
        other = Layer(device, rows, 264, 200, BF16, function="gelu", bias=True, seed=seed)
        layer.x.copy_(other.x)
        layer.grad.copy_(other.grad)
        layer.weights.i_proj.values.copy_(other.weights.i_proj.values)
        for target in targets:
            target.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [target.clone() for target in targets]
        layer.check_forward(projected, out)
        layer.check_backward(projected, grad_x, into)
        run()
        assert all(torch.equal(a, b) for a, b in zip(replayed, targets))


def test_two_streams_with_their_own_scratch(device):
    layers = [Layer(device, 150, 512, 264, BF16, bias=True, seed=s) for s in (1, 2)]
    expected = []
    for layer in layers:
        projected, out = layer.forward()
        into = layer.gradients()
        expected.append((projected, out, layer.backward(projected, into), into.i_values, into.o_values, into.i_bias, into.o_bias))
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    found = [None, None]
    for _ in range(3):
        for index, (stream, layer) in enumerate(zip(streams, layers)):
            with torch.cuda.stream(stream):
                projected, out = layer.forward()
                into = layer.gradients()
                found[index] = (projected, out, layer.backward(projected, into), into.i_values, into.o_values, into.i_bias, into.o_bias)
    torch.cuda.synchronize()
    for wanted, got in zip(expected, found):
        assert all(torch.equal(a, b) for a, b in zip(wanted, got))


def test_gradients_against_differences(device):
    """Directional derivatives of the layer, by central differences of the formula in 64 bits.  fp32 gradients sum at most
    260 products: off by less than 2^-14 of their terms, and the directions' terms add up with random signs."""

    layer = Layer(device, 20, 64, 130, FP32, function="gelu", bias=True)
    projected, _ = layer.forward()
    into = layer.gradients()
    grad_x = layer.backward(projected, into)
    w = layer.weights
    leaves = [t.double() for t in (layer.x, w.i_proj.values, w.o_proj.values, w.i_proj.bias, w.o_proj.bias)]
    grads = [t.double() for t in (grad_x, into.i_values, into.o_values, into.i_bias, into.o_bias)]

    def loss(x, w_in, w_out, b_in, b_out):
        f, _, _, factor, _, _ = layer.terms(x @ w_in.T + b_in)
        return ((f * factor @ w_out.T + b_out) * layer.grad.double()).sum()

    g = torch.Generator(device=device).manual_seed(3)
    for index, grad in enumerate(grads):
        direction = torch.randn(grad.shape, generator=g, device=device, dtype=torch.float64)
        step = 1e-5
        sides = [loss(*(leaf + sign * step * direction if i == index else leaf for i, leaf in enumerate(leaves))) for sign in (1, -1)]
        difference = float((sides[0] - sides[1]) / (2 * step))
        allowed = 2.0**-14 * float((grad.abs() * direction.abs()).sum()) + 1e-6
        assert abs(difference - float((grad * direction).sum())) <= allowed


def test_frozen_layer_carries_adapter_gradients(device):
    """The gradient through a frozen projection is what an adapter's backward pass adds its own part to."""

    from crosspool_amd.adapters import Adapter, AdapterPlan, AdapterWeights

    case = Projection(device, 90, 256, 192, BF16)
    g = torch.Generator(device=device).manual_seed(5)
    a = (torch.randn((2, 8, 256), generator=g, device=device) / 16).to(BF16)
    b = (torch.randn((2, 192, 8), generator=g, device=device) / 3).to(BF16)
    ids = torch.randint(-1, 2, (90,), generator=g, device=device, dtype=torch.int32)
    plan = AdapterPlan.prepare(row_capacity=90, adapter_count=2, max_rank=8, input_width=256, output_width=192, dtype=BF16, backward=True)
    adapter = Adapter(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
    grad_x = torch.empty((90, 256), dtype=BF16, device=device)
    grad_a, grad_b = torch.empty_like(a), torch.empty_like(b)
    case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=grad_x)
    adapter.backward_into(case.x, case.grad, AdapterWeights(a, b), adapter_ids=ids, base=grad_x, grad_inputs=grad_x, grad_a=grad_a,
                          grad_b=grad_b)
    exact = case.grad.double() @ case.weights.values.double()
    for index in range(2):
        taken = (ids == index).double()[:, None]
        exact += taken * (case.grad.double() @ b[index].double() @ a[index].double())
    error = float((grad_x.double() - exact).norm() / exact.norm())
    assert error <= 3 * 2 * 2.0**-9  # two rounded stages, as in the adapters' own tests


def test_refusals(device):
    case = Projection(device, 16, 64, 48, BF16, bias=True)
    good = dict(grad_inputs=torch.empty((16, 64), dtype=BF16, device=device))
    with pytest.raises(ValueError, match="output gradient"):
        case.gemm.backward_into(case.x, case.grad.float(), case.weights, **good)
    with pytest.raises(ValueError, match="inputs"):
        case.gemm.backward_into(case.x[:8], case.grad, case.weights, **good)
    with pytest.raises(ValueError, match="prepared layout"):
        case.gemm.backward_into(torch.cat((case.x, case.x)), torch.cat((case.grad, case.grad)), case.weights)
    with pytest.raises(ValueError, match="contiguous"):
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=torch.empty((64, 16), dtype=BF16, device=device).T)
    with pytest.raises(ValueError, match="grad_values"):
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_values=torch.empty((48, 64), dtype=FP16, device=device))
    with pytest.raises(ValueError, match="bias"):
        case.gemm.backward_into(case.x, case.grad, ProjectionWeights(case.weights.values), **good)
    with pytest.raises(RuntimeError, match="16-byte"):
        wide = torch.zeros((16, 72), dtype=BF16, device=device)
        case.gemm.backward_into(wide[:, 1:65], case.grad, case.weights, grad_values=torch.empty((48, 64), dtype=BF16, device=device))
    with pytest.raises(RuntimeError, match="overlap"):
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=case.x,
                                grad_values=torch.empty((48, 64), dtype=BF16, device=device))
    forward_only = GemmPlan.prepare(
        input_layout=TensorLayout((16, 64), BF16), weight_layout=ProjectionLayout.of(case.weights),
        result_layout=TensorLayout((16, 48), BF16), activation=None)
    gemm = Gemm(forward_only, torch.empty(max(16, forward_only.workspace.nbytes), dtype=torch.uint8, device=device))
    with pytest.raises(ValueError, match="without backward"):
        gemm.backward_into(case.x, case.grad, case.weights, **good)
    layer = Layer(device, 16, 64, 40, BF16)
    projected, _ = layer.forward()
    with pytest.raises(ValueError, match="projected"):
        layer.backward(projected[:, :40], layer.gradients())
    with pytest.raises(ValueError, match="without a bias"):
        layer.backward(projected, DenseGradients(i_bias=torch.empty(80, device=device)))
    with pytest.raises(ValueError, match="i_proj gradient"):
        layer.backward(projected, DenseGradients(i_values=torch.empty((40, 64), dtype=BF16, device=device)))
    with pytest.raises(ValueError, match="projected"):
        layer.dense.run_into(hidden_states=layer.x, layer_weights=layer.weights, output=torch.empty_like(layer.x),
                             projected=torch.empty((16, 80), dtype=FP16, device=device))
    plan = DenseExecutionPlan.prepare(layer.signature)
    dense = Dense(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
    with pytest.raises(ValueError, match="without backward"):
        dense.run_into(hidden_states=layer.x, layer_weights=layer.weights, output=torch.empty_like(layer.x), projected=projected)


def test_the_forward_pass_of_a_trained_layer_is_the_served_one(device):
    """With `projected` a layer gives what it gives without, up to the rounding of the projection."""

    for function, order in (("silu", INTERLEAVED), ("gelu", CONCATENATED)):
        layer = Layer(device, 130, 256, 264, BF16, function=function, order=order)
        _, out = layer.forward()
        served = torch.empty_like(out)
        layer.dense.run_into(hidden_states=layer.x, layer_weights=layer.weights, output=served)
        error = float((out.double() - served.double()).norm() / served.double().norm())
        assert error <= 3 * 2.0**-9  # the projection's, the activation's and the output's half steps


# Sizes whose products take 256 x 256 tiles, both kinds of 128 x 128 ones, and 64 x 64 ones split along long sums, whole
# and with a remainder that is shared out; long sums over rows, and ragged edges of each.
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k,n", [
    (2048, 2560, 4096), (2100, 2048, 8200), (2100, 4096, 2048), (1100, 2056, 5000), (300, 1032, 4096), (8200, 520, 520),
    (8200, 1031, 1545), (9000, 2056, 2056)])
def test_large_projection_gradients(device, rows, k, n, dtype):
    case = Projection(device, rows, k, n, dtype, bias=True)
    apart_x, both_x = (torch.full((rows, k), float("nan"), dtype=dtype, device=device) for _ in range(2))
    apart_w, both_w = (torch.full((n, k), float("nan"), dtype=dtype, device=device) for _ in range(2))
    grad_b = torch.full((n,), float("nan"), device=device)
    case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=apart_x)
    case.gemm.backward_into(case.x, case.grad, case.weights, grad_values=apart_w)
    case.check(apart_x, apart_w, None)
    case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=both_x, grad_values=both_w, grad_bias=grad_b)
    case.check(both_x, both_w, grad_b)
    before = both_w.clone(), grad_b.clone()
    case.gemm.backward_into(case.x, case.grad, case.weights, grad_values=both_w, grad_bias=grad_b, accumulate=True)
    case.check(None, both_w, grad_b, before)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("function,order", [("silu", INTERLEAVED), ("gelu", CONCATENATED), ("gelu_tanh", None)])
@pytest.mark.parametrize("rows,hidden,width", [
    (2100, 2048, 4096), (2500, 2064, 1528), (520, 4096, 520), (4300, 2048, 4096), (777, 1030, 2053)])
def test_large_dense_training(device, rows, hidden, width, function, order, dtype):
    if dtype is FP32 and order is CONCATENATED:
        pytest.skip("gated fp32 layers are INTERLEAVED")
    layer = Layer(device, rows, hidden, width, dtype, function=function, order=order, bias=True)
    projected, out = layer.forward()
    layer.check_forward(projected, out)
    into = layer.gradients()
    grad_x = layer.backward(projected, into)
    layer.check_backward(projected, grad_x, into)
    before = {name: getattr(into, name).clone() for name in ("i_values", "o_values", "i_bias", "o_bias")}
    layer.backward(projected, into, accumulate=True)
    layer.check_backward(projected, None, into, before)


def test_large_gradients_are_the_same_every_time(device):
    """Sums have one order: whatever the scratch held, and in a graph replayed with other work between."""

    layer = Layer(device, 2100, 2048, 4096, BF16, bias=True)
    projected, _ = layer.forward()
    into = layer.gradients()
    expected = [layer.backward(projected, into)] + [t.clone() for t in (into.i_values, into.o_values, into.i_bias, into.o_bias)]
    again = layer.gradients()
    grad_x = torch.empty_like(expected[0])
    layer.dense.training_scratch.fill_(0xFF)

    def run():
        layer.dense.backward_into(hidden_states=layer.x, layer_weights=layer.weights, projected=projected, grad_output=layer.grad,
                                  grad_hidden_states=grad_x, gradients=again)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3):
        layer.dense.training_scratch.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        found = (grad_x, again.i_values, again.o_values, again.i_bias, again.o_bias)
        assert all(torch.equal(a, b) for a, b in zip(expected, found))
        for target in found:
            target.fill_(float("nan"))
        layer.backward(projected, into)


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,hidden,width", [(5, 64, 40), (70, 72, 131), (300, 1032, 520), (1100, 2048, 2056), (4100, 1024, 4096)])
def test_either_order_gives_the_same_layer(device, rows, hidden, width, dtype):
    """Halves and pairs of the same Gate and Up rows: the same sums, so the same bits."""

    pairs = Layer(device, rows, hidden, width, dtype, function="gelu", limit=1.5, offset=0.5, bias=True)
    halves = Layer(device, rows, hidden, width, dtype, function="gelu", order=CONCATENATED, limit=1.5, offset=0.5, bias=True)
    values, bias = pairs.weights.i_proj.values, pairs.weights.i_proj.bias
    halves.weights.i_proj.values.copy_(torch.cat((values[0::2], values[1::2])))
    halves.weights.i_proj.bias.copy_(torch.cat((bias[0::2], bias[1::2])))
    halves.weights.o_proj.values.copy_(pairs.weights.o_proj.values)
    halves.weights.o_proj.bias.copy_(pairs.weights.o_proj.bias)
    halves.x.copy_(pairs.x)
    kept_pairs, out_pairs = pairs.forward()
    kept_halves, out_halves = halves.forward()
    assert torch.equal(torch.cat((kept_pairs[:, 0::2], kept_pairs[:, 1::2]), 1), kept_halves)
    assert torch.equal(out_pairs, out_halves)


def test_halves_past_the_product_s_offsets(device):
    """Weights of 2 GiB in halves take the activation by itself."""

    rows, hidden, width = 3, 16384, 32768
    layer = Layer(device, rows, hidden, width, BF16, order=CONCATENATED)
    projected, out = layer.forward()
    layer.check_forward(projected, out)


def test_kept_values_and_outputs_lie_apart(device):
    """An output over the hidden states or the kept values would spoil what the backward pass reads: refused."""

    for dtype in (BF16, FP32):
        layer = Layer(device, 16, 64, 32, dtype)
        shared = torch.empty((16, 64), dtype=dtype, device=device)
        for projected, output in ((shared, shared), (shared, layer.x), (layer.x, shared)):
            with pytest.raises((ValueError, RuntimeError), match="overlap"):
                layer.dense.run_into(hidden_states=layer.x, layer_weights=layer.weights, output=output, projected=projected)


@pytest.mark.parametrize("rows,k,n", [(1 << 20, 8, 8), (1 << 18, 9, 5), (8, 1 << 20, 8), (20, 1 << 20, 3), (8, 8, 1 << 20), (20, 3, 1 << 20)])
def test_the_longest_rows_and_columns(device, rows, k, n):
    """One extent at its largest, the others small: sums of a million products and outputs of a million columns."""

    case = Projection(device, rows, k, n, BF16, bias=True)
    grad_x = torch.full((rows, k), float("nan"), dtype=BF16, device=device)
    grad_w = torch.full((n, k), float("nan"), device=device)
    grad_b = torch.full((n,), float("nan"), device=device)
    case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=grad_x, grad_values=grad_w, grad_bias=grad_b)
    case.check(grad_x, grad_w, grad_b)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows", [4, 8, 9, 16, 17, 895, 896, 897])
def test_borders_between_the_variants(device, rows, dtype):
    """Row counts where weights' gradients and sums over rows change their kernel, with aligned and odd widths."""

    for k, n in ((264, 136), (61, 131)):
        case = Projection(device, rows, k, n, dtype, bias=True)
        grad_x = torch.full((rows, k), float("nan"), dtype=dtype, device=device)
        grad_w = torch.full((n, k), float("nan"), dtype=dtype, device=device)
        grad_b = torch.full((n,), float("nan"), device=device)
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_inputs=grad_x, grad_values=grad_w, grad_bias=grad_b)
        case.check(grad_x, grad_w, grad_b)
        before = grad_w.clone(), grad_b.clone()
        case.gemm.backward_into(case.x, case.grad, case.weights, grad_values=grad_w, grad_bias=grad_b, accumulate=True)
        case.check(None, grad_w, grad_b, before)


@pytest.mark.parametrize("rows,dtype", [(5, BF16), (13, FP32), (950, FP16), (1500, BF16)])
def test_gradients_of_every_variant_in_a_graph(device, rows, dtype):
    """Few rows in one launch, biases at once and in bands: replayed with other work between, as they are eager."""

    layer = Layer(device, rows, 257, 131, dtype, bias=True)
    projected, _ = layer.forward()
    into, grad_x = layer.gradients(), torch.empty((rows, 257), dtype=dtype, device=device)
    targets = (grad_x, into.i_values, into.o_values, into.i_bias, into.o_bias)

    def run():
        layer.dense.backward_into(hidden_states=layer.x, layer_weights=layer.weights, projected=projected, grad_output=layer.grad,
                                  grad_hidden_states=grad_x, gradients=into)

    run()
    torch.cuda.synchronize()
    expected = [target.clone() for target in targets]
    layer.check_backward(projected, grad_x, into)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3):
        for target in targets:
            target.fill_(float("nan"))
        layer.dense.training_scratch.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(expected, targets))
        run()
