"""The adapter, activation-gradient and balance operators as they are used together.

Serving: the operator layer's Dense with an adapter pool beside each projection.  Fine-tuning: one step of a
layer's adapters, forward through Gemm, Adapter and Activation and backward through their gradients,
against torch's own gradients of the same layer in 64 bits.

Tolerances: every stage rounds its 16-bit output once (half a step, 2^-9 in bf16), and a following linear stage
carries an input's relative error on in the 2-norm, so after s rounded stages the relative 2-norm is at most
about s 2^-9 times the stage's gain over its result, which is near 1 for the random operands used here; each
check allows three times s 2^-9.
"""

from __future__ import annotations

import pytest
import torch

from crosspool_amd import _native
from crosspool_amd.adapters import Adapter, AdapterPlan, AdapterWeights, DenseAdapterWeights
from crosspool_amd.ffn import GateTransform, GateUpOrder, GeluActivation, ReluActivation, SiluActivation
from crosspool_amd.moe import BalanceLoss, MoeRouterWeights, Router
from crosspool_amd.operators import (
    Activation,
    Dense,
    DenseAdapterLayout,
    DenseExecutionPlan,
    DenseSignature,
    Gemm,
    GemmPlan,
    ProjectionLayout,
    TensorLayout,
)
from crosspool_amd.weights import DenseFfnWeights, ProjectionWeights

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0**-9, torch.float16: 2.0**-12, torch.float32: 2.0**-20}


def near(actual, expected, stages, what):
    step = STEP[actual.dtype]
    actual, expected = actual.cpu().double(), expected.detach().cpu().double()
    error = float((actual - expected).norm() / expected.norm())
    assert error <= 3 * stages * step, f"{what}: relative error {error:.2e} above {3 * stages * step:.2e}"


class Layer:
    def __init__(self, device, *, rows, hidden, width, count, rank, dtype, order=GateUpOrder.INTERLEAVED, gated=True,
                 bias=False, seed=0):
        g = torch.Generator().manual_seed(seed)
        wide = 2 * width if gated else width

        def normal(*shape, std):
            return (torch.randn(shape, generator=g) * std).to(dtype)

        self.x = normal(rows, hidden, std=1.0)
        self.w_in, self.w_out = normal(wide, hidden, std=hidden**-0.5), normal(hidden, width, std=width**-0.5)
        self.bias = torch.randn(wide, generator=g) * 0.1 if bias else None
        self.a_in, self.b_in = normal(count, rank, hidden, std=hidden**-0.5), normal(count, wide, rank, std=rank**-0.5)
        self.a_out, self.b_out = normal(count, rank, width, std=width**-0.5), normal(count, hidden, rank, std=rank**-0.5)
        self.scales = torch.rand(count, generator=g) + 0.5
        self.ids = torch.randint(-1, count, (rows,), generator=g, dtype=torch.int32)
        self.order, self.gated, self.device, self.dtype = order, gated, device, dtype
        self.rows, self.hidden, self.width, self.wide, self.count, self.rank = rows, hidden, width, wide, count, rank

    def adapted(self, x, w, a, b, bias=None):
        """x w^T (+ bias) plus the rows' adapters, in 64 bits."""

        out = x @ w.double().T
        if bias is not None:
            out = out + bias.double()
        for adapter in range(self.count):
            taken = ((self.ids == adapter).double() * float(self.scales[adapter]))[:, None]
            out = out + taken * (x @ a[adapter].T @ b[adapter].T)
        return out

    def forward(self, x, function, adapters):
        a_in, b_in, a_out, b_out = adapters
        projected = self.adapted(x, self.w_in, a_in, b_in, self.bias)
        if self.gated:
            if self.order is GateUpOrder.INTERLEAVED:
                gate, up = projected[:, 0::2], projected[:, 1::2]
            else:
                gate, up = projected[:, :self.width], projected[:, self.width:]
            activated = function(gate) * up
        else:
            activated = function(projected)
        return self.adapted(activated, self.w_out, a_out, b_out)


FUNCTIONS = {"silu": (SiluActivation(), torch.nn.functional.silu), "gelu": (GeluActivation(), torch.nn.functional.gelu),
             "relu": (ReluActivation(), torch.relu)}


@pytest.mark.parametrize("dtype,order,gated,name,bias", [
    (torch.bfloat16, GateUpOrder.INTERLEAVED, True, "silu", False),
    (torch.bfloat16, GateUpOrder.CONCATENATED, True, "gelu", True),
    (torch.float16, GateUpOrder.INTERLEAVED, True, "gelu", True),
    (torch.float16, None, False, "relu", False),
    (torch.float32, GateUpOrder.INTERLEAVED, True, "silu", False),
], ids=["bf16_silu", "bf16_gelu_halves_bias", "fp16_gelu_bias", "fp16_relu_ungated", "fp32_silu"])
@pytest.mark.parametrize("rows", [1, 7, 64, 150])
def test_dense_with_adapters(device, rows, dtype, order, gated, name, bias):
    layer = Layer(device, rows=rows, hidden=192, width=272, count=3, rank=8, dtype=dtype, order=order, gated=gated,
                  bias=bias, seed=rows)
    spec, function = FUNCTIONS[name]
    weights = DenseFfnWeights(
        i_proj=ProjectionWeights(layer.w_in.to(device), bias=None if layer.bias is None else layer.bias.to(device)),
        o_proj=ProjectionWeights(layer.w_out.to(device)),
    )
    signature = DenseSignature(
        payload_dtype=dtype, payload_row_capacity=160, hidden_size=layer.hidden, local_intermediate_size=layer.width,
        activation=Activation(spec, GateTransform() if gated else None),
        i_proj=ProjectionLayout.of(weights.i_proj, order=order), o_proj=ProjectionLayout.of(weights.o_proj),
    )
    to = lambda t: t.to(device)  # noqa: E731
    both = DenseAdapterWeights(AdapterWeights(to(layer.a_in), to(layer.b_in), to(layer.scales)),
                               AdapterWeights(to(layer.a_out), to(layer.b_out), to(layer.scales)))
    adapters = tuple(t.double() for t in (layer.a_in, layer.b_in, layer.a_out, layer.b_out))
    zero = tuple(torch.zeros_like(t) for t in adapters)
    for chosen, used in ((both, adapters), (DenseAdapterWeights(both.i_proj, None), adapters[:2] + zero[2:]),
                         (DenseAdapterWeights(None, both.o_proj), zero[:2] + adapters[2:])):
        plan = DenseExecutionPlan.prepare(signature, adapters=DenseAdapterLayout(
            3, None if chosen.i_proj is None else 8, None if chosen.o_proj is None else 8))
        dense = Dense(plan, torch.full((plan.workspace.nbytes,), 0xFF, dtype=torch.uint8, device=device))
        out = torch.full((rows, layer.hidden), float("nan"), dtype=dtype, device=device)
        ids = layer.ids.to(device)
        run = lambda: dense.run_into(hidden_states=x, layer_weights=weights, output=out, adapters=chosen,  # noqa: E731
                                     adapter_ids=ids)
        x = layer.x.to(device)
        run()
        near(out, layer.forward(layer.x.double(), function, used), 4, "dense with adapters")
        eager = out.clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            run()
        out.zero_()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
    # The same plan without adapters.
    if dtype is not torch.float32:
        plan = DenseExecutionPlan.prepare(signature, adapters=DenseAdapterLayout(3, 8, 8))
        dense = Dense(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
        out = torch.empty((rows, layer.hidden), dtype=dtype, device=device)
        dense.run_into(hidden_states=layer.x.to(device), layer_weights=weights, output=out)
        near(out, layer.forward(layer.x.double(), function, zero), 4, "dense without adapters")


def test_dense_adapter_refusals(device):
    layer = Layer(device, rows=4, hidden=64, width=48, count=2, rank=4, dtype=torch.bfloat16)
    weights = DenseFfnWeights.from_tensors(layer.w_in.to(device), layer.w_out.to(device))
    signature = DenseSignature(
        payload_dtype=torch.bfloat16, payload_row_capacity=4, hidden_size=64, local_intermediate_size=48,
        activation=Activation(SiluActivation(), GateTransform()),
        i_proj=ProjectionLayout.of(weights.i_proj, order=GateUpOrder.INTERLEAVED), o_proj=ProjectionLayout.of(weights.o_proj),
    )
    plan = DenseExecutionPlan.prepare(signature, adapters=DenseAdapterLayout(2, 4))
    dense = Dense(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
    pool = AdapterWeights(layer.a_in.to(device), layer.b_in.to(device))
    x, out, ids = layer.x.to(device), torch.empty((4, 64), dtype=torch.bfloat16, device=device), layer.ids.to(device)
    for kwargs in (dict(adapters=DenseAdapterWeights(pool)), dict(adapter_ids=ids),
                   dict(adapters=DenseAdapterWeights(None, pool), adapter_ids=ids),
                   dict(adapters=DenseAdapterWeights(pool, pool), adapter_ids=ids)):
        with pytest.raises(ValueError):
            dense.run_into(hidden_states=x, layer_weights=weights, output=out, **kwargs)
    with pytest.raises(ValueError):
        DenseAdapterLayout(2)
    fault = torch.zeros(1, dtype=torch.int32, device=device)
    ids[2] = 5
    dense.run_into(hidden_states=x, layer_weights=weights, output=out, adapters=DenseAdapterWeights(pool), adapter_ids=ids,
                   fault_word=fault)
    assert int(fault) == _native.XP_FAULT_ADAPTER_OUT_OF_RANGE and bool(out[2].isnan().all())
    assert not bool(out[[0, 1, 3]].isnan().any())


def test_dense_plans_that_cannot_keep_their_word(device):
    """A limit applied apart from the adapters would hide an id out of range; fp32 has no activation apart."""

    layer = Layer(device, rows=4, hidden=64, width=48, count=2, rank=4, dtype=torch.bfloat16)
    weights = DenseFfnWeights.from_tensors(layer.w_in.to(device), layer.w_out.to(device))

    def signature(dtype, order, gate):
        return DenseSignature(
            payload_dtype=dtype, payload_row_capacity=4, hidden_size=64, local_intermediate_size=48,
            activation=Activation(SiluActivation(), gate), i_proj=ProjectionLayout.of(weights.i_proj, order=order),
            o_proj=ProjectionLayout.of(weights.o_proj))

    halves = signature(torch.bfloat16, GateUpOrder.CONCATENATED, GateTransform(7.0, 1.0))
    with pytest.raises(ValueError, match="clipped"):
        DenseExecutionPlan.prepare(halves, adapters=DenseAdapterLayout(2, 4))
    DenseExecutionPlan.prepare(halves, adapters=DenseAdapterLayout(2, 4, 4))
    DenseExecutionPlan.prepare(halves, adapters=DenseAdapterLayout(2, None, 4))

    weights = DenseFfnWeights.from_tensors(layer.w_in.float().to(device), layer.w_out.float().to(device))
    plan = DenseExecutionPlan.prepare(signature(torch.float32, GateUpOrder.INTERLEAVED, GateTransform()),
                                      adapters=DenseAdapterLayout(2, 4))
    dense = Dense(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
    x = layer.x.float().to(device)
    with pytest.raises(ValueError, match="every call"):
        dense.run_into(hidden_states=x, layer_weights=weights, output=torch.empty_like(x))
    pool = AdapterWeights(layer.a_in.float().to(device), layer.b_in.float().to(device))
    out = torch.full_like(x, float("nan"))
    dense.run_into(hidden_states=x, layer_weights=weights, output=out, adapters=DenseAdapterWeights(pool),
                   adapter_ids=torch.full((4,), -1, dtype=torch.int32, device=device))
    assert bool(torch.isfinite(out).all())


def _gemm(device, rows, w):
    plan = GemmPlan.prepare(input_layout=TensorLayout((rows, w.shape[1]), w.dtype),
                            weight_layout=ProjectionLayout.of(w_weights := ProjectionWeights(w)),
                            result_layout=TensorLayout((rows, w.shape[0]), w.dtype), activation=None)
    gemm = Gemm(plan, torch.empty(max(plan.workspace.nbytes, 16), dtype=torch.uint8, device=device))
    return lambda x, out: gemm.run_into(x, w_weights, output=out)


def _adapter(device, rows, k, n, layer):
    plan = AdapterPlan.prepare(row_capacity=rows, adapter_count=layer.count, max_rank=layer.rank, input_width=k,
                               output_width=n, dtype=layer.dtype, backward=True)
    return Adapter(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))


@pytest.mark.parametrize("dtype,order,name", [
    (torch.bfloat16, GateUpOrder.INTERLEAVED, "silu"), (torch.float16, GateUpOrder.CONCATENATED, "gelu"),
])
@pytest.mark.parametrize("rows", [40, 333])
def test_a_fine_tuning_step_of_a_layers_adapters(device, rows, dtype, order, name):
    """Forward and backward of adapters on both projections, with the router's balance gradient added
    at the layer's input, captured into a graph and replayed."""

    layer = Layer(device, rows=rows, hidden=256, width=320, count=3, rank=16, dtype=dtype, order=order, seed=rows)
    spec, function = FUNCTIONS[name]
    activation = Activation(spec, GateTransform())
    to = lambda t: t.to(device)  # noqa: E731
    x, ids = to(layer.x), to(layer.ids)
    pool_in = AdapterWeights(to(layer.a_in), to(layer.b_in), to(layer.scales))
    pool_out = AdapterWeights(to(layer.a_out), to(layer.b_out), to(layer.scales))
    w_in, w_out = to(layer.w_in), to(layer.w_out)
    experts, topk, coefficient = 16, 2, 4.0
    g = torch.Generator().manual_seed(9)
    w_router = (torch.randn((experts, layer.hidden), generator=g) * 0.1).to(dtype)
    router_weights = MoeRouterWeights(to(w_router))
    router = Router(row_capacity=rows, hidden_size=layer.hidden, routed_expert_count=experts, routed_topk=topk,
                    payload_dtype=dtype)
    balance = BalanceLoss(row_capacity=rows, routed_expert_count=experts, routed_topk=topk, coefficient=coefficient)
    project_in, project_out = _gemm(device, rows, w_in), _gemm(device, rows, w_out)
    back_in, back_out = _gemm(device, rows, w_in.t().contiguous()), _gemm(device, rows, w_out.t().contiguous())
    back_router = _gemm(device, rows, to(w_router).t().contiguous())
    adapter_in = _adapter(device, rows, layer.hidden, layer.wide, layer)
    adapter_out = _adapter(device, rows, layer.width, layer.hidden, layer)
    empty = lambda *shape: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
    projected, activated, out = empty(rows, layer.wide), empty(rows, layer.width), empty(rows, layer.hidden)
    grad_activated, grad_projected, grad_x = empty(rows, layer.width), empty(rows, layer.wide), empty(rows, layer.hidden)
    grad_logits, grad_router = empty(rows, experts), empty(rows, layer.hidden)
    grads = [torch.empty_like(t) for t in (pool_in.a, pool_in.b, pool_out.a, pool_out.b)]
    upstream = to((torch.randn((rows, layer.hidden), generator=g) * 0.1).to(dtype))

    def step():
        project_in(x, projected)
        adapter_in.run_into(x, pool_in, adapter_ids=ids, base=projected, output=projected)
        activation.apply_into(inputs=projected, output=activated, order=order)
        project_out(activated, out)
        adapter_out.run_into(activated, pool_out, adapter_ids=ids, base=out, output=out)
        router.run_into(hidden_states=x, router_weights=router_weights)
        balance.run_into(logits=router.logits, ids=router.ids)
        back_out(upstream, grad_activated)
        adapter_out.backward_into(activated, upstream, pool_out, adapter_ids=ids, base=grad_activated,
                                  grad_inputs=grad_activated, grad_a=grads[2], grad_b=grads[3])
        activation.backward_into(inputs=projected, grad_output=grad_activated, grad_inputs=grad_projected, order=order)
        back_in(grad_projected, grad_x)
        adapter_in.backward_into(x, grad_projected, pool_in, adapter_ids=ids, base=grad_x, grad_inputs=grad_x,
                                 grad_a=grads[0], grad_b=grads[1])
        balance.backward_into(logits=router.logits, grad_logits=grad_logits)
        back_router(grad_logits, grad_router)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()

    leaves = [t.double().requires_grad_(True) for t in (layer.a_in, layer.b_in, layer.a_out, layer.b_out)]
    inputs = layer.x.double().requires_grad_(True)
    result = layer.forward(inputs, function, leaves)
    expected = torch.autograd.grad(result, [inputs, *leaves], upstream.cpu().double())
    routed = layer.x.double().requires_grad_(True)
    logits = routed @ w_router.double().T
    counts = torch.bincount(router.ids.cpu().flatten().long(), minlength=experts).double()
    loss = coefficient * (counts * experts / (topk * rows) * torch.softmax(logits, dim=1).mean(dim=0)).sum()
    (expected_router,) = torch.autograd.grad(loss, routed)
    loss = float(loss.detach())
    for replay in range(3):
        if replay:
            for t in (out, grad_x, grad_router, *grads):
                t.fill_(float("nan"))
            graph.replay()
        torch.cuda.synchronize()
        near(out, result, 4, "forward")
        for got, want, what in zip((grad_x, *grads), expected, ("x", "a_in", "b_in", "a_out", "b_out")):
            near(got, want, 9, f"gradient of {what}")
        assert torch.equal(balance.counts.cpu().double(), counts)
        assert abs(float(balance.loss) - loss) <= 3 * 2 * STEP[dtype] * loss
        # The logits' rounding moves p by half a step of values up to about 8: eight times the relative step.
        near(grad_router, expected_router, 3 * 8, "gradient through the router")
