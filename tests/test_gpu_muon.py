"""Orthogonal updates on the GPU, against the formula in 64 bits.

Tolerances, derived before the first run.  Every rounding to fp16 is off by half a step, 2^-12, of a value, and errors of
many values are independent, so a stored matrix is off by less than 2^-12 of its 2-norm.  A step stores three: X, A and
b A + c A A.  X's relative error goes on as it is (|f(x)| >= 0.7 |x| and |f'| <= a over (0, 1.2]: growth by at most a / 0.7 in
the worst direction, near 1 over the spectrum, whose values all grow alike while they are small); A's reaches X'
times |b + 2 c x^2| x^2 <= 4.8 against f(x) / x >= 0.7, b A + c A A's times 4.8 as well.  Five steps of (1 + 4.8 + 4.8)
2^-12 / 0.7 would be 2^-6 if all added up; independent errors add as squares: sqrt(5) * sqrt(1 + 2 * 4.8^2) * 2^-12 / 0.7 =
2^-7.6.  The checks allow 2^-7.6 plus the result's own half step for 16-bit payloads.  fp32: the same with 2^-24 and sums
of n terms, whose errors grow like sqrt(n): 2^-7.6+12-24 = 2^-19.6 sqrt(n).

That is relative to values in fp16's normal range.  An update far below eps has an X0 far below 1, and what is stored of
it times 2^12 is off by half a subnormal step, 2^-25 2^-12 = 2^-37 of a value of X; five steps let it grow by at most a^5 =
485 < 2^9: 2^-28 sqrt(values) in the 2-norm is allowed besides (fp32: 2^-149, nothing).
"""

from __future__ import annotations

import math

import pytest
import torch

from crosspool_amd.muon import Muon, MuonPlan, gate_up_matrices

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
A, B, C = 3.4445, -4.7750, 2.0315


def orthogonal(updates, steps=5, eps=1e-7):
    """In 64 bits, every matrix as it lies."""

    found = []
    for x in updates.double():
        x = x / (x.norm() + eps)
        for _ in range(steps):
            if x.shape[0] <= x.shape[1]:
                gram = x @ x.T.contiguous()
                x = A * x + (B * gram + C * gram @ gram) @ x
            else:
                gram = x.T.contiguous() @ x
                x = A * x + x @ (B * gram + C * gram @ gram)
        found.append(x)
    return torch.stack(found)


def tolerance(dtype, longest):
    if dtype is FP32:
        return 2.0**-19.6 * math.sqrt(longest)
    return 2.0**-7.6 + torch.finfo(dtype).eps / 2


def updates(device, count, rows, columns, dtype, seed=0, std=0.01):
    g = torch.Generator(device=device).manual_seed(seed + rows + 3 * columns)
    rank = min(4, rows, columns)
    strong = torch.randn((count, rows, rank), generator=g, device=device) @ torch.randn((count, rank, columns), generator=g, device=device)
    return ((torch.randn((count, rows, columns), generator=g, device=device) + 0.5 * strong) * std).to(dtype)


def muon(device, count, rows, columns, dtype):
    plan = MuonPlan.prepare(matrices=count, rows=rows, columns=columns, dtype=dtype)
    return Muon(plan, torch.full((plan.workspace.nbytes,), 0xFF, dtype=torch.uint8, device=device))


def near(actual, expected, allowed, what):
    for i, (found, wanted) in enumerate(zip(actual.double(), expected)):
        error, size = float((found - wanted).norm()), float(wanted.norm())
        besides = 0.0 if actual.dtype is FP32 else 2.0**-28 * wanted.numel() ** 0.5
        assert error <= allowed * size + besides, f"{what} {i}: error {error:.2e} of {size:.2e} above {allowed:.2e}"


SIZES = [(1, 1, 1), (2, 1, 7), (1, 9, 1), (3, 5, 8), (1, 64, 64), (2, 65, 200), (1, 200, 65), (4, 128, 264), (1, 257, 1030),
         (1, 1030, 257), (2, 512, 512), (3, 768, 384), (1, 640, 2056)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("count,rows,columns", SIZES)
def test_orthogonalize(device, count, rows, columns, dtype):
    source = updates(device, count, rows, columns, dtype)
    operator = muon(device, count, rows, columns, dtype)
    out = torch.full_like(source, float("nan"))
    operator.orthogonalize_into(source, output=out)
    near(out, orthogonal(source), tolerance(dtype, max(rows, columns)), "matrix")
    again = torch.empty_like(out)
    operator.orthogonalize_into(source, output=again)
    assert torch.equal(out, again)
    operator.orthogonalize_into(source, output=source)  # in place
    assert torch.equal(out, source)


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_number_of_steps(device, steps):
    for rows, columns in ((72, 136), (136, 72)):
        source = updates(device, 2, rows, columns, BF16)
        out = torch.empty_like(source)
        muon(device, 2, rows, columns, BF16).orthogonalize_into(source, output=out, steps=steps)
        # every step more adds its three roundings (see above): sqrt(8 / 5) at most
        near(out, orthogonal(source, steps), 2.0**-7.2 + 2.0**-9, f"{steps} steps")


def test_scales_of_updates(device):
    """The result does not depend on the update's scale, down to eps and up to the dtype's largest."""

    for dtype, scales in ((BF16, (1e-30, 1e-6, 1.0, 1e30)), (FP32, (1e-20, 1.0, 1e30)), (FP16, (2.0**-10, 1.0, 2.0**12))):
        base = updates(device, 1, 96, 200, FP32, std=1.0)
        for scale in scales:
            source = (base * scale).to(dtype)
            out = torch.empty_like(source)
            muon(device, 1, 96, 200, dtype).orthogonalize_into(source, output=out)
            near(out, orthogonal(source), tolerance(dtype, 200), f"{dtype} {scale}")


def test_zero_and_bad_matrices(device):
    source = updates(device, 4, 80, 130, BF16)
    source[1] = 0
    source[2, 3, 4] = float("inf")
    source[3, 79, 129] = float("nan")
    out = torch.full_like(source, 9.0)
    muon(device, 4, 80, 130, BF16).orthogonalize_into(source, output=out)
    assert bool((out[1] == 0).all()) and bool(out[2].isnan().all()) and bool(out[3].isnan().all())
    near(out[:1], orthogonal(source[:1]), tolerance(BF16, 130), "the good matrix")


@pytest.mark.parametrize("rows,columns", [(48, 64), (61, 37)])
def test_strided_matrices(device, rows, columns):
    for dtype in (BF16, FP32):
        dense = updates(device, 3, rows, columns, dtype)
        wide = torch.full((3, rows + 2, columns + 5), 4.0, dtype=dtype, device=device)
        view = wide[:, 1:rows + 1, 2:columns + 2]
        view.copy_(dense)
        target = torch.full((rows, 3, columns + 3), 5.0, dtype=dtype, device=device)
        out = target.transpose(0, 1)[:, :, :columns]
        muon(device, 3, rows, columns, dtype).orthogonalize_into(view, output=out)
        near(out, orthogonal(dense), tolerance(dtype, max(rows, columns)), "strided")
        assert bool((target[:, :, columns:] == 5.0).all())


def reference_step(weights, gradients, momentum, rate, decay, factor, nesterov, scale):
    momentum = factor * momentum.double() + gradients.double()
    update = orthogonal(gradients.double() + factor * momentum if nesterov else momentum)
    return (1 - rate * decay) * weights.double() - rate * scale * update, momentum, update


@pytest.mark.parametrize("dtype,kept", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP32, FP32)])
@pytest.mark.parametrize("rows,columns,nesterov", [(64, 200, True), (200, 64, False), (45, 131, True)])
def test_optimiser_step(device, rows, columns, nesterov, dtype, kept):
    g = torch.Generator(device=device).manual_seed(rows)
    gradients = updates(device, 2, rows, columns, dtype)
    momentum = torch.randn((2, rows, columns), generator=g, device=device) * 0.05
    weights = (torch.randn((2, rows, columns), generator=g, device=device) * 0.1).to(kept)
    rate, decay, factor = 0.5, 0.1, 0.9
    scale = max(1.0, rows / columns) ** 0.5
    wanted, new, update = reference_step(weights, gradients, momentum, rate, decay, factor, nesterov, scale)
    operator = muon(device, 2, rows, columns, dtype)
    arguments = dict(weights=weights, gradients=gradients, momentum=momentum, learning_rate=rate, weight_decay=decay,
                     momentum_factor=factor, nesterov=nesterov)
    new_weights, new_momentum = torch.full_like(weights, float("nan")), torch.full_like(momentum, float("nan"))
    before = weights.clone(), momentum.clone()
    operator.step_into(**arguments, new_weights=new_weights, new_momentum=new_momentum)
    assert torch.equal(weights, before[0]) and torch.equal(momentum, before[1])
    # two fp32 roundings of the momentum's terms
    assert bool(((new_momentum.double() - new).abs() <= 2.0**-23 * (factor * momentum.double().abs() + gradients.double().abs())).all())
    for found, target, moved, held in zip(new_weights.double(), wanted, update, weights.double()):
        # the update's own error, in its 2-norm, and the weights' rounding
        allowed = rate * scale * (2.0**-7.6 if dtype is not FP32 else tolerance(FP32, 200)) * float(moved.norm())
        allowed += (torch.finfo(kept).eps / 2 + 2.0**-22) * float(target.norm() + held.norm())
        assert float((found - target).norm()) <= allowed
    operator.step_into(**arguments)
    assert torch.equal(weights, new_weights) and torch.equal(momentum, new_momentum)


def test_gate_and_up_apart(device):
    """An INTERLEAVED i_proj in one tensor gives what Gate and Up give in tensors of their own."""

    rows, columns = 72, 136
    g = torch.Generator(device=device).manual_seed(1)
    gradients, weights = (torch.randn((2 * rows, columns), generator=g, device=device).to(BF16) for _ in range(2))
    momentum = torch.randn((2 * rows, columns), generator=g, device=device)
    apart = [gate_up_matrices(t).contiguous() for t in (weights, gradients, momentum)]
    operator = muon(device, 2, rows, columns, BF16)
    operator.step_into(weights=apart[0], gradients=apart[1], momentum=apart[2], learning_rate=0.1)
    operator.step_into(weights=gate_up_matrices(weights), gradients=gate_up_matrices(gradients), momentum=gate_up_matrices(momentum),
                       learning_rate=0.1)
    assert torch.equal(gate_up_matrices(weights), apart[0]) and torch.equal(gate_up_matrices(momentum), apart[2])


def test_step_in_a_graph(device):
    rows, columns = 136, 200
    operator = muon(device, 2, rows, columns, BF16)
    gradients = updates(device, 2, rows, columns, BF16)
    weights = torch.randn((2, rows, columns), device=device).to(BF16)
    momentum = torch.zeros((2, rows, columns), device=device)
    run = lambda: operator.step_into(weights=weights, gradients=gradients, momentum=momentum, learning_rate=0.1)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in (1, 2, 3):
        gradients.copy_(updates(device, 2, rows, columns, BF16, seed=seed))
        held = weights.clone(), momentum.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed = weights.clone(), momentum.clone()
        weights.copy_(held[0])
        momentum.copy_(held[1])
        run()
        assert torch.equal(weights, replayed[0]) and torch.equal(momentum, replayed[1])


def test_training_a_layer(device):
    """Forward, backward and an orthogonal update of both matrices, several steps in place: every step is that of the
    formulas in 64 bits on the values that it starts from, and the loss's gradient is what torch has."""

    from crosspool_amd.ffn import GateTransform, GateUpOrder, SiluActivation
    from crosspool_amd.operators import Activation, Dense, DenseExecutionPlan, DenseGradients, DenseSignature, ProjectionLayout
    from crosspool_amd.weights import DenseFfnWeights, ProjectionWeights

    rows, hidden, width = 96, 128, 192
    g = torch.Generator(device=device).manual_seed(7)
    normal = lambda *shape, std: (torch.randn(shape, generator=g, device=device) * std).to(BF16)  # noqa: E731
    weights = DenseFfnWeights(ProjectionWeights(normal(2 * width, hidden, std=hidden**-0.5)),
                              ProjectionWeights(normal(hidden, width, std=width**-0.5)))
    signature = DenseSignature(
        payload_dtype=BF16, payload_row_capacity=rows, hidden_size=hidden, local_intermediate_size=width,
        activation=Activation(SiluActivation(), GateTransform()),
        i_proj=ProjectionLayout.of(weights.i_proj, order=GateUpOrder.INTERLEAVED), o_proj=ProjectionLayout.of(weights.o_proj))
    plan = DenseExecutionPlan.prepare(signature, backward=True)
    dense = Dense(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
    into = DenseGradients(torch.empty_like(weights.i_proj.values), torch.empty_like(weights.o_proj.values))
    updates_of = (muon(device, 2, width, hidden, BF16), muon(device, 1, hidden, width, BF16))
    momenta = [torch.zeros_like(t, dtype=FP32) for t in (weights.i_proj.values, weights.o_proj.values)]
    projected, out = normal(rows, 2 * width, std=1.0), normal(rows, hidden, std=1.0)
    for _ in range(3):
        x, target = normal(rows, hidden, std=1.0), normal(rows, hidden, std=1.0)
        dense.run_into(hidden_states=x, layer_weights=weights, output=out, projected=projected)
        grad = ((out.float() - target.float()) / rows).to(BF16)
        dense.backward_into(hidden_states=x, layer_weights=weights, projected=projected, grad_output=grad, gradients=into)
        leaves = [t.double().requires_grad_(True) for t in (weights.i_proj.values, weights.o_proj.values)]
        p = x.double() @ leaves[0].T
        y = (torch.nn.functional.silu(p[:, 0::2]) * p[:, 1::2]) @ leaves[1].T
        exact = torch.autograd.grad(y, leaves, grad.double())
        for found, wanted in zip((into.i_values, into.o_values), exact):
            # rounded on the way: the projection, its gradient (or the activated values), the result
            assert float((found.double() - wanted).norm() / wanted.norm()) <= 3 * 3 * 2.0**-9
        held = [(t.clone(), m.clone()) for t, m in zip((weights.i_proj.values, weights.o_proj.values), momenta)]
        updates_of[0].step_into(weights=gate_up_matrices(weights.i_proj.values), gradients=gate_up_matrices(into.i_values),
                                momentum=gate_up_matrices(momenta[0]), learning_rate=0.05)
        updates_of[1].step_into(weights=weights.o_proj.values, gradients=into.o_values, momentum=momenta[1], learning_rate=0.05)
        for index, split in ((0, gate_up_matrices), (1, lambda t: t.unsqueeze(0))):
            now = (weights.i_proj.values, weights.o_proj.values)[index]
            gradient = (into.i_values, into.o_values)[index]
            shape = split(now).shape
            wanted, new, update = reference_step(split(held[index][0]), split(gradient), split(held[index][1]), 0.05, 0.0, 0.95, True,
                                                 max(1.0, shape[1] / shape[2]) ** 0.5)
            scale = 0.05 * max(1.0, shape[1] / shape[2]) ** 0.5
            allowed = scale * 2.0**-7.6 * float(update.norm()) + (2.0**-9 + 2.0**-22) * 2 * float(wanted.norm())
            assert float((split(now).double() - wanted).norm()) <= allowed


def test_refusals(device):
    operator = muon(device, 2, 48, 64, BF16)
    good = torch.zeros((2, 48, 64), dtype=BF16, device=device)
    out = torch.empty_like(good)
    for bad in (good[:1], good.float(), good[:, :, ::2], good.transpose(1, 2), good.cpu()):
        with pytest.raises(ValueError):
            operator.orthogonalize_into(bad, output=out)
    with pytest.raises(RuntimeError, match="steps"):
        operator.orthogonalize_into(good, output=out, steps=0)
    with pytest.raises(RuntimeError, match="whole"):
        flat = torch.zeros(2 * 48 * 64 + 64, dtype=BF16, device=device)
        operator.orthogonalize_into(flat[:-64].view(2, 48, 64), output=flat[64:].view(2, 48, 64))
    with pytest.raises(RuntimeError, match="separate"):
        operator.orthogonalize_into(good, output=out[:1].expand(2, 48, 64))
    momentum = torch.zeros((2, 48, 64), device=device)
    with pytest.raises(ValueError, match="momentum"):
        operator.step_into(weights=good, gradients=out, momentum=good, learning_rate=0.1)
    with pytest.raises(ValueError, match="new weights"):
        operator.step_into(weights=good, gradients=out, momentum=momentum, new_weights=good.float(), learning_rate=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        operator.step_into(weights=good, gradients=good, momentum=momentum, learning_rate=0.1)
    with pytest.raises(ValueError, match="GPU|device"):
        Muon(operator.plan, torch.empty(operator.plan.workspace.nbytes, dtype=torch.uint8))


# Gram matrices and products of 256 x 256 and 128 x 128 tiles and of split ones, mirrored, in batches, wide and tall.
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("count,rows,columns", [(1, 1536, 6144), (1, 6144, 1536), (1, 2300, 2300), (2, 1031, 4103), (1, 2048, 5120),
                                                (1, 4096, 12288), (3, 2561, 1025)])
def test_large_orthogonalize(device, count, rows, columns, dtype):
    if dtype is FP32 and columns > 12000:
        pytest.skip("the 16-bit tiles' size")
    source = updates(device, count, rows, columns, dtype)
    operator = muon(device, count, rows, columns, dtype)
    out = torch.full_like(source, float("nan"))
    operator.orthogonalize_into(source, output=out)
    near(out, orthogonal(source), tolerance(dtype, max(rows, columns)), "matrix")
    operator.scratch.fill_(0xFF)
    again = torch.empty_like(out)
    operator.orthogonalize_into(source, output=again)
    assert torch.equal(out, again)


def test_large_step_in_place(device):
    """Weights and momentum of a batch, in place and apart: the same bits, and the formula's."""

    g = torch.Generator(device=device).manual_seed(11)
    gradients = updates(device, 2, 2304, 2048, BF16, seed=4)
    weights = (torch.randn(gradients.shape, generator=g, device=device) * 0.02).to(BF16)
    momentum = torch.randn(gradients.shape, generator=g, device=device) * 0.01
    operator = muon(device, 2, 2304, 2048, BF16)
    new_weights, new_momentum = torch.full_like(weights, float("nan")), torch.full_like(momentum, float("nan"))
    options = dict(learning_rate=0.02, weight_decay=0.1, momentum_factor=0.9)
    operator.step_into(weights=weights, gradients=gradients, momentum=momentum, new_weights=new_weights, new_momentum=new_momentum,
                       **options)
    kept = 0.9 * momentum.double() + gradients.double()
    exact = orthogonal(gradients.double() + 0.9 * kept)
    step = 0.02 * math.sqrt(2304 / 2048)
    expected = (1 - 0.002) * weights.double() - step * exact
    # the factor, the product and the sum are off by half a step each, 2^-24 of terms no larger than the two magnitudes' sum
    size = float((0.9 * momentum.double().abs() + gradients.double().abs()).max())
    assert float((new_momentum.double() - kept).abs().max()) <= 3 * 2.0**-24 * size
    # the update's error (its half step is not taken: it is added in fp32), and half a step of the new weights
    for found, wanted, update in zip(new_weights.double(), expected, exact):
        allowed = 2.0**-7.6 * step * float(update.norm()) + 2.0**-9 * float(wanted.norm()) * 2
        assert float((found - wanted).norm()) <= allowed
    operator.step_into(weights=weights, gradients=gradients, momentum=momentum, **options)
    assert torch.equal(weights, new_weights) and torch.equal(momentum, new_momentum)


@pytest.mark.parametrize("count,rows,columns", [(4096, 5, 9), (1000, 33, 8), (2, 3, 1 << 20), (1, 1 << 20, 2)])
def test_many_and_long_matrices(device, count, rows, columns):
    source = updates(device, count, rows, columns, BF16)
    out = torch.full_like(source, float("nan"))
    muon(device, count, rows, columns, BF16).orthogonalize_into(source, output=out)
    exact = source.double()
    exact = exact / (exact.flatten(1).norm(dim=1)[:, None, None] + 1e-7)
    for _ in range(5):
        if rows <= columns:
            gram = torch.matmul(exact, exact.transpose(1, 2).contiguous())
            exact = A * exact + torch.matmul(B * gram + C * torch.matmul(gram, gram), exact)
        else:
            gram = torch.matmul(exact.transpose(1, 2).contiguous(), exact)
            exact = A * exact + torch.matmul(exact, B * gram + C * torch.matmul(gram, gram))
    near(out, exact, tolerance(BF16, max(rows, columns)), "matrix")
