"""Performance cases of a layer's training operators: projection gradients, the gated block, orthogonal updates.

Five kinds of pass:

``projection_grad``  the gradients of a projection ``x w^T + b``: of its input rows, its weights and its bias, or
                     through a frozen projection of its input rows alone.
``dense_forward``    a layer's forward pass in training: both projections and the activation, and the projected
                     Gate/Up values that its backward pass reads.
``dense_backward``   the gradients of the same layer: of its input rows, of both weight matrices and of the biases.
``muon``             the orthogonalisation of an update by five Newton-Schulz steps.
``muon_step``        the same within an optimiser's step: momentum, orthogonal update, decay and new weights.

With ``own`` false every pass is computed by elementary torch operations in fp32; with ``own`` true by this
framework's operators.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
RATE, DECAY, MOMENTUM = 0.02, 0.1, 0.95


# ------------------------------------------------------------------ cases
def _projection(name, rows, k, n, dtype="bf16", frozen=False, bias=False, grads="payload"):
    return {"name": name, "kind": "projection_grad", "rows": rows, "k": k, "n": n, "dtype": dtype, "frozen": frozen,
            "bias": bias, "grads": grads}


def _dense(name, kind, rows, hidden, width, dtype="bf16", function="silu", order="interleaved", limit=0.0, bias=False):
    return {"name": name, "kind": kind, "rows": rows, "hidden": hidden, "width": width, "dtype": dtype,
            "function": function, "order": order, "limit": limit, "bias": bias}


def _muon(name, kind, matrices, rows, columns, dtype="bf16", interleaved=False):
    return {"name": name, "kind": kind, "matrices": matrices, "rows": rows, "columns": columns, "dtype": dtype,
            "interleaved": interleaved}


def listed():
    return [
        # A few tokens through the down projection of a 1.7B model: launches and the weight gradient's stores.
        _projection("projection_grad_down_5", 5, 6144, 2048),
        # Adapters fine-tuned through the frozen gate_up of an 8B model: the gradient of its input rows alone.
        _projection("projection_grad_frozen_4096", 4096, 4096, 24576, frozen=True),
        # Odd sizes, fp16, a bias, weight gradients kept in fp32.
        _projection("projection_grad_2053_777_fp16", 777, 1030, 2053, "fp16", bias=True, grads="fp32"),
        # fp32 training of a small model's square projection.
        _projection("projection_grad_1536_700_fp32", 700, 1536, 1536, "fp32"),
        # An 8B model's layer over a batch of 4096 tokens, forward and backward.
        _dense("dense_forward_4096", "dense_forward", 4096, 4096, 12288),
        _dense("dense_backward_4096", "dense_backward", 4096, 4096, 12288),
        # A short batch through a layer of odd width, biases, GELU.
        _dense("dense_forward_1030_33_fp16", "dense_forward", 33, 1030, 2053, "fp16", "gelu", bias=True),
        # A 1.7B model's layer with a clipped gate over CONCATENATED rows and biases.
        _dense("dense_backward_2048_1000_fp16", "dense_backward", 1000, 2048, 6144, "fp16", "gelu", "concatenated", 1.5, True),
        # The down projection of an 8B model.
        _muon("muon_4096_12288", "muon", 1, 4096, 12288),
        # Gate and Up of a 1.7B model, interleaved rows of one tensor, each orthogonalised by itself.
        _muon("muon_step_gate_up_6144", "muon_step", 2, 6144, 2048, interleaved=True),
        # Down projections of a MoE layer's experts.
        _muon("muon_step_experts_32", "muon_step", 32, 2048, 768),
        # A small fp32 matrix: launches.
        _muon("muon_1030_257_fp32", "muon", 1, 1030, 257, "fp32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _cost(case):
    amount = work(case)
    rate = 1.5e14 if case["dtype"] == "fp32" else 2.5e15
    return max(amount["bytes"] / 8e12, amount["flops"] / rate)


def draw(rng):
    kind = rng.choices(("projection_grad", "dense_forward", "dense_backward", "muon", "muon_step"), (28, 14, 24, 18, 16))[0]
    dtype = rng.choices(("bf16", "fp16", "fp32"), (60, 25, 15))[0]
    most = max(_cost(case) for case in listed())
    if kind == "projection_grad":
        k, n = _widths(rng)
        case = _projection("", _log(rng, 1, 8192), k, n, dtype, rng.random() < 0.25, rng.random() < 0.4,
                           rng.choice(("payload", "payload", "fp32")))
        case["bias"] = case["bias"] and not case["frozen"]
    elif kind in ("dense_forward", "dense_backward"):
        hidden, width = _widths(rng)
        case = _dense("", kind, _log(rng, 1, 8192), hidden, width, dtype, rng.choice(("silu", "silu", "gelu", "relu")),
                      rng.choice(("interleaved", "interleaved", "concatenated", "ungated")), 0.0, rng.random() < 0.3)
        if case["order"] == "concatenated" and dtype == "fp32":
            case["order"] = "interleaved"
        if case["order"] != "ungated" and rng.random() < 0.3:
            case["limit"] = 1.5
    else:
        short, long = sorted(_widths(rng))
        if rng.random() < 0.5:
            short, long = long, short
        interleaved = kind == "muon_step" and rng.random() < 0.4
        matrices = 2 if interleaved else rng.choice((1, 1, 2, 3, 8, 24))
        case = _muon("", kind, matrices, short, long, dtype, interleaved)
    del case["name"]
    while _cost(case) > most:
        if "matrices" in case and case["matrices"] > 2:
            case["matrices"] //= 2
        elif rng.random() < 0.5:
            name = "columns" if "columns" in case else "rows"
            case[name] = max(1, case[name] * 3 // 4)
        else:
            name = "rows"
            case[name] = max(1, case[name] * 3 // 4)
    return case


def _widths(rng):
    if rng.random() < 0.6:  # widths of whole 16-byte rows
        return 8 * _log(rng, 24, 1536), 8 * _log(rng, 24, 1536)
    return _log(rng, 129, 9000), _log(rng, 129, 9000)


def _wide(case):
    return case["width"] if case["order"] == "ungated" else 2 * case["width"]


def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "projection_grad":
        rows, k, n = case["rows"], case["k"], case["n"]
        if case["frozen"]:
            return {"bytes": size * (rows * (k + n) + n * k), "flops": 2.0 * rows * k * n}
        kept = 4 if case["grads"] == "fp32" else size
        return {"bytes": size * (rows * (2 * k + n) + n * k) + kept * n * k + (4 * n if case["bias"] else 0),
                "flops": 4.0 * rows * k * n}
    if case["kind"] in ("dense_forward", "dense_backward"):
        rows, hidden, width, wide = case["rows"], case["hidden"], case["width"], _wide(case)
        weights = hidden * (wide + width)
        if case["kind"] == "dense_forward":
            return {"bytes": size * (rows * (2 * hidden + wide) + weights), "flops": 2.0 * rows * weights}
        return {"bytes": size * (rows * (3 * hidden + wide) + 2 * weights), "flops": 4.0 * rows * weights}
    # The two symmetric products of a step count one half.
    short, long = sorted((case["rows"], case["columns"]))
    values = case["matrices"] * short * long
    flops = STEPS * case["matrices"] * (3.0 * short * short * long + float(short) ** 3)
    return {"bytes": values * (2 * size if case["kind"] == "muon" else 3 * size + 8), "flops": flops}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=device).mul_(std).to(dtype)

    def empty(*shape, kind=dtype):
        return torch.empty(shape, dtype=kind, device=device)

    state = {"case": case}
    if case["kind"] == "projection_grad":
        rows, k, n = case["rows"], case["k"], case["n"]
        state["x"], state["grad"] = normal(rows, k), normal(rows, n, std=0.05)
        state["w"] = normal(n, k, std=1 / math.sqrt(k))
        state["bias"] = torch.randn(n, generator=g, device=device) * 0.1 if case["bias"] else None
        state["grad_x"] = empty(rows, k)
        if not case["frozen"]:
            state["grad_w"] = empty(n, k, kind=torch.float32 if case["grads"] == "fp32" else dtype)
            state["grad_bias"] = empty(n, kind=torch.float32) if case["bias"] else None
    elif case["kind"] in ("dense_forward", "dense_backward"):
        rows, hidden, width, wide = case["rows"], case["hidden"], case["width"], _wide(case)
        state["x"] = normal(rows, hidden)
        state["w_in"], state["w_out"] = normal(wide, hidden, std=1 / math.sqrt(hidden)), normal(hidden, width, std=1 / math.sqrt(width))
        state["bias_in"] = state["bias_out"] = None
        if case["bias"]:
            state["bias_in"] = torch.randn(wide, generator=g, device=device) * 0.1
            state["bias_out"] = torch.randn(hidden, generator=g, device=device) * 0.1
        if case["kind"] == "dense_forward":
            state["projected"], state["out"] = empty(rows, wide), empty(rows, hidden)
        else:
            # What the forward pass kept: values of its distribution.
            state["projected"] = normal(rows, wide)
            state["grad"] = normal(rows, hidden, std=0.05)
            state["grad_x"], state["grad_in"], state["grad_out"] = empty(rows, hidden), empty(wide, hidden), empty(hidden, width)
            if case["bias"]:
                state["grad_bias_in"], state["grad_bias_out"] = empty(wide, kind=torch.float32), empty(hidden, kind=torch.float32)
    else:
        count, rows, columns = case["matrices"], case["rows"], case["columns"]
        # A few strong directions over a floor of noise, as gradients have them.
        strong = min(16, rows, columns)
        gradients = torch.randn((count, rows, columns), generator=g, device=device)
        left = torch.randn((count, rows, strong), generator=g, device=device)
        right = torch.randn((count, strong, columns), generator=g, device=device)
        gradients = (gradients.add_(left @ right, alpha=0.3)).mul_(0.01)
        state["gradients"] = _stored(case, gradients.to(dtype))
        if case["kind"] == "muon":
            state["out"] = empty(count, rows, columns)
        else:
            state["momentum"] = _stored(case, torch.randn((count, rows, columns), generator=g, device=device).mul_(0.05))
            state["weights"] = _stored(case, normal(count, rows, columns, std=1 / math.sqrt(columns)))
            state["new_momentum"] = torch.empty_like(state["momentum"])
            state["new_weights"] = torch.empty_like(state["weights"])
    if own:
        _plan(state)
    return state


def _stored(case, matrices):
    """INTERLEAVED Gate and Up: row 2j of one tensor is Gate's row j, row 2j + 1 Up's."""

    return matrices.transpose(0, 1).flatten(0, 1).contiguous() if case["interleaved"] else matrices


def _matrices(case, stored):
    """The matrices of a tensor in the order that it is stored in: a view."""

    return stored.view(case["rows"], 2, case["columns"]).transpose(0, 1) if case["interleaved"] else stored


def _plan(state):
    """What a program of this framework makes once: the operator with its workspace."""

    case = state["case"]
    device = torch.device("cuda", torch.cuda.current_device())
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "projection_grad":
        from crosspool_amd.operators import Gemm, GemmPlan, ProjectionLayout, TensorLayout
        from crosspool_amd.weights import ProjectionWeights

        weights = ProjectionWeights(state["w"], bias=state["bias"])
        plan = GemmPlan.prepare(input_layout=TensorLayout((case["rows"], case["k"]), dtype),
                                weight_layout=ProjectionLayout.of(weights),
                                result_layout=TensorLayout((case["rows"], case["n"]), dtype), activation=None, backward=True)
        state["operator"] = Gemm(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
        state["weights"] = weights
    elif case["kind"] in ("dense_forward", "dense_backward"):
        from crosspool_amd.ffn import GateTransform, GateUpOrder, GeluActivation, ReluActivation, SiluActivation
        from crosspool_amd.operators import Activation, Dense, DenseExecutionPlan, DenseGradients, DenseSignature, ProjectionLayout
        from crosspool_amd.weights import DenseFfnWeights, ProjectionWeights

        function = {"silu": SiluActivation(), "gelu": GeluActivation(), "relu": ReluActivation()}[case["function"]]
        gated = case["order"] != "ungated"
        order = {"interleaved": GateUpOrder.INTERLEAVED, "concatenated": GateUpOrder.CONCATENATED}.get(case["order"])
        weights = DenseFfnWeights(ProjectionWeights(state["w_in"], bias=state["bias_in"]),
                                  ProjectionWeights(state["w_out"], bias=state["bias_out"]))
        signature = DenseSignature(payload_dtype=dtype, payload_row_capacity=case["rows"], hidden_size=case["hidden"],
                                   local_intermediate_size=case["width"],
                                   activation=Activation(function, GateTransform(case["limit"] or None) if gated else None),
                                   i_proj=ProjectionLayout.of(weights.i_proj, order=order),
                                   o_proj=ProjectionLayout.of(weights.o_proj))
        plan = DenseExecutionPlan.prepare(signature, backward=True)
        state["operator"] = Dense(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
        state["weights"] = weights
        if case["kind"] == "dense_backward":
            state["gradients"] = DenseGradients(i_values=state["grad_in"], o_values=state["grad_out"],
                                                i_bias=state.get("grad_bias_in"), o_bias=state.get("grad_bias_out"))
    else:
        from crosspool_amd.muon import Muon, MuonPlan

        plan = MuonPlan.prepare(matrices=case["matrices"], rows=case["rows"], columns=case["columns"], dtype=dtype)
        state["operator"] = Muon(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))


# ------------------------------------------------------------------ passes
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state, kind)
    if kind == "projection_grad":
        return _projection_plain(state)
    if kind == "dense_forward":
        return _dense_forward_plain(state)
    if kind == "dense_backward":
        return _dense_backward_plain(state)
    return _muon_plain(state) if kind == "muon" else _muon_step_plain(state)


def _run_own(state, kind):
    operator = state["operator"]
    if kind == "projection_grad":
        frozen = state["case"]["frozen"]
        operator.backward_into(state["x"], state["grad"], state["weights"], grad_inputs=state["grad_x"],
                               grad_values=None if frozen else state["grad_w"],
                               grad_bias=None if frozen else state["grad_bias"])
        return _named(x=state["grad_x"], w=state.get("grad_w"), bias=state.get("grad_bias"))
    if kind == "dense_forward":
        operator.run_into(hidden_states=state["x"], layer_weights=state["weights"], output=state["out"],
                          projected=state["projected"])
        return {"projected": state["projected"], "out": state["out"]}
    if kind == "dense_backward":
        operator.backward_into(hidden_states=state["x"], layer_weights=state["weights"], projected=state["projected"],
                               grad_output=state["grad"], grad_hidden_states=state["grad_x"], gradients=state["gradients"])
        return _named(x=state["grad_x"], w_in=state["grad_in"], w_out=state["grad_out"],
                      bias_in=state.get("grad_bias_in"), bias_out=state.get("grad_bias_out"))
    case = state["case"]
    if kind == "muon":
        operator.orthogonalize_into(state["gradients"], output=state["out"])
        return state["out"]
    operator.step_into(weights=_matrices(case, state["weights"]), gradients=_matrices(case, state["gradients"]),
                       momentum=_matrices(case, state["momentum"]), new_weights=_matrices(case, state["new_weights"]),
                       new_momentum=_matrices(case, state["new_momentum"]), learning_rate=RATE, weight_decay=DECAY,
                       momentum_factor=MOMENTUM)
    return {"weights": state["new_weights"], "momentum": state["new_momentum"]}


def _named(**found):
    return {name: value for name, value in found.items() if value is not None}


def _projection_plain(state):
    grad, dtype = state["grad"].float(), state["x"].dtype
    found = {"x": (grad @ state["w"].float()).to(dtype)}
    if not state["case"]["frozen"]:
        found["w"] = (grad.T @ state["x"].float()).to(state["grad_w"].dtype)
        if state["bias"] is not None:
            found["bias"] = grad.sum(dim=0)
    return found


def _halves(case, values):
    if case["order"] == "interleaved":
        return values[:, 0::2], values[:, 1::2]
    return (values, None) if case["order"] == "ungated" else (values[:, :case["width"]], values[:, case["width"]:])


def _value_and_slope(function, v):
    if function == "silu":
        share = 1 / (1 + torch.exp(-v))
        return v * share, share * (1 + v * (1 - share))
    if function == "relu":
        return torch.clamp(v, min=0), (v > 0).float()
    share = 0.5 * torch.special.erfc(v * -math.sqrt(0.5))
    return v * share, share + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)


def _dense_forward_plain(state):
    case, dtype = state["case"], state["x"].dtype
    projected = state["x"].float() @ state["w_in"].float().T
    if state["bias_in"] is not None:
        projected = projected + state["bias_in"]
    gate, up = _halves(case, projected)
    limit = case["limit"]
    value, _ = _value_and_slope(case["function"], torch.clamp(gate, max=limit) if limit else gate)
    if up is not None:
        value = value * (torch.clamp(up, -limit, limit) if limit else up)
    out = value @ state["w_out"].float().T
    if state["bias_out"] is not None:
        out = out + state["bias_out"]
    return {"projected": projected.to(dtype), "out": out.to(dtype)}


def _dense_backward_plain(state):
    case, dtype = state["case"], state["x"].dtype
    x, grad, limit = state["x"].float(), state["grad"].float(), case["limit"]
    gate, up = _halves(case, state["projected"].float())
    value, slope = _value_and_slope(case["function"], torch.clamp(gate, max=limit) if limit else gate)
    grad_value = grad @ state["w_out"].float()
    if up is None:
        activated, through = value, grad_value * slope
    else:
        factor = torch.clamp(up, -limit, limit) if limit else up
        activated = value * factor
        grad_gate, grad_up = grad_value * slope * factor, grad_value * value
        if limit:
            grad_gate, grad_up = grad_gate * (gate <= limit), grad_up * (up.abs() <= limit)
        if case["order"] == "interleaved":
            through = torch.stack((grad_gate, grad_up), dim=2).flatten(1)
        else:
            through = torch.cat((grad_gate, grad_up), dim=1)
    found = {"x": (through @ state["w_in"].float()).to(dtype), "w_in": (through.T @ x).to(dtype),
             "w_out": (grad.T @ activated).to(dtype)}
    if case["bias"]:
        found |= {"bias_in": through.sum(dim=0), "bias_out": grad.sum(dim=0)}
    return found


def _newton_schulz(update):
    """Five steps over [matrices, rows, columns] fp32, on the short side's Gram matrices."""

    a, b, c = COEFFICIENTS
    x = update / (update.square().sum(dim=(1, 2), keepdim=True).sqrt() + EPS)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(1, 2).contiguous() if tall else x


def _muon_plain(state):
    return _newton_schulz(state["gradients"].float()).to(state["gradients"].dtype)


def _muon_step_plain(state):
    case = state["case"]
    gradients, weights = _matrices(case, state["gradients"]).float(), _matrices(case, state["weights"])
    momentum = MOMENTUM * _matrices(case, state["momentum"]) + gradients
    update = _newton_schulz(gradients + MOMENTUM * momentum)
    scale = RATE * math.sqrt(max(1.0, case["rows"] / case["columns"]))
    new = weights.float() * (1 - RATE * DECAY) - scale * update
    return {"weights": _stored(case, new.to(weights.dtype)), "momentum": _stored(case, momentum)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"projection_grad": _projection_exact, "dense_forward": _dense_forward_exact,
            "dense_backward": _dense_backward_exact, "muon": _muon_exact, "muon_step": _muon_step_exact}[case["kind"]](state)


def _projection_exact(state):
    grad, x, w = (state[name].double() for name in ("grad", "x", "w"))
    found = {"x": grad @ w}
    if not state["case"]["frozen"]:
        found["w"] = grad.t().contiguous() @ x
        if state["case"]["bias"]:
            found["bias"] = grad.sum(0)
    return found


def _activated(case, projected):
    """The block's activation, for torch's own gradients."""

    limit = case["limit"] or None
    gate, up = _halves(case, projected)
    names = {"silu": torch.nn.functional.silu, "relu": torch.relu, "gelu": torch.nn.functional.gelu}
    out = names[case["function"]](gate.clamp(max=limit) if limit else gate)
    return out if up is None else out * (up.clamp(-limit, limit) if limit else up)


def _dense_forward_exact(state):
    projected = state["x"].double() @ state["w_in"].double().t().contiguous()
    if state["bias_in"] is not None:
        projected += state["bias_in"].double()
    out = _activated(state["case"], projected) @ state["w_out"].double().t().contiguous()
    return {"projected": projected, "out": out if state["bias_out"] is None else out + state["bias_out"].double()}


def _dense_backward_exact(state):
    projected = state["projected"].double().requires_grad_(True)
    grad = state["grad"].double()
    activated = _activated(state["case"], projected)
    (through,) = torch.autograd.grad(activated, projected, grad @ state["w_out"].double())
    found = {"x": through @ state["w_in"].double(), "w_in": through.t().contiguous() @ state["x"].double(),
             "w_out": grad.t().contiguous() @ activated.detach()}
    if state["case"]["bias"]:
        found |= {"bias_in": through.sum(0), "bias_out": grad.sum(0)}
    return found


def _orthogonal_exact(matrix):
    """One matrix [rows, columns]: every step applied to the matrix as it stands."""

    a, b, c = COEFFICIENTS
    x = matrix / (torch.linalg.vector_norm(matrix) + EPS)
    for _ in range(STEPS):
        if x.shape[0] <= x.shape[1]:
            gram = torch.mm(x, x.t().contiguous())
            x = torch.addmm(x, torch.addmm(gram, gram, gram, beta=b, alpha=c), x, beta=a)
        else:
            gram = torch.mm(x.t().contiguous(), x)
            x = torch.addmm(x, x, torch.addmm(gram, gram, gram, beta=b, alpha=c), beta=a)
    return x


def _muon_exact(state):
    return torch.stack([_orthogonal_exact(matrix.double()) for matrix in state["gradients"]])


def _muon_step_exact(state):
    case = state["case"]
    gradients, momentum, weights = (_matrices(case, state[name]).double() for name in ("gradients", "momentum", "weights"))
    momentum = momentum * MOMENTUM + gradients
    updates = torch.stack([_orthogonal_exact(matrix) for matrix in gradients + momentum * MOMENTUM])
    step = RATE * max(1.0, case["rows"] / case["columns"]) ** 0.5
    return {"weights": _stored(case, weights - RATE * DECAY * weights - step * updates), "momentum": _stored(case, momentum)}
