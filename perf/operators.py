"""Performance cases of the adapter, activation-gradient and expert-balance operators.

Five kinds of pass:

``adapt``       low-rank adapters of many requests beside a shared projection: every token row carries the
                index of its request's adapter (-1: none) and gets ``base + scale (x A^T) B^T``; with an
                activation the sum goes through it (gate_up of a gated layer).
``adapt_grad``  the gradients of the same for fine-tuning: of the input rows (added to the projection's own),
                of every adapter's A and of its B.
``act_grad``    the gradient of a layer's activation, gated or not, between the two projections.
``balance``     per-expert counts of the routes and the balance loss of a Router's logits.
``balance_step``  the same with the gradient of the logits, as a training step takes it.

With ``own`` false every pass is computed by elementary torch operations in fp32; with ``own`` true by this
framework's operators.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases
def _adapt(name, rows, k, n, adapters, rank, requests, dtype="bf16", activation="none", shuffled=False, kind="adapt"):
    return {"name": name, "kind": kind, "rows": rows, "k": k, "n": n, "adapters": adapters, "rank": rank,
            "requests": requests, "dtype": dtype, "activation": activation, "shuffled": shuffled}


def _act(name, rows, width, function, order, dtype="bf16", limit=0.0, offset=0.0):
    return {"name": name, "kind": "act_grad", "rows": rows, "width": width, "function": function, "order": order,
            "dtype": dtype, "limit": limit, "offset": offset}


def _balance(name, kind, rows, experts, topk, dtype, scores, padded):
    return {"name": name, "kind": kind, "rows": rows, "experts": experts, "topk": topk, "dtype": dtype,
            "scores": scores, "padded": padded}


def listed():
    return [
        # One request decoding through the down projection of an 8B model: latency and launches.
        _adapt("adapt_down_1", 1, 12288, 4096, 16, 16, 1),
        # A decode batch of an 8B model's gate_up, nearly every request with an adapter of its own.
        _adapt("adapt_gate_up_48", 48, 4096, 24576, 32, 32, 48, activation="silu"),
        # Chunked prefill beside decode: few hundred rows in scattered order, fp16, odd sizes.
        _adapt("adapt_2053_333_fp16", 333, 1030, 2053, 12, 24, 40, "fp16", shuffled=True),
        # Prefill of the gate_up of an 8B model with a handful of long requests.
        _adapt("adapt_gate_up_2048", 2048, 4096, 24576, 8, 32, 6, activation="silu"),
        # The largest prefill: down projection of an 8B model, ranks up to 64.
        _adapt("adapt_down_8192", 8192, 12288, 4096, 8, 64, 20),
        # fp32 adapters of a small model's square projection.
        _adapt("adapt_1536_700_fp32", 700, 1536, 1536, 4, 8, 9, "fp32"),
        # Fine-tuning one adapter on the gate_up of an 8B model.
        _adapt("adapt_grad_gate_up_4096", 4096, 4096, 24576, 1, 16, 1, kind="adapt_grad"),
        # Fine-tuning several adapters in one batch: fp16, odd sizes.
        _adapt("adapt_grad_2053_777_fp16", 777, 1030, 2053, 5, 24, 13, "fp16", shuffled=True, kind="adapt_grad"),
        # The SiLU gate of an 8B model's layer in a training step.
        _act("act_grad_4096_12288", 4096, 12288, "silu", "interleaved"),
        # A clipped GELU gate over CONCATENATED rows of odd width.
        _act("act_grad_333_2053_fp16", 333, 2053, "gelu", "concatenated", "fp16", limit=2.0, offset=1.0),
        # Expert load of a decode step.
        _balance("balance_128_64", "balance", 64, 128, 8, "bf16", "softmax", True),
        # The balance loss of a training step over a long batch.
        _balance("balance_step_128_65536", "balance_step", 65536, 128, 8, "fp32", "softmax", False),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _cost(case):
    amount = work(case)
    return max(amount["bytes"] / 8e12, amount["flops"] / 2.5e15)


def draw(rng):
    kind = rng.choices(("adapt", "adapt_grad", "act_grad", "balance", "balance_step"), (45, 20, 12, 8, 15))[0]
    dtype = rng.choices(("bf16", "fp16", "fp32"), (60, 25, 15))[0]
    most = max(_cost(case) for case in listed())
    if kind in ("adapt", "adapt_grad"):
        rows = _log(rng, 1, 8192)
        if rng.random() < 0.6:  # widths of whole 16-byte rows
            k, n = 8 * _log(rng, 32, 1536), 16 * _log(rng, 16, 1536)
        else:
            k, n = _log(rng, 257, 9000), _log(rng, 257, 9000)
        activation = rng.choice(("none", "none", "silu", "gelu")) if kind == "adapt" else "none"
        n += n % 2 if activation != "none" else 0
        requests = rows if rows <= 32 or rng.random() < 0.2 else _log(rng, 1, min(rows, 64))
        case = _adapt("", rows, k, n, _log(rng, 1, 48), rng.choice((4, 8, 12, 16, 24, 32, 33, 64, 100, 128)), requests,
                      dtype, activation, rng.random() < 0.3, kind)
    elif kind == "act_grad":
        case = _act("", _log(rng, 1, 8192), _log(rng, 100, 14336), rng.choice(("silu", "gelu", "gelu_tanh", "relu")),
                    rng.choice(("interleaved", "concatenated", "ungated")), rng.choice(("bf16", "fp16")))
        if case["order"] != "ungated" and rng.random() < 0.3:
            case["limit"], case["offset"] = 1.5, rng.choice((0.0, 1.0))
    else:
        experts = rng.choice((8, 16, 60, 64, 128, 160, 256, 384, 512, 1000))
        if kind == "balance_step" and dtype == "fp16":
            dtype = "bf16"  # a mean's gradients over thousands of rows are below fp16's normal numbers
        case = _balance("", kind, _log(rng, 1, 65536), experts, rng.choice((1, 2, 4, 6, 8)), dtype,
                        rng.choice(("softmax", "sigmoid")), rng.random() < 0.5)
    del case["name"]
    while _cost(case) > most:
        case["rows"] = case["rows"] * 3 // 4
        if "requests" in case:
            case["requests"] = min(case["requests"], case["rows"])
    return case


def _ranks(case):
    """Ranks of the pool's adapters, the largest first: real pools mix them."""

    rank = case["rank"]
    cycle = (rank, max(1, rank // 2), rank, max(1, rank // 4))
    return [cycle[i % 4] for i in range(case["adapters"])]


def _request_adapters(case):
    """Adapter of every request: one of eight requests has none, the others go round the pool."""

    if case["requests"] == 1:
        return [0]
    return [-1 if q % 8 == 5 else (q - (q + 2) // 8) % case["adapters"] for q in range(case["requests"])]


def work(case):
    rows, size = case["rows"], BYTES[case["dtype"]]
    if case["kind"] in ("adapt", "adapt_grad"):
        k, n, ranks = case["k"], case["n"], _ranks(case)
        chosen = _request_adapters(case)
        weights = sum(ranks[a] for a in set(chosen) if a >= 0) * (k + n)
        mean_rank = sum(ranks[a] for a in chosen if a >= 0) / len(chosen)
        if case["kind"] == "adapt":
            out = n if case["activation"] == "none" else n // 2
            return {"bytes": size * (rows * (k + n + out) + weights) + 4 * rows, "flops": 2.0 * rows * mean_rank * (k + n)}
        grads = case["adapters"] * case["rank"] * (k + n)
        return {"bytes": size * (rows * (3 * k + n) + weights + grads) + 4 * rows,
                "flops": 2.0 * rows * mean_rank * (3 * k + 2 * n)}
    if case["kind"] == "act_grad":
        wide = 1 if case["order"] == "ungated" else 2
        return {"bytes": size * rows * case["width"] * (2 * wide + 1), "flops": 20.0 * rows * case["width"]}
    live = _live(case)
    read = live * (case["experts"] * size + case["topk"] * 4)
    step = case["kind"] == "balance_step"
    return {"bytes": read + (rows * case["experts"] * size if step else 0) + case["experts"] * 4,
            "flops": (12.0 if step else 6.0) * live * case["experts"]}


def _live(case):
    return case["rows"] - case["rows"] // 7 if case["padded"] else case["rows"]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=device) * std).to(dtype)

    rows = case["rows"]
    state = {"case": case}
    if case["kind"] in ("adapt", "adapt_grad"):
        k, n, count, rank = case["k"], case["n"], case["adapters"], case["rank"]
        ranks = _ranks(case)
        state["ranks"] = torch.tensor(ranks, dtype=torch.int32, device=device)
        state["scales"] = torch.rand(count, generator=g, device=device) + 0.5
        state["a"] = normal(count, rank, k, std=1 / math.sqrt(k))
        state["b"] = normal(count, n, rank, std=1 / math.sqrt(rank))
        state["ids"] = _ids(case, g, device)
        state["x"] = normal(rows, k)
        out = n if case["activation"] == "none" else n // 2
        if case["kind"] == "adapt":
            state["base"] = normal(rows, n)
            state["out"] = torch.empty((rows, out), dtype=dtype, device=device)
        else:
            state["grad"] = normal(rows, n, std=0.05)
            state["base"] = normal(rows, k, std=0.5)
            state["out"] = torch.empty((rows, k), dtype=dtype, device=device)
            state["grad_a"] = torch.empty((count, rank, k), dtype=dtype, device=device)
            state["grad_b"] = torch.empty((count, n, rank), dtype=dtype, device=device)
    elif case["kind"] == "act_grad":
        wide = case["width"] * (1 if case["order"] == "ungated" else 2)
        state["inputs"] = normal(rows, wide)
        state["grad"] = normal(rows, case["width"], std=0.1)
        state["out"] = torch.empty((rows, wide), dtype=dtype, device=device)
    else:
        experts, topk = case["experts"], case["topk"]
        # Some experts are favoured, as those of a router that is not balanced yet.
        favour = torch.randn(experts, generator=g, device=device)
        state["logits"] = (torch.randn((rows, experts), generator=g, device=device) * 1.5 + favour).to(dtype)
        state["ids"] = torch.topk(state["logits"].float(), topk, dim=1).indices.to(torch.int32)
        live = _live(case)
        state["ids"][live:] = -1
        state["live"] = torch.tensor([live], dtype=torch.int32, device=device)
        state["grad_loss"] = torch.rand(1, generator=g, device=device) + 0.5
        if case["kind"] == "balance_step":
            state["out"] = torch.empty_like(state["logits"])
    if own:
        _plan(state)
    return state


def _ids(case, g, device):
    """Adapter of every token row: requests of random lengths one after another, or rows in any order."""

    rows, requests = case["rows"], case["requests"]
    adapters = torch.tensor(_request_adapters(case), dtype=torch.int32, device=device)
    cuts = torch.randperm(rows - 1, generator=g, device=device)[: requests - 1] + 1
    starts = torch.zeros(rows, dtype=torch.int64, device=device)
    starts[cuts] = 1
    ids = adapters[starts.cumsum(0)]
    return ids[torch.randperm(rows, generator=g, device=device)] if case["shuffled"] else ids


def _plan(state):
    """What a program of this framework makes once: the operator with its workspace."""

    case = state["case"]
    device = torch.device("cuda", torch.cuda.current_device())
    if case["kind"] in ("adapt", "adapt_grad"):
        from crosspool_amd.adapters import Adapter, AdapterPlan, AdapterWeights

        plan = AdapterPlan.prepare(row_capacity=case["rows"], adapter_count=case["adapters"], max_rank=case["rank"],
                                   input_width=case["k"], output_width=case["n"], dtype=DTYPES[case["dtype"]],
                                   backward=case["kind"] == "adapt_grad")
        state["operator"] = Adapter(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
        state["weights"] = AdapterWeights(state["a"], state["b"], state["scales"], state["ranks"])
        state["activation"] = _activation(case["activation"], 0.0, 0.0, True) if case["activation"] != "none" else None
    elif case["kind"] == "act_grad":
        from crosspool_amd.ffn import GateUpOrder

        gated = case["order"] != "ungated"
        state["activation"] = _activation(case["function"], case["limit"], case["offset"], gated)
        state["order"] = {"interleaved": GateUpOrder.INTERLEAVED, "concatenated": GateUpOrder.CONCATENATED}.get(case["order"])
    else:
        from crosspool_amd.ffn import RouterAlgorithm
        from crosspool_amd.moe import BalanceLoss

        scores = {"softmax": RouterAlgorithm.SOFTMAX, "sigmoid": RouterAlgorithm.SIGMOID}[case["scores"]]
        state["operator"] = BalanceLoss(row_capacity=case["rows"], routed_expert_count=case["experts"],
                                        routed_topk=case["topk"], algorithm=scores, coefficient=0.01, device=device)


def _activation(name, limit, offset, gated):
    from crosspool_amd.ffn import GateTransform, GeluActivation, ReluActivation, SiluActivation
    from crosspool_amd.operators import Activation

    function = {"silu": SiluActivation(), "relu": ReluActivation(), "gelu": GeluActivation(),
                "gelu_tanh": GeluActivation("tanh")}[name]
    return Activation(function, GateTransform(limit or None, offset) if gated else None)


# ------------------------------------------------------------------ passes
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state, kind)
    if kind == "adapt":
        return _adapt_plain(state)
    if kind == "adapt_grad":
        return _adapt_grad_plain(state)
    if kind == "act_grad":
        return _act_grad_plain(state)
    return _balance_plain(state, kind == "balance_step")


def _run_own(state, kind):
    if kind == "adapt":
        state["operator"].run_into(state["x"], state["weights"], adapter_ids=state["ids"], base=state["base"],
                                   output=state["out"], activation=state["activation"])
        return state["out"]
    if kind == "adapt_grad":
        state["operator"].backward_into(state["x"], state["grad"], state["weights"], adapter_ids=state["ids"],
                                        base=state["base"], grad_inputs=state["out"], grad_a=state["grad_a"],
                                        grad_b=state["grad_b"])
        return {"inputs": state["out"], "a": state["grad_a"], "b": state["grad_b"]}
    if kind == "act_grad":
        state["activation"].backward_into(inputs=state["inputs"], grad_output=state["grad"], grad_inputs=state["out"],
                                          order=state["order"])
        return state["out"]
    operator = state["operator"]
    operator.run_into(logits=state["logits"], ids=state["ids"], payload_rows=state["live"])
    if kind == "balance":
        return {"counts": operator.counts, "loss": operator.loss}
    operator.backward_into(logits=state["logits"], grad_logits=state["out"], grad_loss=state["grad_loss"],
                           payload_rows=state["live"])
    return {"counts": operator.counts, "loss": operator.loss, "logits": state["out"]}


def _pool(state):
    """All adapters as one pair of matrices ([A R, K] and [N, A R]), columns past a rank cleared, and what each
    row takes of them ([rows, A R]: its adapter's scale or zero)."""

    count, rank, k = state["a"].shape
    n = state["b"].shape[1]
    device = state["a"].device
    within = torch.arange(rank, device=device) < state["ranks"][:, None]
    a = (state["a"].float() * within[:, :, None]).reshape(count * rank, k)
    b = (state["b"].float() * within[:, None, :]).transpose(0, 1).reshape(n, count * rank)
    taken = (state["ids"][:, None] == torch.arange(count, device=device)) * state["scales"]
    return a, b, taken.repeat_interleave(rank, dim=1)


def _gelu(v):
    return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))


def _adapt_plain(state):
    a, b, taken = _pool(state)
    x = state["x"].float()
    out = state["base"].float() + ((x @ a.T) * taken) @ b.T
    activation = state["case"]["activation"]
    if activation != "none":
        gate, up = out[:, 0::2], out[:, 1::2]
        out = (gate / (1 + torch.exp(-gate)) if activation == "silu" else _gelu(gate)) * up
    return out.to(state["x"].dtype)


def _adapt_grad_plain(state):
    a, b, taken = _pool(state)
    count, rank, k = state["a"].shape
    x, grad, dtype = state["x"].float(), state["grad"].float(), state["x"].dtype
    up = (grad @ b) * taken
    down = (x @ a.T) * taken
    grad_a = (up.T @ x).reshape(count, rank, k)
    grad_b = (grad.T @ down).reshape(-1, count, rank).transpose(0, 1)
    return {"inputs": (state["base"].float() + up @ a).to(dtype), "a": grad_a.to(dtype),
            "b": grad_b.contiguous().to(dtype)}


def _act_grad_plain(state):
    case = state["case"]
    values, grad = state["inputs"].float(), state["grad"].float()
    width = case["width"]
    if case["order"] == "interleaved":
        gate, up = values[:, 0::2], values[:, 1::2]
    elif case["order"] == "concatenated":
        gate, up = values[:, :width], values[:, width:]
    else:
        gate, up = values, None
    limit, function = case["limit"], case["function"]
    clipped = torch.clamp(gate, max=limit) if limit else gate
    if function == "silu":
        share = 1 / (1 + torch.exp(-clipped))
        value, slope = clipped * share, share * (1 + clipped * (1 - share))
    elif function == "relu":
        value, slope = torch.clamp(clipped, min=0), (clipped > 0).float()
    elif function == "gelu":
        share = 0.5 * (1 + torch.erf(clipped * math.sqrt(0.5)))
        value, slope = clipped * share, share + clipped * torch.exp(-0.5 * clipped * clipped) / math.sqrt(2 * math.pi)
    else:
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (clipped + 0.044715 * clipped * clipped * clipped))
        value = 0.5 * clipped * (1 + t)
        slope = 0.5 * (1 + t) + 0.5 * clipped * (1 - t * t) * c * (1 + 3 * 0.044715 * clipped * clipped)
    dtype = state["inputs"].dtype
    if up is None:
        return (grad * slope).to(dtype)
    factor = torch.clamp(up, -limit, limit) if limit else up
    grad_gate, grad_up = grad * slope * (factor + case["offset"]), grad * value
    if limit:
        grad_gate, grad_up = grad_gate * (gate <= limit), grad_up * (up.abs() <= limit)
    if case["order"] == "interleaved":
        return torch.stack((grad_gate, grad_up), dim=2).flatten(1).to(dtype)
    return torch.cat((grad_gate, grad_up), dim=1).to(dtype)


def _balance_plain(state, step):
    case = state["case"]
    experts, topk = case["experts"], case["topk"]
    logits, ids = state["logits"].float(), state["ids"]
    rows = torch.arange(logits.shape[0], device=logits.device)[:, None] < state["live"]
    chosen = torch.where((ids >= 0) & rows, ids, experts).flatten().long()
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=logits.device)
    counts = counts.scatter_add(0, chosen, torch.ones_like(chosen, dtype=torch.int32))[:experts]
    live = state["live"].float()
    if case["scores"] == "softmax":
        score = torch.exp(logits - logits.amax(dim=1, keepdim=True))
        slope = 1.0
    else:
        score = 1 / (1 + torch.exp(-logits))
        slope = 1 - score
    share = torch.where(rows, score / score.sum(dim=1, keepdim=True), 0.0)
    load = counts * (experts / (topk * live))
    mean = share.sum(dim=0, dtype=torch.float64) / live
    found = {"counts": counts, "loss": (0.01 * (load * mean).sum(dtype=torch.float64)).float().reshape(1)}
    if step:
        centred = load - (share * load).sum(dim=1, keepdim=True)
        found["logits"] = (0.01 * state["grad_loss"] / live * share * slope * centred).to(state["logits"].dtype)
    return found


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"adapt": _adapt_exact, "adapt_grad": _adapt_grad_exact, "act_grad": _act_grad_exact,
            "balance": _balance_exact, "balance_step": _balance_exact}[case["kind"]](state)


def _groups(state):
    """(rows, adapter, rank, scale) of each adapter that has rows."""

    for adapter, rank in enumerate(_ranks(state["case"])):
        rows = (state["ids"] == adapter).nonzero().flatten()
        if rows.numel():
            yield rows, adapter, rank, float(state["scales"][adapter])


def _adapt_exact(state):
    out = state["base"].double()
    for rows, adapter, rank, scale in _groups(state):
        low = state["x"][rows].double() @ state["a"][adapter, :rank].double().t().contiguous()
        out[rows] += scale * (low @ state["b"][adapter, :, :rank].double().t().contiguous())
    activation = state["case"]["activation"]
    if activation == "none":
        return out
    pairs = out.view(out.shape[0], -1, 2)
    gate = pairs[..., 0]
    return gate * (torch.sigmoid(gate) if activation == "silu" else torch.special.ndtr(gate)) * pairs[..., 1]


def _adapt_grad_exact(state):
    grad_inputs = state["base"].double()
    grad_a, grad_b = torch.zeros_like(state["a"], dtype=torch.float64), torch.zeros_like(state["b"], dtype=torch.float64)
    for rows, adapter, rank, scale in _groups(state):
        a, b = state["a"][adapter, :rank].double(), state["b"][adapter, :, :rank].double().contiguous()
        x, grad = state["x"][rows].double(), state["grad"][rows].double()
        through = scale * (grad @ b)
        grad_inputs[rows] += through @ a
        grad_a[adapter, :rank] = through.t().contiguous() @ x
        grad_b[adapter, :, :rank] = scale * (grad.t().contiguous() @ (x @ a.t().contiguous()))
    return {"inputs": grad_inputs, "a": grad_a, "b": grad_b}


def _act_grad_exact(state):
    """Through torch's own gradients of the definition."""

    case = state["case"]
    values = state["inputs"].double().requires_grad_(True)
    width, limit = case["width"], case["limit"] or None
    gated = case["order"] != "ungated"
    gate = values[:, 0::2] if case["order"] == "interleaved" else values[:, :width]
    if limit:
        gate = gate.clamp(max=limit)
    names = {"silu": torch.nn.functional.silu, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}
    out = names[case["function"]](gate)
    if gated:
        up = values[:, 1::2] if case["order"] == "interleaved" else values[:, width:]
        out = out * ((up.clamp(-limit, limit) if limit else up) + case["offset"])
    (found,) = torch.autograd.grad(out, values, state["grad"].double())
    return found


def _balance_exact(state):
    case = state["case"]
    experts, topk, live = case["experts"], case["topk"], _live(case)
    logits = state["logits"][:live].double().requires_grad_(True)
    if case["scores"] == "softmax":
        share = torch.softmax(logits, dim=1)
    else:
        share = torch.sigmoid(logits)
        share = share / share.sum(dim=1, keepdim=True)
    counts = torch.bincount(state["ids"][:live].flatten().long(), minlength=experts)
    loss = 0.01 * (counts.double() * experts / (topk * live) * share.mean(dim=0)).sum()
    found = {"counts": counts.to(torch.int32), "loss": loss.detach().reshape(1)}
    if case["kind"] == "balance_step":
        (grad,) = torch.autograd.grad(loss, logits)
        full = torch.zeros(state["logits"].shape, dtype=torch.float64, device=grad.device)
        full[:live] = grad * state["grad_loss"].double()
        found["logits"] = full
    return found
