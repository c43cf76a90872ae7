"""Per-expert counts, the balance loss and its gradient, against the definition in 64 bits.

Tolerances, from the arithmetic: a score is exp of an fp32 difference x (off by |x| 2^-24, so its
exponential by as much relatively, plus 2 units in the last place), divided by a sum of E of them; the loss
adds at most T such values per expert.  With X the largest |x| of a case: relative errors of at most
(E + T + 2 X + 16) 2^-24 for the loss (all terms positive) and (2 E + 4 X + 32) 2^-24 of
c/T p (f + sum f p) for the gradient, plus half a step of the logits' dtype at its store.
"""

from __future__ import annotations

import pytest
import torch

from crosspool_amd import _native
from crosspool_amd.ffn import RouterAlgorithm
from crosspool_amd.moe import BalanceLoss, MoeRouterWeights, Router

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
UNIT = 2.0**-24


def rounding(value, dtype):
    smallest = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}[dtype]
    return value.abs() * torch.finfo(dtype).eps / 2 + smallest


def make(rows, experts, topk, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((rows, experts), generator=g) * 2 + torch.randn(experts, generator=g)).to(DTYPES[dtype])
    ids = torch.topk(logits.float(), topk, dim=1).indices.to(torch.int32)
    return logits, ids


def definition(logits, ids, experts, topk, live, coefficient, algorithm, upstream=1.0):
    """(counts, loss, gradient [rows, experts], its magnitude) in 64 bits; all-(-inf) rows score nothing."""

    values = logits[:live].double()
    if algorithm is RouterAlgorithm.SOFTMAX:
        most = values.amax(dim=1, keepdim=True)
        score = torch.exp(values - torch.where(most == float("-inf"), 0.0, most))
        slope = torch.ones_like(score)
    else:
        score = torch.sigmoid(values)
        slope = 1 - score
    total = score.sum(dim=1, keepdim=True)
    share = torch.where(total == 0, 0.0, score / total)
    chosen = ids[:live].flatten().long()
    counts = torch.bincount(chosen[(chosen >= 0) & (chosen < experts)], minlength=experts)
    load = counts.double() * experts / (topk * max(live, 1))
    loss = coefficient * float((load * share.sum(dim=0)).sum()) / max(live, 1)
    factor = coefficient * upstream / max(live, 1)
    mean = (share * load).sum(dim=1, keepdim=True)
    grad = torch.zeros(logits.shape, dtype=torch.float64)
    size = torch.zeros_like(grad)
    grad[:live] = factor * share * slope * (load - mean)
    size[:live] = abs(factor) * share * (load + mean)
    return counts.to(torch.int32), loss, grad, size


def check(operator, logits, ids, *, live=None, upstream=None, device):
    rows, experts = logits.shape
    effective = rows if live is None else max(0, min(live, rows))
    payload = None if live is None else torch.tensor([live], dtype=torch.int32, device=device)
    gl = None if upstream is None else torch.tensor([upstream], device=device)
    on_device = logits.to(device)
    grad = torch.full_like(on_device, float("nan"))
    operator.counts.fill_(-7)
    operator.loss.fill_(float("nan"))
    operator.run_into(logits=on_device, ids=ids.to(device), payload_rows=payload)
    operator.backward_into(logits=on_device, grad_logits=grad, grad_loss=gl, payload_rows=payload)
    counts, loss, expected, size = definition(logits, ids, experts, operator.routed_topk, effective,
                                              operator.coefficient, operator.algorithm, 1.0 if upstream is None else upstream)
    finite = logits[:effective].double()
    finite = finite[finite.isfinite()]
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    assert torch.equal(operator.counts.cpu(), counts)
    assert abs(float(operator.loss) - loss) <= abs(loss) * (experts + effective + 2 * spread + 16) * UNIT + 2.0**-149
    got = grad.cpu().double()
    allowed = size * (2 * experts + 4 * spread + 32) * UNIT
    allowed = allowed + rounding(expected.abs() + allowed, logits.dtype)
    assert bool(((got - expected).abs() <= allowed).all()), float(((got - expected).abs() - allowed).max())
    return grad


@pytest.mark.parametrize("algorithm", list(RouterAlgorithm))
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,experts,topk", [
    (1, 1, 1), (1, 8, 2), (3, 5, 5), (64, 128, 8), (17, 60, 4), (255, 64, 6), (256, 65, 1), (257, 128, 8), (300, 129, 8),
    (1000, 256, 8), (515, 257, 3), (700, 511, 8), (400, 1000, 8), (333, 1024, 64), (20000, 8, 2), (70001, 16, 2),
])
def test_counts_loss_and_gradient_match_the_definition(device, rows, experts, topk, dtype, algorithm):
    logits, ids = make(rows, experts, topk, dtype, seed=rows + experts)
    operator = BalanceLoss(row_capacity=rows, routed_expert_count=experts, routed_topk=topk, algorithm=algorithm,
                           coefficient=0.5)
    check(operator, logits, ids, device=device)
    # fp16 gradients of a mean are small: a loss scale as training uses brings them among normal numbers.
    check(operator, logits, ids, upstream=float(rows) * 16, device=device)


@pytest.mark.parametrize("live", [-3, 0, 1, 99, 300, 1000])
def test_live_rows(device, live):
    logits, ids = make(300, 96, 4, "fp32", seed=2)
    logits[max(live, 0):] = float("nan")  # what lies behind the live rows must not matter
    operator = BalanceLoss(row_capacity=512, routed_expert_count=96, routed_topk=4, coefficient=0.01)
    grad = check(operator, logits, ids, live=live, upstream=3.0, device=device)
    assert not bool(grad[max(live, 0):].any())


@pytest.mark.parametrize("algorithm", list(RouterAlgorithm))
def test_masked_experts_and_rows_that_mask_them_all(device, algorithm):
    logits, ids = make(400, 72, 3, "fp32", seed=3)
    logits[:, 5] = float("-inf")
    logits[7] = float("-inf")
    logits[8] = torch.finfo(torch.float32).min
    logits[399, 1:] = float("-inf")
    ids[7] = -1
    ids[9, 1] = 72   # a shared expert's id
    ids[10, 2] = 2_000_000_000
    operator = BalanceLoss(row_capacity=400, routed_expert_count=72, routed_topk=3, algorithm=algorithm)
    if algorithm is RouterAlgorithm.SIGMOID:
        logits[8] = -80.0  # the lowest value's sigmoids are all zero: a row like 7
    grad = check(operator, logits, ids, device=device)
    # Row 8 holds the type's lowest value everywhere, expert 5 among them: equal scores, nothing masked.
    masked = grad[:, 5][torch.arange(400, device=device) != 8]
    assert not bool(grad[7].any()) and not bool(masked.any())


def test_nan_stays_in_its_row_of_the_gradient(device):
    logits, ids = make(300, 64, 2, "bf16", seed=4)
    operator = BalanceLoss(row_capacity=300, routed_expert_count=64, routed_topk=2)
    clean = check(operator, logits, ids, device=device)
    logits[11, 3] = float("nan")
    grad = torch.empty_like(clean)
    operator.run_into(logits=logits.to(device), ids=ids.to(device))
    assert bool(operator.loss.isnan())
    operator.backward_into(logits=logits.to(device), grad_logits=grad)
    assert bool(grad[11].isnan().all())
    keep = torch.arange(300, device=device) != 11
    assert torch.equal(grad[keep], clean[keep])


def test_scores_at_the_end_of_the_exponents_range(device):
    """exp(88.72) is within half a unit of the largest fp32 number, and the inverse of its inverse past it."""

    first = torch.linspace(-88.75, -88.69, 61)
    logits = torch.full((61, 8), -200.0)
    logits[:, 3] = first
    ids = torch.full((61, 2), 3, dtype=torch.int32)
    operator = BalanceLoss(row_capacity=61, routed_expert_count=8, routed_topk=2, coefficient=0.5,
                           algorithm=RouterAlgorithm.SIGMOID)
    grad = torch.full((61, 8), float("nan"), device=device)
    operator.run_into(logits=logits.to(device), ids=ids.to(device))
    operator.backward_into(logits=logits.to(device), grad_logits=grad)
    assert bool(torch.isfinite(grad).all()) and 0.0 <= float(operator.loss) <= 0.5 * 8 * (1 + 2.0**-16)


def test_gradient_matches_differences(device):
    """Central differences with a step of 2^-6: the third derivative (below c f_max / T) leaves h^2 / 6 of it,
    and the fp32 loss (about 1) 2^-24 / 2^-6 of rounding: 2^-13 / T in all is ample for the first."""

    rows, experts = 40, 12
    logits, ids = make(rows, experts, 2, "fp32", seed=5)
    operator = BalanceLoss(row_capacity=rows, routed_expert_count=experts, routed_topk=2)
    grad = check(operator, logits, ids, device=device).cpu()

    def loss():
        operator.run_into(logits=logits.to(device), ids=ids.to(device))
        return float(operator.loss)

    h = 2.0**-6
    for place in ((0, 0), (39, 11), (20, 3)):
        kept = float(logits[place])
        logits[place] = kept + h
        above = loss()
        logits[place] = kept - h
        below = loss()
        logits[place] = kept
        assert abs((above - below) / (2 * h) - float(grad[place])) <= 12 * h * h / 6 / rows + 2 * 2.0**-23 / (2 * h)


def test_counts_alone_repeatability_and_gradient_in_place(device):
    logits, ids = make(5000, 128, 8, "fp32", seed=6)
    operator = BalanceLoss(row_capacity=8192, routed_expert_count=128, routed_topk=8)
    first = check(operator, logits, ids, device=device)
    counts, loss = operator.counts.clone(), operator.loss.clone()
    operator.loss.fill_(42.0)
    operator.counts.zero_()
    operator.run_into(ids=ids.to(device))
    assert torch.equal(operator.counts, counts) and float(operator.loss) == 42.0
    operator.run_into(logits=logits.to(device), ids=ids.to(device))
    assert torch.equal(operator.loss, loss)
    inplace = logits.to(device)
    operator.backward_into(logits=inplace, grad_logits=inplace, counts=counts)
    assert torch.equal(inplace, first)


def test_no_rows(device):
    operator = BalanceLoss(row_capacity=4, routed_expert_count=8, routed_topk=2)
    operator.counts.fill_(3)
    operator.loss.fill_(3.0)
    empty = torch.empty((0, 8), device=device)
    operator.run_into(logits=empty, ids=torch.empty((0, 2), dtype=torch.int32, device=device))
    assert not bool(operator.counts.any()) and float(operator.loss) == 0.0
    operator.backward_into(logits=empty, grad_logits=empty)


def test_captured_step_replays_over_new_logits_and_live_rows(device):
    logits, ids = make(1500, 128, 8, "bf16", seed=7)
    operator = BalanceLoss(row_capacity=1500, routed_expert_count=128, routed_topk=8, coefficient=0.1)
    x, i = logits.to(device), ids.to(device)
    payload = torch.tensor([1500], dtype=torch.int32, device=device)
    upstream = torch.ones(1, device=device)
    grad = torch.empty_like(x)

    def step():
        operator.run_into(logits=x, ids=i, payload_rows=payload)
        operator.backward_into(logits=x, grad_logits=grad, grad_loss=upstream, payload_rows=payload)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    other = BalanceLoss(row_capacity=1500, routed_expert_count=128, routed_topk=8, coefficient=0.1)
    for seed, live in ((8, 1500), (9, 700), (10, 3)):
        logits, ids = make(1500, 128, 8, "bf16", seed=seed)
        x.copy_(logits)
        i.copy_(ids)
        payload.fill_(live)
        upstream.fill_(float(seed))
        graph.replay()
        torch.cuda.synchronize()
        expected = check(other, logits, ids, live=live, upstream=float(seed), device=device)
        assert torch.equal(operator.counts, other.counts) and torch.equal(operator.loss, other.loss)
        assert torch.equal(grad, expected)


def test_balance_of_a_router(device):
    """A Router's own logits and ids, as a training step has them."""

    rows, hidden, experts, topk = 200, 256, 32, 4
    g = torch.Generator().manual_seed(0)
    x = torch.randn((rows, hidden), generator=g).to(torch.bfloat16)
    w = (torch.randn((experts, hidden), generator=g) * 0.1).to(torch.bfloat16)
    router = Router(row_capacity=rows, hidden_size=hidden, routed_expert_count=experts, routed_topk=topk)
    router.run_into(hidden_states=x.to(device), router_weights=MoeRouterWeights(w.to(device)))
    operator = BalanceLoss(row_capacity=rows, routed_expert_count=experts, routed_topk=topk, coefficient=0.01)
    check(operator, router.logits.cpu(), router.ids.cpu(), device=device)


def test_refusals_on_the_device(device):
    logits, ids = make(10, 16, 2, "fp32")
    logits, ids = logits.to(device), ids.to(device)
    operator = BalanceLoss(row_capacity=10, routed_expert_count=16, routed_topk=2)
    for kwargs in (
        dict(logits=logits[:9], ids=ids), dict(logits=logits.double(), ids=ids), dict(logits=logits, ids=ids.long()),
        dict(logits=logits, ids=ids[:, :1]), dict(logits=logits.cpu(), ids=ids),
        dict(logits=logits, ids=ids, payload_rows=torch.tensor([3], device=device)),
        dict(logits=logits.t().contiguous().t(), ids=ids),
    ):
        with pytest.raises(ValueError):
            operator.run_into(**kwargs)
    with pytest.raises(ValueError, match="capacity"):
        operator.run_into(ids=torch.cat((ids, ids)))
    with pytest.raises(ValueError):
        operator.backward_into(logits=logits, grad_logits=logits.half())
    with pytest.raises(ValueError):
        operator.backward_into(logits=logits, grad_logits=torch.empty_like(logits), grad_loss=torch.ones(2, device=device))
    assert operator.workspace.numel() == 16
    big = BalanceLoss(row_capacity=4096, routed_expert_count=16, routed_topk=2)
    assert big.workspace.numel() == _native.library().xp_moe_balance_workspace_bytes(4096, 16) > 0


def sigmoid_definition(logits, ids, topk, coefficient, upstream=1.0):
    """(loss, gradient, its size) of the sigmoid scores in 64 bits for logits of any finite size: with m the row's
    largest logit or 0, score_e = exp(min(l, 0) - m) / (1 + exp(-|l|)) keeps the ratios where sigmoids underflow."""

    rows, experts = logits.shape
    values = logits.double()
    most = values.amax(dim=1, keepdim=True).clamp(max=0)
    small = torch.exp(-values.abs())
    score = torch.exp(values.clamp(max=0) - most) / (1 + small)
    slope = torch.where(values > 0, small, 1.0) / (1 + small)
    share = score / score.sum(dim=1, keepdim=True)
    counts = torch.bincount(ids.flatten().long(), minlength=experts)
    load = counts.double() * experts / (topk * rows)
    loss = coefficient * float((load * share.sum(dim=0)).sum()) / rows
    factor = coefficient * upstream / rows
    mean = (share * load).sum(dim=1, keepdim=True)
    return loss, factor * share * slope * (load - mean), abs(factor) * share * slope * (load + mean)


def check_sigmoid(device, logits, ids, topk, spread):
    """``spread``: the largest exponent that an exp of the case takes (the file's X)."""

    rows, experts = logits.shape
    operator = BalanceLoss(row_capacity=rows, routed_expert_count=experts, routed_topk=topk, coefficient=0.5,
                           algorithm=RouterAlgorithm.SIGMOID)
    grad = torch.full_like(logits.to(device), float("nan"))
    upstream = torch.tensor([float(rows) * 16], device=device)
    operator.run_into(logits=logits.to(device), ids=ids.to(device))
    operator.backward_into(logits=logits.to(device), grad_logits=grad, grad_loss=upstream)
    loss, expected, size = sigmoid_definition(logits, ids, topk, 0.5, float(rows) * 16)
    assert abs(float(operator.loss) - loss) <= abs(loss) * (experts + rows + 2 * spread + 16) * UNIT
    allowed = size * (2 * experts + 4 * spread + 32) * UNIT
    allowed = allowed + rounding(expected.abs() + allowed, logits.dtype)
    assert bool(((grad.cpu().double() - expected).abs() <= allowed).all())
    return grad


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("experts", [8, 128, 300])
def test_saturated_sigmoids_keep_their_slope(device, experts, dtype):
    """Logits of 10 to 30: 1 - sigmoid is e^-l / (1 + e^-l), from 5e-5 to 1e-13 and not zero."""

    g = torch.Generator().manual_seed(experts)
    logits = (torch.rand((300, experts), generator=g) * 20 + 10).to(DTYPES[dtype])
    ids = torch.topk(logits.float(), 2, dim=1).indices.to(torch.int32)
    grad = check_sigmoid(device, logits, ids, 2, 30.0)
    # Every share is 1 / experts within 2^-14: an expert of the average load, f = 1, is alone in having no gradient.
    uneven = torch.bincount(ids.flatten().long(), minlength=experts) * experts != ids.numel()
    assert bool((grad.cpu()[:, uneven] != 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("experts", [8, 64, 100, 300])
@pytest.mark.parametrize("level", [-70.0, -95.0, -200.0, -30000.0])
def test_rows_of_low_sigmoid_logits_keep_their_ratios(device, level, experts, dtype):
    """A row of finite logits has a share for each of them, however low they all are."""

    logits, ids = make(300, experts, 2, dtype, seed=experts)
    logits[5:] = (logits[5:].float() + level).to(DTYPES[dtype])   # beside rows of ordinary ones
    grad = check_sigmoid(device, logits, ids, 2, 40.0)
    if dtype == "fp32":   # (in 16 bits the lowest levels round to ties)
        assert bool((grad[5:].abs().amax(dim=1) > 0).all())


def test_the_lowest_logits_share_alike(device):
    logits = torch.full((300, 16), torch.finfo(torch.float32).min)
    ids = torch.zeros((300, 1), dtype=torch.int32)
    check_sigmoid(device, logits, ids, 1, 1.0)


def test_an_operators_buffers_stay_its_own(device):
    operator = BalanceLoss(row_capacity=4096, routed_expert_count=16, routed_topk=2)
    for name in ("workspace", "counts", "loss"):
        with pytest.raises(AttributeError):
            setattr(operator, name, getattr(operator, name)[:1].clone())
    logits, ids = make(4096, 16, 2, "fp32")
    check(operator, logits, ids, device=device)
