"""Low-rank adapters beside a projection and their gradients, against the definition in 64 bits.

Tolerances follow from the kernels' arithmetic, before any run.  Every sum is fp32 over exact products
(16-bit payloads) or fp32 products (fp32 payloads): a sum of n terms is off by at most n 2^-24 of the
sum of its terms' magnitudes, the bound used here with those magnitudes computed in 64 bits.  16-bit
payloads multiply t (u) as two bf16 terms, off by at most 2^-16 of its magnitude.  The result is rounded
once to the payload dtype, off by half a step: ``finfo.eps / 2`` of the value, or half the smallest
subnormal of fp16.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from crosspool_amd import _native
from crosspool_amd.adapters import Adapter, AdapterPlan, AdapterWeights, interleave_gate_up_adapters
from crosspool_amd.ffn import GateTransform, GeluActivation, ReluActivation, SiluActivation
from crosspool_amd.operators import Activation

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
UNIT = 2.0**-24


def rounding(value: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Half a step of ``dtype`` at ``value`` (and at its smallest subnormal)."""

    smallest = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}[dtype]
    return value.abs() * torch.finfo(dtype).eps / 2 + smallest


class Case:
    """A pool, a batch and what the operators must give for it (on the CPU, in 64 bits)."""

    def __init__(self, device, *, rows, k, n, count, max_rank, dtype="bf16", ranks=None, ids="random", seed=0):
        g = torch.Generator().manual_seed(seed)
        self.device, self.dtype = device, DTYPES[dtype]
        self.rows, self.k, self.n, self.count, self.max_rank = rows, k, n, count, max_rank

        def normal(*shape, std):
            return (torch.randn(shape, generator=g) * std).to(self.dtype)

        self.a = normal(count, max_rank, k, std=k**-0.5)
        self.b = normal(count, n, max_rank, std=max_rank**-0.5)
        self.scales = torch.rand(count, generator=g) + 0.5
        self.ranks = None if ranks is None else torch.tensor(ranks, dtype=torch.int32)
        if ids == "random":
            self.ids = torch.randint(-1, count, (rows,), generator=g, dtype=torch.int32)
        else:
            self.ids = torch.tensor(ids, dtype=torch.int32)
        self.x = normal(rows, k, std=1.0)
        self.base = normal(rows, n, std=1.0)
        self.grad = normal(rows, n, std=0.1)
        self.grad_base = normal(rows, k, std=0.5)

    def rank(self, adapter):
        return self.max_rank if self.ranks is None else max(0, min(int(self.ranks[adapter]), self.max_rank))

    def weights(self):
        to = lambda t: None if t is None else t.to(self.device)  # noqa: E731
        return AdapterWeights(to(self.a), to(self.b), to(self.scales), to(self.ranks))

    def operator(self, backward=False, capacity=None):
        plan = AdapterPlan.prepare(row_capacity=capacity or max(self.rows, 1), adapter_count=self.count,
                                   max_rank=self.max_rank, input_width=self.k, output_width=self.n, dtype=self.dtype,
                                   backward=backward)
        # NaN bytes: whatever the scratch holds must not matter.
        return Adapter(plan, torch.full((plan.workspace.nbytes,), 0xFF, dtype=torch.uint8, device=self.device))

    def groups(self):
        for adapter in range(self.count):
            rows = (self.ids == adapter).nonzero().flatten()
            rank = self.rank(adapter)
            if rows.numel():
                yield rows, self.a[adapter, :rank].double(), self.b[adapter, :, :rank].double(), \
                    float(self.scales[adapter]), adapter, rank

    @property
    def terms(self):
        """Relative error of the multiplied t: two bf16 terms, or fp32 as it is."""

        return 0.0 if self.dtype is torch.float32 else 2.0**-16

    def forward(self):
        """(the sums in 64 bits, a bound on the fp32 error before the store)."""

        value = self.base.double()
        bound = value.abs() * 2 * UNIT
        for rows, a, b, scale, _, rank in self.groups():
            x = self.x[rows].double()
            t, t_size = x @ a.T, x.abs() @ a.abs().T
            low = scale * (t @ b.T)
            # t: k terms; the product: rank terms (twice with the two-term split); scale and base: 2 roundings.
            size = t_size @ b.abs().T
            bound[rows] += scale * size * ((self.k + 2 * rank + 8) * UNIT) + scale * (t.abs() @ b.abs().T) * self.terms
            value[rows] += low
        return value, bound + value.abs() * 2 * UNIT

    def backward(self):
        """{name: (value in 64 bits, bound before the store)} of the three gradients."""

        gx = self.grad_base.double()
        gx_bound = gx.abs() * 2 * UNIT
        ga = torch.zeros(self.a.shape, dtype=torch.float64)
        gb = torch.zeros(self.b.shape, dtype=torch.float64)
        ga_bound, gb_bound = torch.zeros_like(ga), torch.zeros_like(gb)
        for rows, a, b, scale, adapter, rank in self.groups():
            x, dy = self.x[rows].double(), self.grad[rows].double()
            t, t_size = x @ a.T, x.abs() @ a.abs().T
            u, u_size = dy @ b, dy.abs() @ b.abs()
            gx[rows] += scale * (u @ a)
            gx_bound[rows] += scale * (u_size @ a.abs()) * ((self.n + 2 * rank + 8) * UNIT) \
                + scale * (u.abs() @ a.abs()) * self.terms
            ga[adapter, :rank] = scale * (u.T @ x)
            gb[adapter, :, :rank] = scale * (dy.T @ t)
            m = rows.numel()
            ga_bound[adapter, :rank] = scale * (u_size.T @ x.abs()) * ((self.n + 2 * m + 8) * UNIT) \
                + scale * (u.abs().T @ x.abs()) * self.terms
            gb_bound[adapter, :, :rank] = scale * (dy.abs().T @ t_size) * ((self.k + 2 * m + 8) * UNIT) \
                + scale * (dy.abs().T @ t.abs()) * self.terms
        return {"x": (gx, gx_bound + gx.abs() * 2 * UNIT), "a": (ga, ga_bound), "b": (gb, gb_bound)}


def assert_within(actual: torch.Tensor, value: torch.Tensor, bound: torch.Tensor, dtype: torch.dtype, what: str) -> None:
    actual = actual.detach().cpu().double()
    assert actual.shape == value.shape
    allowed = bound + rounding(value.abs() + bound, dtype)
    excess = (actual - value).abs() - allowed
    assert bool((excess <= 0).all()), \
        f"{what}: {int((~(excess <= 0)).sum())} of {excess.numel()} beyond the bound, worst by {float(excess.max()):.3e}"


def run(case, operator=None, **kwargs):
    out = torch.full((case.rows, case.n), float("nan"), dtype=case.dtype, device=case.device)
    (operator or case.operator()).run_into(case.x.to(case.device), case.weights(), adapter_ids=case.ids.to(case.device),
                                           base=case.base.to(case.device), output=out, **kwargs)
    return out


def check_forward(case, out):
    value, bound = case.forward()
    assert_within(out, value, bound, case.dtype, "output")
    none = case.ids == -1
    # Rows without an adapter are base's bits.
    bits = torch.int32 if case.dtype is torch.float32 else torch.int16
    assert torch.equal(out.cpu()[none].view(bits), case.base[none].view(bits))


FORWARD = [
    # rows, k, n, count, max_rank, ranks
    (1, 64, 48, 1, 8, None),
    (1, 1, 1, 1, 1, None),
    (1, 4096, 1024, 3, 16, None),
    (2, 33, 7, 2, 3, [3, 1]),
    (15, 257, 130, 4, 16, [16, 5, 0, 9]),
    (17, 512, 333, 1, 32, None),
    (40, 1000, 264, 3, 33, [33, 32, 17]),
    (64, 768, 520, 64, 64, None),
    (64, 2048, 96, 2, 128, [128, 65]),
    (65, 320, 200, 5, 24, [24, 8, 16, 1, 24]),
    (127, 513, 1027, 3, 100, None),
    (300, 260, 515, 7, 12, [12, 4, 6, 12, 3, 200, -5]),
    (1000, 640, 384, 16, 16, None),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k,n,count,max_rank,ranks", FORWARD)
def test_forward_matches_the_definition(device, rows, k, n, count, max_rank, ranks, dtype):
    case = Case(device, rows=rows, k=k, n=n, count=count, max_rank=max_rank, ranks=ranks, dtype=dtype, seed=rows + k)
    check_forward(case, run(case))


@pytest.mark.parametrize("ids", ["none", "one", "last", "runs"])
@pytest.mark.parametrize("rows", [1, 63, 64, 65, 200])
def test_batches_of_one_adapter_or_none(device, rows, ids):
    chosen = {"none": [-1] * rows, "one": [0] * rows, "last": [4] * rows,
              "runs": [i * 6 // rows - 1 for i in range(rows)]}[ids]
    case = Case(device, rows=rows, k=384, n=272, count=5, max_rank=16, ids=chosen, seed=rows)
    check_forward(case, run(case))


def test_large_pools_and_many_groups(device):
    case = Case(device, rows=2500, k=72, n=40, count=1024, max_rank=4, seed=5)
    check_forward(case, run(case))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("k", [3, 4, 5, 7, 8, 9, 15, 31, 32, 39, 66, 1030])
def test_widths_that_cut_a_chunk(device, k, dtype):
    for rows in (7, 80):
        case = Case(device, rows=rows, k=k, n=k, count=2, max_rank=20, ranks=[20, 9], dtype=dtype, seed=k)
        check_forward(case, run(case))
        check_backward(case, backward(case))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [5, 70])
def test_an_infinity_before_a_cut_chunk_is_counted_once(device, rows, dtype):
    """Rank 1: an infinite product is the sum, its sign B's; taken a second time times zero it would be NaN."""

    for column in (5, 6, 11, 12):
        case = Case(device, rows=rows, k=13, n=24, count=1, max_rank=1, dtype=dtype, ids=[0] * rows)
        case.a.abs_().clamp_(min=0.25)
        case.x[2, column] = float("inf")
        got = run(case).cpu()
        expected = torch.where(case.b[0, :, 0] > 0, float("inf"), -float("inf"))
        assert torch.equal(got[2].float(), expected)
        assert bool(torch.isfinite(got[torch.arange(rows) != 2]).all())


@pytest.mark.parametrize("count", [5, 70])
@pytest.mark.parametrize("rows", [8192, 8193, 20011])
def test_more_rows_than_the_sort_keeps(device, rows, count):
    case = Case(device, rows=rows, k=24, n=40, count=count, max_rank=4, seed=rows)
    check_forward(case, run(case))
    got = backward(case)
    check_backward(case, got)
    again = backward(case)
    assert all(torch.equal(got[name], again[name]) for name in got)


def test_padding_of_the_pool_is_ignored(device):
    for rows in (20, 150):
        case = Case(device, rows=rows, k=200, n=96, count=3, max_rank=20, ranks=[20, 7, 8], seed=rows)
        expected = run(case)
        case.a[1, 7:] = float("nan")
        case.b[1, :, 7:] = float("inf")
        case.a[2, 8:] = float("inf")
        case.b[2, :, 8:] = float("nan")
        assert torch.equal(run(case), expected)


@pytest.mark.parametrize("rows", [5, 90])
def test_infinities_and_nan_stay_in_their_rows(device, rows):
    case = Case(device, rows=rows, k=100, n=60, count=2, max_rank=8, ids=[i % 2 for i in range(rows)])
    expected = run(case).cpu()
    case.x[1, 3] = float("nan")
    case.base[2, 5] = float("inf")
    got = run(case).cpu()
    assert bool(got[1].isnan().all())
    assert got[2, 5] == float("inf")
    keep = [r for r in range(rows) if r not in (1, 2)]
    assert torch.equal(got[keep], expected[keep])
    assert torch.equal(got[2, :5], expected[2, :5]) and torch.equal(got[2, 6:], expected[2, 6:])


@pytest.mark.parametrize("rows", [6, 100])
def test_ids_out_of_range_poison_their_rows_and_raise_the_fault(device, rows):
    ids = [i % 3 for i in range(rows)]
    case = Case(device, rows=rows, k=64, n=72, count=3, max_rank=8, ids=ids)
    fault = torch.zeros(1, dtype=torch.int32, device=device)
    expected = run(case, fault_word=fault).cpu()
    assert int(fault) == 0
    case.ids[1], case.ids[4] = 3, -2
    got = run(case, fault_word=fault).cpu()
    assert int(fault) == _native.XP_FAULT_ADAPTER_OUT_OF_RANGE
    assert bool(got[[1, 4]].isnan().all())
    keep = [r for r in range(rows) if r not in (1, 4)]
    assert torch.equal(got[keep], expected[keep])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [6, 100])
@pytest.mark.parametrize("activation", [
    Activation(SiluActivation(1.7), GateTransform(1.5, 1.0)),
    Activation(GeluActivation(), GateTransform(2.0)),
    Activation(ReluActivation(), None),
], ids=["silu_clipped", "gelu_clipped", "relu_ungated"])
def test_no_limit_hides_the_nan_of_an_id_out_of_range(device, activation, rows, dtype):
    ids = [i % 4 - 1 for i in range(rows)]
    case = Case(device, rows=rows, k=64, n=542, count=3, max_rank=8, dtype=dtype, ids=ids)
    outs = []
    for bad in (False, True):
        if bad:
            case.ids[1], case.ids[4] = 3, -2
        out = torch.zeros((rows, 271 if activation.gate is not None else 542), dtype=case.dtype, device=device)
        case.operator().run_into(case.x.to(device), case.weights(), adapter_ids=case.ids.to(device),
                                 base=case.base.to(device), output=out, activation=activation)
        outs.append(out.cpu())
    assert bool(outs[1][[1, 4]].isnan().all())
    keep = [r for r in range(rows) if r not in (1, 4)]
    assert torch.equal(outs[1][keep], outs[0][keep])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [3, 130])
@pytest.mark.parametrize("activation", [
    Activation(SiluActivation(), GateTransform()),
    Activation(SiluActivation(1.7), GateTransform(1.5, 1.0)),
    Activation(GeluActivation(), GateTransform()),
    Activation(GeluActivation("tanh"), None),
    Activation(ReluActivation(), None),
], ids=["silu", "silu_clipped", "gelu", "gelu_tanh_ungated", "relu_ungated"])
def test_activation_of_the_sum(device, activation, rows, dtype):
    case = Case(device, rows=rows, k=200, n=154, count=3, max_rank=16, dtype=dtype, seed=rows)
    width = case.n // 2 if activation.gate is not None else case.n
    out = torch.full((rows, width), float("nan"), dtype=case.dtype, device=device)
    case.operator().run_into(case.x.to(device), case.weights(), adapter_ids=case.ids.to(device),
                             base=case.base.to(device), output=out, activation=activation)
    value, bound = case.forward()
    function = activation.function
    if isinstance(function, SiluActivation):
        f = lambda v: v * torch.sigmoid(function.alpha * v)  # noqa: E731
    elif isinstance(function, GeluActivation):
        f = lambda v: torch.nn.functional.gelu(v, approximate=function.approximate)  # noqa: E731
    else:
        f = torch.relu
    # No slope of the functions passes 1.13 (SiLU and GELU overshoot 1 slightly); expf, erff and tanhf are
    # off by a few units in the last place of values near 1: 2^-20 of the magnitudes.
    slope = 1.13 * max(1.0, getattr(function, "alpha", 1.0))
    if activation.gate is None:
        expected, allowed = f(value), slope * bound + (value.abs() + 1) * 2.0**-20
    else:
        limit = activation.gate.limit
        gate, up = value[:, 0::2], value[:, 1::2]
        if limit is not None:
            gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
        up = up + activation.gate.up_offset
        expected = f(gate) * up
        allowed = slope * bound[:, 0::2] * (up.abs() + bound[:, 1::2]) + (f(gate).abs() + bound[:, 0::2]) * bound[:, 1::2] \
            + (gate.abs() + 1) * (up.abs() + 1) * 2.0**-20
    assert_within(out, expected, allowed, case.dtype, "activated")


@pytest.mark.parametrize("rows", [9, 140])
def test_in_place_base_absent_base_and_strided_rows(device, rows):
    case = Case(device, rows=rows, k=136, n=104, count=3, max_rank=12, seed=rows)
    expected = run(case)
    operator, weights, ids = case.operator(), case.weights(), case.ids.to(device)
    # In place.
    out = case.base.to(device)
    operator.run_into(case.x.to(device), weights, adapter_ids=ids, base=out, output=out)
    assert torch.equal(out, expected)
    # Rows of wider tensors, at odd element offsets; what lies between them stays.
    wide_x = torch.full((rows, case.k + 7), float("nan"), dtype=case.dtype, device=device)
    wide_base = torch.full((rows, case.n + 5), float("nan"), dtype=case.dtype, device=device)
    wide_out = torch.full((rows, case.n + 3), 7.0, dtype=case.dtype, device=device)
    wide_x[:, 3:3 + case.k] = case.x.to(device)
    wide_base[:, 1:1 + case.n] = case.base.to(device)
    operator.run_into(wide_x[:, 3:3 + case.k], weights, adapter_ids=ids, base=wide_base[:, 1:1 + case.n],
                      output=wide_out[:, 1:1 + case.n])
    assert torch.equal(wide_out[:, 1:1 + case.n], expected)
    assert bool((wide_out[:, 0] == 7).all()) and bool((wide_out[:, 1 + case.n:] == 7).all())
    # Without base.
    case.base.zero_()
    with_zero = run(case)
    out = torch.full_like(with_zero, float("nan"))
    operator.run_into(case.x.to(device), weights, adapter_ids=ids, base=None, output=out)
    assert torch.equal(out + 0.0, with_zero + 0.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("max_rank", [8, 16, 32, 100])
@pytest.mark.parametrize("rows", [60, 200])
def test_rows_do_not_depend_on_who_shares_their_adapter(device, rows, max_rank, dtype):
    """fp32 bits (bf16 ones of a sum that the store's rounding would hide are spread by a base of zero)."""

    outs = []
    for alone in (False, True):
        ids = [0 if i < 5 or not alone else 1 for i in range(rows)]
        case = Case(device, rows=rows, k=2100, n=136, count=2, max_rank=max_rank, dtype=dtype, ids=ids, seed=11)
        case.base.zero_()
        outs.append(run(case).cpu()[:5])
    assert torch.equal(outs[0], outs[1])


def test_rows_of_a_batch_do_not_depend_on_their_order(device):
    case = Case(device, rows=333, k=264, n=136, count=6, max_rank=16, seed=11)
    out = run(case)
    order = torch.randperm(333, generator=torch.Generator().manual_seed(3))
    case.x, case.base, case.ids = case.x[order], case.base[order], case.ids[order]
    assert torch.equal(run(case).cpu(), out.cpu()[order])


def test_smaller_batches_use_a_plan_for_more(device):
    case = Case(device, rows=700, k=1600, n=200, count=4, max_rank=8, seed=2)
    operator = case.operator(backward=True, capacity=700)
    for rows in (700, 449, 64, 3, 1):
        part = Case(device, rows=rows, k=1600, n=200, count=4, max_rank=8, seed=rows)
        check_forward(part, run(part, operator))
        check_backward(part, backward(part, operator))


# ------------------------------------------------------------------ gradients
def backward(case, operator=None, **kwargs):
    operator = operator or case.operator(backward=True)
    gx = torch.full((case.rows, case.k), float("nan"), dtype=case.dtype, device=case.device)
    ga = torch.full(case.a.shape, float("nan"), dtype=case.dtype, device=case.device)
    gb = torch.full(case.b.shape, float("nan"), dtype=case.dtype, device=case.device)
    operator.backward_into(case.x.to(case.device), case.grad.to(case.device), case.weights(),
                           adapter_ids=case.ids.to(case.device), base=case.grad_base.to(case.device), grad_inputs=gx,
                           grad_a=ga, grad_b=gb, **kwargs)
    return {"x": gx, "a": ga, "b": gb}


def check_backward(case, got):
    for name, (value, bound) in case.backward().items():
        assert_within(got[name], value, bound, case.dtype, f"gradient of {name}")
    for adapter in range(case.count):
        rank = case.rank(adapter)
        assert not bool(got["a"][adapter, rank:].any()) and not bool(got["b"][adapter, :, rank:].any())
        if not bool((case.ids == adapter).any()):
            assert not bool(got["a"][adapter].any()) and not bool(got["b"][adapter].any())


BACKWARD = [
    (1, 64, 48, 1, 8, None),
    (1, 1, 1, 1, 1, None),
    (3, 33, 7, 2, 3, [3, 1]),
    (40, 257, 131, 3, 33, [33, 0, 17]),
    (64, 320, 200, 5, 24, [24, 8, 16, 1, 24]),
    (65, 130, 70, 2, 128, [128, 64]),
    (257, 72, 200, 1, 16, None),
    (600, 130, 129, 2, 12, None),
    (1500, 264, 72, 3, 64, [64, 40, 16]),
    (2500, 24, 40, 300, 4, None),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k,n,count,max_rank,ranks", BACKWARD)
def test_gradients_match_the_formulas(device, rows, k, n, count, max_rank, ranks, dtype):
    case = Case(device, rows=rows, k=k, n=n, count=count, max_rank=max_rank, ranks=ranks, dtype=dtype, seed=rows + n)
    check_backward(case, backward(case))


def test_gradients_match_differences(device):
    """Central differences of a weighted sum of the outputs, fp32 payloads.

    The outputs are linear in x, in A and in B apart, so a difference of any width is exact but for the
    rounding of the sums: steps of 1 against sums of a few hundred terms of size 1 leave 1e-3.
    """

    case = Case(device, rows=70, k=40, n=30, count=2, max_rank=8, dtype="fp32", ids=[i % 2 for i in range(70)])
    case.grad_base.zero_()
    case.base.zero_()
    got = {name: value.cpu() for name, value in backward(case).items()}

    def loss():
        return float((run(case).cpu().double() * case.grad.double()).sum())

    for tensor, name, places in ((case.x, "x", [(0, 0), (33, 17)]), (case.a, "a", [(0, 3, 5), (1, 7, 39)]),
                                 (case.b, "b", [(0, 29, 0), (1, 11, 6)])):
        for place in places:
            kept = float(tensor[place])
            tensor[place] = kept + 1
            above = loss()
            tensor[place] = kept - 1
            below = loss()
            tensor[place] = kept
            assert abs((above - below) / 2 - float(got[name][place])) < 1e-3


def test_gradients_are_repeatable_and_parts_can_be_left_out(device):
    case = Case(device, rows=900, k=200, n=136, count=3, max_rank=16, seed=4)
    first, second = backward(case), backward(case)
    assert all(torch.equal(first[name], second[name]) for name in first)
    operator, weights, ids = case.operator(backward=True), case.weights(), case.ids.to(device)
    x, grad = case.x.to(device), case.grad.to(device)
    ga, gb = torch.empty_like(first["a"]), torch.empty_like(first["b"])
    operator.backward_into(x, grad, weights, adapter_ids=ids, grad_a=ga, grad_b=gb)
    assert torch.equal(ga, first["a"]) and torch.equal(gb, first["b"])
    gx = case.grad_base.to(device)
    operator.backward_into(x, grad, weights, adapter_ids=ids, base=gx, grad_inputs=gx)
    assert torch.equal(gx, first["x"])


def test_backward_of_no_rows_clears_the_gradients(device):
    case = Case(device, rows=0, k=64, n=48, count=2, max_rank=8)
    got = backward(case)
    assert not bool(got["a"].any()) and not bool(got["b"].any())
    run(case)


@pytest.mark.parametrize("wide", ["x", "base", "out", "grad", "grad_base", "grad_x"])
def test_rows_whose_offsets_pass_32_bits(device, wide):
    """2100 rows, 2^21 elements apart: 8.8 GB from the first row to the last."""

    case = Case(device, rows=2100, k=72, n=48, count=3, max_rank=8, seed=3)
    expected, gradients = run(case), backward(case)
    far = torch.empty((2100, 1 << 21), dtype=case.dtype, device=device)
    operands = {"x": case.x.to(device), "base": case.base.to(device), "grad": case.grad.to(device),
                "grad_base": case.grad_base.to(device), "out": torch.zeros_like(expected),
                "grad_x": torch.zeros_like(gradients["x"])}
    spread = far[:, -operands[wide].shape[1]:]
    spread.copy_(operands[wide])
    operands[wide] = spread
    operator, weights, ids = case.operator(backward=True), case.weights(), case.ids.to(device)
    operator.run_into(operands["x"], weights, adapter_ids=ids, base=operands["base"], output=operands["out"])
    assert torch.equal(operands["out"], expected)
    ga, gb = torch.empty_like(gradients["a"]), torch.empty_like(gradients["b"])
    operator.backward_into(operands["x"], operands["grad"], weights, adapter_ids=ids, base=operands["grad_base"],
                           grad_inputs=operands["grad_x"], grad_a=ga, grad_b=gb)
    assert torch.equal(operands["grad_x"], gradients["x"])
    assert torch.equal(ga, gradients["a"]) and torch.equal(gb, gradients["b"])


@pytest.mark.parametrize("k,n", [(20000, 64), (64, 20000)])
def test_pools_whose_offsets_pass_32_bits(device, k, n):
    """1024 adapters of 5 MB each, two of them in use at the end, against a pool of those two."""

    for rows in (40, 150):
        small = Case(device, rows=rows, k=k, n=n, count=2, max_rank=128, seed=rows)
        expected, gradients = run(small), backward(small)
        a = torch.zeros((1024, 128, k), dtype=small.dtype, device=device)
        b = torch.zeros((1024, n, 128), dtype=small.dtype, device=device)
        scales = torch.ones(1024, device=device)
        used = [1022, 1023]
        a[used], b[used], scales[used] = small.a.to(device), small.b.to(device), small.scales.to(device)
        plan = AdapterPlan.prepare(row_capacity=rows, adapter_count=1024, max_rank=128, input_width=k, output_width=n,
                                   dtype=small.dtype, backward=True)
        operator = Adapter(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
        weights = AdapterWeights(a, b, scales)
        ids = torch.where(small.ids >= 0, small.ids + 1022, -1).to(device)
        x, out = small.x.to(device), torch.empty_like(expected)
        operator.run_into(x, weights, adapter_ids=ids, base=small.base.to(device), output=out)
        assert torch.equal(out, expected)
        gx, ga, gb = torch.empty_like(x), torch.full_like(a, 1.0), torch.full_like(b, 1.0)
        operator.backward_into(x, small.grad.to(device), weights, adapter_ids=ids, base=small.grad_base.to(device),
                               grad_inputs=gx, grad_a=ga, grad_b=gb)
        assert torch.equal(gx, gradients["x"])
        assert torch.equal(ga[used], gradients["a"]) and torch.equal(gb[used], gradients["b"])
        assert not bool(ga[:1022].any()) and not bool(gb[:1022].any())


@pytest.mark.parametrize("rows", [9, 700])
def test_scales_of_unused_adapters_do_not_matter(device, rows):
    case = Case(device, rows=rows, k=72, n=40, count=4, max_rank=8, ids=[(i % 3 - 1) * 2 if i % 3 else 0 for i in range(rows)])
    case.ids[case.ids < 0] = -1
    unused = [adapter for adapter in range(4) if not bool((case.ids == adapter).any())]
    assert unused
    expected, gradients = run(case), backward(case)
    case.scales[unused] = float("inf")
    got = backward(case)
    assert torch.equal(run(case), expected)
    assert all(torch.equal(got[name], gradients[name]) for name in got)


def test_bad_ids_and_nan_rows_in_the_backward(device):
    case = Case(device, rows=100, k=64, n=72, count=3, max_rank=8, ids=[i % 3 for i in range(100)])
    case.ids[7] = 9
    fault = torch.zeros(1, dtype=torch.int32, device=device)
    got = backward(case, fault_word=fault)
    assert int(fault) == _native.XP_FAULT_ADAPTER_OUT_OF_RANGE
    assert bool(got["x"][7].isnan().all())
    for name in ("a", "b"):
        value, bound = case.backward()[name]
        assert_within(got[name], value, bound, case.dtype, name)
    # NaN in a row of adapter 1 reaches adapter 1's gradients only, and no row without an adapter matters.
    case.ids[7] = -1
    case.x[7], case.grad[7] = float("nan"), float("inf")
    clean = backward(case)
    assert not bool(clean["a"].isnan().any()) and not bool(clean["b"].isnan().any())
    case.x[4, 9] = float("nan")
    dirty = backward(case)
    assert torch.equal(dirty["a"][[0, 2]], clean["a"][[0, 2]]) and torch.equal(dirty["b"][[0, 2]], clean["b"][[0, 2]])
    assert bool(dirty["a"][1, :, 9].isnan().all()) and bool(dirty["b"][1].isnan().all())


# ------------------------------------------------------------------ graphs, streams
@pytest.mark.parametrize("rows", [30, 500])
def test_captured_calls_replay_over_new_rows_ids_and_weights(device, rows):
    case = Case(device, rows=rows, k=200, n=120, count=4, max_rank=16, seed=1)
    operator, weights = case.operator(backward=True), case.weights()
    ids, x, base = case.ids.to(device), case.x.to(device), case.base.to(device)
    grad, grad_base = case.grad.to(device), case.grad_base.to(device)
    out = torch.empty_like(base)
    got = {"x": torch.empty_like(x), "a": torch.empty_like(weights.a), "b": torch.empty_like(weights.b)}

    def both():
        operator.run_into(x, weights, adapter_ids=ids, base=base, output=out)
        operator.backward_into(x, grad, weights, adapter_ids=ids, base=grad_base, grad_inputs=got["x"],
                               grad_a=got["a"], grad_b=got["b"])

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for seed in (1, 2, 3):
        other = Case(device, rows=rows, k=200, n=120, count=4, max_rank=16, seed=seed)
        for target, source in ((ids, other.ids), (x, other.x), (base, other.base), (grad, other.grad),
                               (grad_base, other.grad_base), (weights.a, other.a), (weights.b, other.b),
                               (weights.scales, other.scales)):
            target.copy_(source)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check_forward(other, out)
        check_backward(other, got)
        eager = run(other)
        assert torch.equal(eager, out)


def test_two_streams_with_their_own_scratch(device):
    cases = [Case(device, rows=200, k=512, n=264, count=3, max_rank=16, seed=s) for s in (1, 2)]
    expected = [run(case) for case in cases]
    operators = [case.operator() for case in cases]
    inputs = [(c.x.to(device), c.weights(), c.ids.to(device), c.base.to(device)) for c in cases]
    outs = [torch.empty_like(e) for e in expected]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for stream, operator, (x, weights, ids, base), out in zip(streams, operators, inputs, outs):
            with torch.cuda.stream(stream):
                operator.run_into(x, weights, adapter_ids=ids, base=base, output=out)
    torch.cuda.synchronize()
    for out, want in zip(outs, expected):
        assert torch.equal(out, want)


def test_gate_and_up_adapters_of_one_interleaved_projection(device):
    g = torch.Generator().manual_seed(0)
    k, width = 96, 40
    gate_a, up_a = torch.randn((4, k), generator=g), torch.randn((6, k), generator=g)
    gate_b, up_b = torch.randn((width, 4), generator=g), torch.randn((width, 6), generator=g)
    a, b = interleave_gate_up_adapters(gate_a, gate_b, up_a, up_b)
    x = torch.randn((5, k), generator=g)
    expected = torch.stack((x @ gate_a.T @ gate_b.T, x @ up_a.T @ up_b.T), dim=2).flatten(1)
    weights = AdapterWeights(a[None].to(device), b[None].to(device))
    plan = AdapterPlan.prepare(row_capacity=5, adapter_count=1, max_rank=10, input_width=k, output_width=2 * width,
                               dtype=torch.float32)
    out = torch.empty((5, 2 * width), device=device)
    Adapter(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device)).run_into(
        x.to(device), weights, adapter_ids=torch.zeros(5, dtype=torch.int32, device=device), base=None, output=out)
    assert torch.allclose(out.cpu(), expected, rtol=1e-5, atol=1e-4)


def test_refusals_on_the_device(device):
    case = Case(device, rows=4, k=64, n=48, count=2, max_rank=8)
    operator, weights, ids = case.operator(), case.weights(), case.ids.to(device)
    x, base = case.x.to(device), case.base.to(device)
    out = torch.empty_like(base)
    good = dict(adapter_ids=ids, base=base, output=out)
    for bad in (
        dict(good, adapter_ids=ids.long()), dict(good, adapter_ids=ids[:3]), dict(good, adapter_ids=ids.cpu()),
        dict(good, base=base.float()), dict(good, base=base[:, :47]), dict(good, output=out[:3]),
        dict(good, output=out.t().contiguous().t()), dict(good, fault_word=torch.zeros(1, device=device)),
        dict(good, activation=Activation(SiluActivation(), GateTransform())),
    ):
        with pytest.raises(ValueError):
            operator.run_into(x, weights, **bad)
    with pytest.raises(ValueError, match="capacity"):
        operator.run_into(torch.cat((x, x)), weights, adapter_ids=torch.cat((ids, ids)), base=torch.cat((base, base)),
                          output=torch.cat((out, out)))
    with pytest.raises(ValueError, match="without backward"):
        operator.backward_into(x, base, weights, adapter_ids=ids, grad_inputs=torch.empty_like(x))
    with pytest.raises(ValueError, match="workspace"):
        Adapter(operator.plan, torch.empty(16, dtype=torch.uint8, device=device))
    with pytest.raises(ValueError):
        AdapterWeights(weights.a, weights.b[:, :, :4].contiguous())
    with pytest.raises(ValueError):
        AdapterWeights(weights.a, weights.b, ranks=torch.ones(2, device=device))
    # The output over the input, or over part of its base: refused by the library before any launch.
    square = Case(device, rows=4, k=48, n=48, count=2, max_rank=8)
    xs = square.x.to(device)
    with pytest.raises(_native.NativeError, match="overlap"):
        square.operator().run_into(xs, square.weights(), adapter_ids=square.ids.to(device), base=None, output=xs)
    both = torch.zeros((5, 48), dtype=torch.bfloat16, device=device)
    with pytest.raises(_native.NativeError, match="base"):
        square.operator().run_into(xs, square.weights(), adapter_ids=square.ids.to(device), base=both[:4], output=both[1:])


def powers(shape, g, dtype):
    """Signed powers of two: exact in bf16, so that every rest of a two-term split is zero."""

    return (torch.randint(0, 2, shape, generator=g) * 2.0 - 1.0).mul(2.0 ** torch.randint(-2, 3, shape, generator=g)).to(dtype)


def assert_same_kinds(actual, value, what):
    """Infinities with their signs and NaN exactly where the definition has them."""

    actual = actual.cpu().double()
    assert torch.equal(actual.isnan(), value.isnan()), f"{what}: NaN at {(actual.isnan() != value.isnan()).nonzero()[:4].tolist()}"
    for sign in (1, -1):
        assert torch.equal(actual == sign * float("inf"), value == sign * float("inf")), what


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [5, 90])
@pytest.mark.parametrize("where", ["x", "a", "b", "grad", "x_and_b"])
@pytest.mark.parametrize("exact", [True, False], ids=["powers_of_two", "random"])
def test_infinities_are_those_of_the_definition(device, exact, where, rows, dtype):
    """An infinite factor times a finite one is infinite, whatever terms the finite one is split into."""

    g = torch.Generator().manual_seed(rows)
    case = Case(device, rows=rows, k=70, n=146, count=2, max_rank=12, ranks=[12, 1], dtype=dtype,
                ids=[i % 3 - 1 for i in range(rows)])
    if exact:
        case.a, case.b = powers(case.a.shape, g, case.dtype), powers(case.b.shape, g, case.dtype)
        case.x, case.grad = powers(case.x.shape, g, case.dtype), powers(case.grad.shape, g, case.dtype)
    infinity = float("inf")
    if where in ("x", "x_and_b"):
        case.x[2, 33], case.x[4, 69] = infinity, -infinity
    if where in ("b", "x_and_b"):
        case.b[1, 7, 0], case.b[1, 145, 0], case.b[0, 100, 3] = infinity, -infinity, infinity
    if where == "a":
        case.a[1, 0, 9], case.a[0, 3, 69] = -infinity, infinity
    if where == "grad":
        case.grad[2, 5], case.grad[4, 140] = infinity, -infinity
    value, _ = case.forward()
    assert_same_kinds(run(case), value, "output")
    got = backward(case)
    for name, (value, _) in case.backward().items():
        assert_same_kinds(got[name], value, f"gradient of {name}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [6, 100])
@pytest.mark.parametrize("function", [SiluActivation(), GeluActivation(), ReluActivation()], ids=["silu", "gelu", "relu"])
def test_no_limit_hides_a_nan_of_the_sum(device, function, rows, dtype):
    """NaN in a row, in a base's Gate or in its Up: neither is below a limit nor above one."""

    case = Case(device, rows=rows, k=64, n=542, count=3, max_rank=8, dtype=dtype, ids=[i % 4 - 1 for i in range(rows)])
    activation = Activation(function, GateTransform(1.5, 1.0))
    outs = []
    for bad in (False, True):
        if bad:
            case.x[1, 5] = float("nan")
            case.base[2, 40], case.base[3, 41] = float("nan"), float("nan")   # Gate and Up of column 20
            case.base[2, 540], case.base[3, 541] = float("nan"), float("nan")  # of the last column, past whole chunks
            case.base[0, 100], case.base[0, 103] = float("inf"), -float("inf")  # clipped
        out = torch.zeros((rows, 271), dtype=case.dtype, device=device)
        case.operator().run_into(case.x.to(device), case.weights(), adapter_ids=case.ids.to(device),
                                 base=case.base.to(device), output=out, activation=activation)
        outs.append(out.cpu())
    clean, got = outs
    assert bool(got[1].isnan().all())
    expected = torch.zeros_like(got, dtype=torch.bool)
    expected[1] = True
    expected[2:4, [20, 270]] = True
    assert torch.equal(got.isnan(), expected)
    assert bool(got[0].isfinite().all())
    keep = torch.ones_like(expected)
    keep[:4] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("count", [3, 70])
def test_no_rows_with_the_scratch_asked_for_them(device, count):
    case = Case(device, rows=0, k=300, n=520, count=count, max_rank=12)
    nbytes = _native.library().xp_adapter_workspace_bytes(0, count, 12, 300, 520, _native.XP_DTYPE_BF16, 1)
    scratch = torch.full((nbytes + 64,), 0xFF, dtype=torch.uint8, device=device)
    weights = case.weights()
    ga, gb = torch.full_like(weights.a, float("nan")), torch.full_like(weights.b, float("nan"))
    _native.call("xp_adapter_backward", ctypes.byref(weights.descriptor), None, 0, None, 0, None, 0, None, 0, None, 0,
                 ga.data_ptr(), gb.data_ptr(), scratch.data_ptr(), nbytes, None, torch.cuda.current_stream().cuda_stream)
    assert not bool(ga.any()) and not bool(gb.any())
    assert bool((scratch[nbytes:] == 0xFF).all())


def test_a_pool_keeps_the_tensors_that_it_was_made_of(device):
    case = Case(device, rows=4, k=64, n=48, count=2, max_rank=8, ranks=[8, 4])
    weights = case.weights()
    for name in ("a", "b", "scales", "ranks", "descriptor"):
        with pytest.raises(AttributeError):
            setattr(weights, name, getattr(weights, name))
    operator, ids = case.operator(backward=True), case.ids.to(device)
    x, base = case.x.to(device), case.base.to(device)
    out, gx = torch.empty_like(base), torch.empty_like(x)
    # Storage that moved under a tensor (as a module's conversion moves its parameters).
    for name in ("a", "b", "scales", "ranks"):
        moved = case.weights()
        tensor = getattr(moved, name)
        kept = tensor.data
        tensor.data = kept.clone()
        with pytest.raises(ValueError, match="pool"):
            operator.run_into(x, moved, adapter_ids=ids, base=base, output=out)
        with pytest.raises(ValueError, match="pool"):
            operator.backward_into(x, base, moved, adapter_ids=ids, grad_inputs=gx)
        tensor.data = kept
        operator.run_into(x, moved, adapter_ids=ids, base=base, output=out)
    moved = case.weights()
    moved.b.data = moved.b.data[:, :, :4]
    with pytest.raises(ValueError, match="pool|plan"):
        operator.run_into(x, moved, adapter_ids=ids, base=base, output=out)
    check_forward(case, run(case))


@pytest.mark.parametrize("rows", [5, 200])
def test_operands_in_columns_of_one_tensor(device, rows):
    """Rows of several operands side by side in one buffer share no byte."""

    case = Case(device, rows=rows, k=72, n=104, count=3, max_rank=8, seed=rows)
    expected, gradients = run(case), backward(case)
    wide = torch.zeros((rows, 600), dtype=case.dtype, device=device)
    places = {"x": (0, 72), "base": (72, 176), "out": (176, 280), "grad": (281, 385), "grad_base": (385, 457),
              "grad_x": (457, 529)}
    views = {name: wide[:, begin:end] for name, (begin, end) in places.items()}
    for name, source in (("x", case.x), ("base", case.base), ("grad", case.grad), ("grad_base", case.grad_base)):
        views[name].copy_(source)
    operator, weights, ids = case.operator(backward=True), case.weights(), case.ids.to(device)
    operator.run_into(views["x"], weights, adapter_ids=ids, base=views["base"], output=views["out"])
    assert torch.equal(views["out"], expected)
    ga, gb = torch.empty_like(gradients["a"]), torch.empty_like(gradients["b"])
    operator.backward_into(views["x"], views["grad"], weights, adapter_ids=ids, base=views["grad_base"],
                           grad_inputs=views["grad_x"], grad_a=ga, grad_b=gb)
    assert torch.equal(views["grad_x"], gradients["x"])
    assert torch.equal(ga, gradients["a"]) and torch.equal(gb, gradients["b"])
    assert not bool(wide[:, 280].any()) and not bool(wide[:, 529:].any())
    for name, source in (("x", case.x), ("base", case.base), ("grad", case.grad), ("grad_base", case.grad_base)):
        assert torch.equal(views[name].cpu(), source)
    # One column in common, or rows of one operand among those of another.
    with pytest.raises(_native.NativeError, match="overlap"):
        operator.run_into(views["x"], weights, adapter_ids=ids, base=None, output=wide[:, 71:175])
    tall = torch.zeros((2 * rows, 104), dtype=case.dtype, device=device)
    operator.run_into(tall[0::2, :72], weights, adapter_ids=ids, base=None, output=tall[1::2])
    with pytest.raises(_native.NativeError, match="overlap"):
        operator.run_into(tall[0::2, :72], weights, adapter_ids=ids, base=None, output=tall[:rows])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,count,used", [
    (1, 33, [32]), (2, 1024, [5, 1023]), (40, 33, [0, 3, 31, 32]), (64, 200, list(range(64, 128))), (70, 40, [39]),
    (500, 100, [7, 8, 50, 99, -1]), (500, 32, [7, 31, -1]), (8193, 40, [1, 38, -1]), (8193, 32, [1, 30, -1]),
])
def test_backward_of_large_pools_stays_in_its_scratch(device, rows, count, used, dtype):
    """Few of a pool's adapters in use, in scratch of the size asked for and no larger."""

    case = Case(device, rows=rows, k=136, n=72, count=count, max_rank=12, dtype=dtype,
                ids=[used[i * 7 % len(used)] for i in range(rows)], seed=rows + count)
    plan = case.operator(backward=True).plan
    nbytes = plan.workspace.nbytes
    assert nbytes - 256 <= _native.library().xp_adapter_workspace_bytes(
        rows, count, 12, 136, 72, {"bf16": _native.XP_DTYPE_BF16, "fp32": _native.XP_DTYPE_F32}[dtype], 1) <= nbytes
    scratch = torch.full((nbytes + (1 << 20),), 0xFF, dtype=torch.uint8, device=device)
    check_backward(case, backward(case, Adapter(plan, scratch[:nbytes])))
    assert bool((scratch[nbytes:] == 0xFF).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [64, 128])
def test_rows_without_an_adapter_keep_every_bit_of_any_value(device, rows, dtype):
    """All 65536 patterns: zeros of both signs, subnormals and infinities as they are, NaN as some NaN."""

    case = Case(device, rows=rows, k=16, n=65536 // rows, count=2, max_rank=4, dtype=dtype, ids=[-1] * rows)
    case.base = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(case.dtype).reshape(rows, -1)
    case.a.fill_(float("nan"))
    got = run(case).cpu()
    assert torch.equal(got.isnan(), case.base.isnan())
    keep = ~case.base.isnan()
    assert torch.equal(got.view(torch.int16)[keep], case.base.view(torch.int16)[keep])


def test_an_operators_scratch_stays_its_own(device):
    case = Case(device, rows=70, k=64, n=48, count=2, max_rank=8)
    operator = case.operator()
    for name in ("scratch", "plan"):
        with pytest.raises(AttributeError):
            setattr(operator, name, getattr(case.operator(), name))
    check_forward(case, run(case, operator))


@pytest.mark.parametrize("k,n", [(20000, 64), (64, 20000)])
def test_transposes_whose_offsets_pass_32_bits(device, k, n):
    """1024 adapters with rows, the last two's weights alone not zero: their transposes lie past 5 GB."""

    rows, used = 1100, [1022, 1023]
    small = Case(device, rows=rows, k=k, n=n, count=2, max_rank=128, ids=[i % 3 - 1 if i < 60 else -1 for i in range(rows)])
    gradients = backward(small)
    a = torch.zeros((1024, 128, k), dtype=small.dtype, device=device)
    b = torch.zeros((1024, n, 128), dtype=small.dtype, device=device)
    scales = torch.ones(1024, device=device)
    a[used], b[used], scales[used] = small.a.to(device), small.b.to(device), small.scales.to(device)
    ids = torch.where(small.ids >= 0, small.ids + 1022, -1)
    ids[60:60 + 1022] = torch.arange(1022, dtype=torch.int32)
    plan = AdapterPlan.prepare(row_capacity=rows, adapter_count=1024, max_rank=128, input_width=k, output_width=n,
                               dtype=small.dtype, backward=True)
    operator = Adapter(plan, torch.empty(plan.workspace.nbytes, dtype=torch.uint8, device=device))
    x, gx, ga, gb = small.x.to(device), torch.empty_like(gradients["x"]), torch.full_like(a, 1.0), torch.full_like(b, 1.0)
    operator.backward_into(x, small.grad.to(device), AdapterWeights(a, b, scales), adapter_ids=ids.to(device),
                           base=small.grad_base.to(device), grad_inputs=gx, grad_a=ga, grad_b=gb)
    assert torch.equal(gx, gradients["x"])
    assert torch.equal(ga[used], gradients["a"]) and torch.equal(gb[used], gradients["b"])
    assert not bool(ga[:1022].any()) and not bool(gb[:1022].any())
