"""Orthogonal updates on the GPU, against the formula in 64 bits.

Tolerances, derived before the first run.  Every rounding to fp16 is off by half a step, 2^-12, of a value, and errors of
many values are independent, so a stored matrix is off by less than 2^-12 of its 2-norm.  A step stores three: X, A and
b A + c A A.  X's relative error goes on as it is (|f(x)| >= 0.7 |x| and |f'| <= a over (0, 1.2]: growth by at most a / 0.7 in
the worst direction, near 1 over the spectrum, whose values all grow alike while they are small); A's reaches X'
times |b + 2 c x^2| x^2 <= 4.8 against f(x) / x >= 0.7, b A + c A A's times 4.8 as well.  Five steps of (1 + 4.8 + 4.8)
2^-12 / 0.7 would be 2^-6 if all added up; independent errors add as squares: sqrt(5) * sqrt(1 + 2 * 4.8^2) * 2^-12 / 0.7 =
2^-7.6.  The checks allow 2^-7.6 plus the result's own half step for 16-bit payloads.  fp32: the same with 2^-24 and sums
of n terms, whose errors grow like sqrt(n): 2^-7.6+12-24 = 2^-19.6 sqrt(n).
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
        error = float((found - wanted).norm() / wanted.norm())
        assert error <= allowed, f"{what} {i}: relative error {error:.2e} above {allowed:.2e}"


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
