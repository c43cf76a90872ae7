"""Orthogonal updates at the ends of their ranges on the GPU.  Tolerances are those of test_gpu_muon, whose operator and
64-bit formula these tests use."""

from __future__ import annotations

import pytest
import torch

from test_gpu_muon import A, B, C, muon, near, orthogonal, tolerance, updates

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rank_one(source, eps=1e-7, steps=5):
    """The update of matrices of one row or column in 64 bits: their only singular value runs through the polynomial."""

    x = source.double()
    norm = x.flatten(1).norm(dim=1)[:, None, None]
    value = norm / (norm + eps)
    for _ in range(steps):
        value = A * value + B * value**3 + C * value**5
    return x / norm * value


def parts(count, size=64):
    return [slice(first, min(first + size, count)) for first in range(0, count, size)]


@pytest.mark.parametrize("count,rows,columns", [(512, 1, 1 << 20), (600, 1 << 20, 1), (4096, 1, 1 << 20)])
def test_more_tiles_than_a_launch_holds(device, count, rows, columns):
    """Products of 2^24 tiles and more: other tiles, or several launches, each matrix as it is alone."""

    g = torch.Generator(device=device).manual_seed(count)
    source = torch.randn((count, rows, columns), generator=g, device=device, dtype=BF16)
    out = torch.full_like(source, float("nan"))
    muon(device, count, rows, columns, BF16).orthogonalize_into(source, output=out)
    for part in parts(count):
        near(out[part], rank_one(source[part]), tolerance(BF16, max(rows, columns)), "matrix")


def test_step_of_more_tiles_than_a_launch_holds(device):
    """A step that several launches share writes the momentum and every matrix's weights once."""

    count, columns = 4096, 1 << 18
    g = torch.Generator(device=device).manual_seed(9)
    gradients = torch.randn((count, 1, columns), generator=g, device=device, dtype=BF16)
    weights = torch.randn((count, 1, columns), generator=g, device=device, dtype=BF16)
    momentum = torch.randn((count, 1, columns), generator=g, device=device)
    held = weights.clone(), momentum.clone()
    muon(device, count, 1, columns, BF16).step_into(weights=weights, gradients=gradients, momentum=momentum, learning_rate=0.5,
                                                    weight_decay=0.1, momentum_factor=0.9)
    for part in parts(count):
        wanted = 0.9 * held[1][part].double() + gradients[part].double()
        size = 0.9 * held[1][part].double().abs() + gradients[part].double().abs()
        assert bool(((momentum[part].double() - wanted).abs() <= 2.0**-23 * size).all())
        update = rank_one(gradients[part].double() + 0.9 * wanted)
        moved = (1 - 0.5 * 0.1) * held[0][part].double() - 0.5 * update
        for found, target, step in zip(weights[part].double(), moved, update):
            allowed = 0.5 * 2.0**-7.6 * float(step.norm()) + (2.0**-9 + 2.0**-22) * 2 * float(target.norm())
            assert float((found - target).norm()) <= allowed


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("eps", [1.2e-38, 1e-41, 1.4e-45])
def test_zero_matrix_with_a_tiny_eps(device, dtype, eps):
    """The reciprocal of a tiny eps is past fp32: a zero matrix stays zero beside one that is not."""

    source = updates(device, 3, 72, 136, dtype)
    source[1] = 0
    out = torch.full_like(source, float("nan"))
    muon(device, 3, 72, 136, dtype).orthogonalize_into(source, output=out, eps=eps)
    assert bool((out[1] == 0).all())
    near(out[0::2], orthogonal(source[0::2], eps=0.0), tolerance(dtype, 136), "matrix beside a zero one")


@pytest.mark.parametrize("dtype,std", [(BF16, 2.0**-128), (FP32, 2.0**-130), (FP32, 2.0**125), (BF16, 2.0**124)])
@pytest.mark.parametrize("rows,columns", [(1, 9), (72, 136), (1030, 1024)])
def test_norms_at_the_ends_of_the_range(device, rows, columns, dtype, std):
    """Values down to subnormal ones and up to the largest, whose norm or its reciprocal fp32 does not hold."""

    g = torch.Generator(device=device).manual_seed(rows)
    source = ((torch.randn((2, rows, columns), generator=g, device=device).clamp(-3.5, 3.5)).double() * std).to(dtype)
    assert bool(source.isfinite().all())
    eps = 2.0**-149  # fp32's smallest value
    out = torch.full_like(source, float("nan"))
    muon(device, 2, rows, columns, dtype).orthogonalize_into(source, output=out, eps=eps)
    near(out, orthogonal(source, eps=eps), tolerance(dtype, max(rows, columns)), "matrix")
