"""Orthogonal updates of weight matrices by Newton-Schulz products, alone or inside an optimiser's step.

A matrix ``G = U S V^T`` becomes nearly ``U V^T``:

    ``X = G / (|G| + eps)``, then ``steps`` times ``X = a X + (b A + c A A) X`` with ``A = X X^T``

``a, b, c = 3.4445, -4.7750, 2.0315``, on the short side of the matrix.  One call serves a batch of matrices: the
experts of a layer, or Gate and Up of an INTERLEAVED i_proj as a view (:func:`gate_up_matrices`).  The reference has no
counterpart; plans and caller-owned workspaces follow the projections' (operators/linear.py:28-257).

bf16 and fp16 matrices run on fp16 products with fp32 sums (a result carries about 2^-9.7 of itself, which bf16 rounds to
2^-9; in fp16 that is less than the type holds), fp32 ones on fp32 products.  An update whose norm is a thousandth of ``eps``
or less, whose result is small too, loses digits in the 16-bit types and goes to zero.  Every launch goes to the HIP
library on the current torch stream and allocates nothing, so a call can be captured into a graph.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from crosspool_amd import _native
from crosspool_amd.execution import WorkspaceLayout
from crosspool_amd.operators import _DTYPE_CODES

__all__ = ["Muon", "MuonPlan", "gate_up_matrices"]


def gate_up_matrices(values: torch.Tensor) -> torch.Tensor:
    """Gate and Up of an INTERLEAVED i_proj ``[2 I, K]`` as a view ``[2, I, K]``: two matrices of one batch."""

    if values.ndim != 2 or values.shape[0] % 2:
        raise ValueError("an INTERLEAVED i_proj has an even number of rows")
    return values.unflatten(0, (-1, 2)).transpose(0, 1)


@dataclass(frozen=True, slots=True)
class MuonPlan:
    """Address-free geometry and scratch of a batch of ``matrices`` updates ``[rows, columns]``."""

    matrices: int
    rows: int
    columns: int
    dtype: torch.dtype
    workspace: WorkspaceLayout

    @classmethod
    def prepare(cls, *, rows: int, columns: int, dtype: torch.dtype, matrices: int = 1) -> MuonPlan:
        """``dtype`` is that of the updates or gradients (bf16, fp16 or fp32)."""

        if dtype not in _DTYPE_CODES:
            raise ValueError("orthogonal updates are bf16, fp16 or fp32")
        nbytes = int(_native.library().xp_muon_workspace_bytes(matrices, rows, columns, _DTYPE_CODES[dtype]))
        if nbytes == 0:
            raise ValueError(
                "orthogonal updates take 1 to 4096 matrices with a short side of 1 to 65536 and a long side of at most 1048576, "
                "2^36 values in all"
            )
        return cls(matrices, rows, columns, dtype, WorkspaceLayout.from_regions(((torch.uint8, (nbytes,)),)))


class Muon:
    """Orthogonal updates borrowing their plan and scratch.

    Operands are ``[matrices, rows, columns]`` (or ``[rows, columns]`` of a plan for one matrix); columns are contiguous,
    and rows and matrices may lie any stride apart that keeps their rows apart.  Calls on one ``Muon`` share its
    scratch: order them on one stream, or give each stream its own.
    """

    def __init__(self, plan: MuonPlan, workspace: torch.Tensor) -> None:
        if workspace.device.type != "cuda":
            raise ValueError("the scratch of orthogonal updates must reside on its execution device")
        (self._workspace,) = plan.workspace.views(workspace)
        self._plan = plan
        self._index = workspace.device.index

    @property
    def plan(self) -> MuonPlan:
        return self._plan

    @property
    def scratch(self) -> torch.Tensor:
        return self._workspace

    def _matrices(self, tensor: torch.Tensor, name: str, dtypes: tuple[torch.dtype, ...]) -> _native.Matrices:
        plan = self._plan
        shape = (plan.matrices, plan.rows, plan.columns)
        if tensor.ndim == 2 and plan.matrices == 1:
            tensor = tensor.unsqueeze(0)
        if tensor.shape != shape or tensor.dtype not in dtypes or tensor.get_device() != self._index:
            raise ValueError(f"{name} must be a tensor of shape {shape} on cuda:{self._index}, {' or '.join(map(str, dtypes))}")
        matrix, row, column = tensor.stride()
        if column != 1 and plan.columns > 1:
            raise ValueError(f"{name} must have contiguous rows")
        if plan.rows == 1:
            row = plan.columns
        return _native.Matrices(tensor.data_ptr(), matrix if plan.matrices > 1 else plan.rows * row, row)

    def _ready(self) -> None:
        if _native.current_device() != self._index:
            raise ValueError(f"orthogonal updates on cuda:{self._index} need it as the current device")

    def orthogonalize_into(self, updates: torch.Tensor, *, output: torch.Tensor, steps: int = 5, eps: float = 1e-7) -> None:
        """Write the orthogonalised ``updates`` to ``output``, which may be ``updates`` itself.

        A zero matrix stays zero; one with an infinity or NaN becomes NaN.
        """

        plan = self._plan
        source = self._matrices(updates, "updates", (plan.dtype,))
        target = self._matrices(output, "output", (plan.dtype,))
        self._ready()
        _native.call(
            "xp_muon_orthogonalize", ctypes.byref(source), plan.matrices, plan.rows, plan.columns, _DTYPE_CODES[plan.dtype],
            steps, eps, ctypes.byref(target), self._workspace.data_ptr(), self._workspace.numel(),
            _native.current_stream(self._index),
        )

    def step_into(
        self,
        *,
        weights: torch.Tensor,
        gradients: torch.Tensor,
        momentum: torch.Tensor,
        learning_rate: float,
        new_weights: torch.Tensor | None = None,
        new_momentum: torch.Tensor | None = None,
        weight_decay: float = 0.0,
        momentum_factor: float = 0.95,
        nesterov: bool = True,
        update_scale: float | None = None,
        steps: int = 5,
        eps: float = 1e-7,
    ) -> None:
        """One step of the optimiser, in place unless ``new_weights`` or ``new_momentum`` are given.

        ``momentum = momentum_factor * momentum + gradients`` (fp32); the update is ``gradients + momentum_factor *
        momentum`` (``nesterov``) or the momentum, orthogonalised; ``weights = (1 - learning_rate * weight_decay) *
        weights - learning_rate * update_scale * update`` in fp32, rounded once.  ``weights`` are of the gradients' dtype
        or fp32; ``update_scale`` is ``sqrt(max(1, rows / columns))`` unless given.
        """

        plan = self._plan
        kinds = (plan.dtype, torch.float32)
        new_weights = weights if new_weights is None else new_weights
        new_momentum = momentum if new_momentum is None else new_momentum
        if new_weights.dtype is not weights.dtype:
            raise ValueError("new weights must be of the weights' dtype")
        if update_scale is None:
            update_scale = math.sqrt(max(1.0, plan.rows / plan.columns))
        operands = [
            ctypes.byref(self._matrices(tensor, name, allowed)) for tensor, name, allowed in (
                (weights, "weights", kinds), (gradients, "gradients", (plan.dtype,)), (momentum, "momentum", (torch.float32,)),
                (new_weights, "new weights", kinds), (new_momentum, "new momentum", (torch.float32,)),
            )
        ]
        self._ready()
        _native.call(
            "xp_muon_step", *operands, plan.matrices, plan.rows, plan.columns, _DTYPE_CODES[plan.dtype],
            _DTYPE_CODES[weights.dtype], steps, eps, learning_rate, weight_decay, momentum_factor, int(nesterov), update_scale,
            self._workspace.data_ptr(), self._workspace.numel(), _native.current_stream(self._index),
        )
