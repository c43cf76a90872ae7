"""Low-rank adapters of many requests beside a shared projection, and their gradients.

Every token row carries the index of its request's adapter in a pool on the device (-1: none):

    ``output[i] = act(base[i] + scales[a] * (inputs[i] @ A[a].T) @ B[a].T)``,  ``a = adapter_ids[i]``

``base`` being the shared projection's result (:class:`crosspool_amd.operators.Gemm`).  One call serves
a batch of any mix of adapters, ranks and rows, from one decoding request to a prefill of thousands.
:meth:`Adapter.backward_into` gives the gradients for fine-tuning.  The reference has no counterpart;
plans, caller-owned workspaces and ``run_into`` follow the projections' (operators/linear.py:28-257).

Every launch goes to the HIP library on the current torch stream and allocates nothing, so a call can
be captured into a graph; replays read the ids, weights and rows that the tensors hold then.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import torch

from crosspool_amd import _native
from crosspool_amd.execution import WorkspaceLayout
from crosspool_amd.operators import _DTYPE_CODES, Activation

MAX_RANK = 128
MAX_ADAPTERS = 1024

__all__ = ["Adapter", "AdapterPlan", "AdapterWeights", "DenseAdapterWeights", "interleave_gate_up_adapters"]


def _require_pool(tensor: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple[int, ...], device: torch.device) -> None:
    if tensor.device != device or tensor.dtype is not dtype or tuple(tensor.shape) != shape or not tensor.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {device}")


@dataclass(frozen=True, slots=True, eq=False)
class AdapterWeights:
    """A pool of adapters of one projection: ``a`` ``[adapters, max_rank, K]``, ``b`` ``[adapters, N, max_rank]``.

    ``scales`` (fp32, default 1) holds every adapter's factor and ``ranks`` (int32, default
    ``max_rank``) its rank: what ``a`` and ``b`` hold past it is ignored, and a rank of 0 is an empty
    slot.  The tensors are borrowed; a slot may be rewritten in place between calls, but a tensor whose
    storage is exchanged needs a pool of its own.
    """

    a: torch.Tensor
    b: torch.Tensor
    scales: torch.Tensor | None = None
    ranks: torch.Tensor | None = None
    descriptor: _native.AdapterPool = field(init=False, repr=False)

    def __post_init__(self) -> None:
        a, b = self.a, self.b
        if a.device.type != "cuda":
            raise ValueError("adapter weights must be GPU-resident")
        if a.dtype not in _DTYPE_CODES or a.ndim != 3 or b.ndim != 3 or not a.is_contiguous():
            raise ValueError("adapter weights must be contiguous bf16, fp16 or fp32 tensors [adapters, R, K] and [adapters, N, R]")
        count, max_rank, input_width = a.shape
        if not 1 <= count <= MAX_ADAPTERS or not 1 <= max_rank <= MAX_RANK or input_width < 1 or b.shape[1] < 1:
            raise ValueError(f"an adapter pool holds 1 to {MAX_ADAPTERS} adapters of 1 to {MAX_RANK} ranks and positive widths")
        _require_pool(b, "adapter b", a.dtype, (count, b.shape[1], max_rank), a.device)
        if self.scales is not None:
            _require_pool(self.scales, "adapter scales", torch.float32, (count,), a.device)
        if self.ranks is not None:
            _require_pool(self.ranks, "adapter ranks", torch.int32, (count,), a.device)
        object.__setattr__(self, "descriptor", _native.AdapterPool(
            a=a.data_ptr(), b=b.data_ptr(), ranks=None if self.ranks is None else self.ranks.data_ptr(),
            scales=None if self.scales is None else self.scales.data_ptr(), count=count, max_rank=max_rank,
            input_width=input_width, output_width=b.shape[1], dtype=_DTYPE_CODES[a.dtype],
        ))

    def keeps_storage(self) -> bool:
        """Whether the tensors still are where the pool was made (``.data`` can be exchanged under them)."""

        pool = self.descriptor
        return (
            self.a.data_ptr() == pool.a and self.b.data_ptr() == pool.b
            and (self.scales is None or self.scales.data_ptr() == pool.scales)
            and (self.ranks is None or self.ranks.data_ptr() == pool.ranks)
        )


@dataclass(frozen=True, slots=True)
class DenseAdapterWeights:
    """Adapter pools of a Dense layer's projections (``operators.Dense.run_into``), either left out."""

    i_proj: AdapterWeights | None = None
    o_proj: AdapterWeights | None = None


def interleave_gate_up_adapters(
    gate_a: torch.Tensor, gate_b: torch.Tensor, up_a: torch.Tensor, up_b: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor]:
    """One adapter of an INTERLEAVED i_proj from separate adapters of its Gate and its Up projection.

    ``gate_a`` ``[r, K]``, ``gate_b`` ``[I, r]`` and the same of Up (of any rank) become ``a``
    ``[r + r', K]`` and ``b`` ``[2 I, r + r']``: row 2j of ``b`` is Gate's row j over the first ranks,
    row 2j + 1 Up's over the others (``interleave_gate_up`` of the weights).
    """

    if gate_b.shape[0] != up_b.shape[0] or gate_a.shape[1] != up_a.shape[1]:
        raise ValueError("gate and up adapters must share their widths")
    if gate_a.shape[0] != gate_b.shape[1] or up_a.shape[0] != up_b.shape[1]:
        raise ValueError("an adapter's a and b must share their rank")
    gate = torch.cat((gate_b, torch.zeros_like(up_b)), dim=1)
    up = torch.cat((torch.zeros_like(gate_b), up_b), dim=1)
    return torch.cat((gate_a, up_a), dim=0).contiguous(), torch.stack((gate, up), dim=1).flatten(0, 1).contiguous()


@dataclass(frozen=True, slots=True)
class AdapterPlan:
    """Address-free geometry and scratch of a projection's adapters for up to ``row_capacity`` rows."""

    row_capacity: int
    adapter_count: int
    max_rank: int
    input_width: int
    output_width: int
    dtype: torch.dtype
    backward: bool
    workspace: WorkspaceLayout

    @classmethod
    def prepare(
        cls,
        *,
        row_capacity: int,
        adapter_count: int,
        max_rank: int,
        input_width: int,
        output_width: int,
        dtype: torch.dtype,
        backward: bool = False,
    ) -> AdapterPlan:
        """``backward``: the scratch of ``backward_into`` too (transposed weights and gradient sums)."""

        if dtype not in _DTYPE_CODES:
            raise ValueError("adapter payloads are bf16, fp16 or fp32")
        if row_capacity < 1:
            raise ValueError("an adapter plan serves at least one row")
        query = _native.library().xp_adapter_workspace_bytes
        sizes = (row_capacity, adapter_count, max_rank, input_width, output_width, _DTYPE_CODES[dtype])
        nbytes = int(query(*sizes, 0))
        if nbytes == 0:
            raise ValueError(
                f"an adapter pool holds 1 to {MAX_ADAPTERS} adapters of 1 to {MAX_RANK} ranks and positive widths"
            )
        if backward:
            nbytes = max(nbytes, int(query(*sizes, 1)))
        return cls(row_capacity, adapter_count, max_rank, input_width, output_width, dtype, backward,
                   WorkspaceLayout.from_regions(((torch.uint8, (nbytes,)),)))


class Adapter:
    """A projection's adapters borrowing their plan and scratch.

    Rows are 2-D tensors whose columns are contiguous; their rows may lie any stride apart.  Calls on
    one ``Adapter`` share its scratch: order them on one stream, or give each stream its own.
    """

    def __init__(self, plan: AdapterPlan, workspace: torch.Tensor) -> None:
        if workspace.device.type != "cuda":
            raise ValueError("adapter scratch must reside on its execution device")
        (self._workspace,) = plan.workspace.views(workspace)
        self._plan = plan
        self._device = workspace.device
        self._index = workspace.device.index
        self._scratch = self._workspace.data_ptr()
        self._scratch_bytes = self._workspace.numel()
        self._pool_shape = (plan.adapter_count, plan.max_rank, plan.input_width)
        self._output_shape = (plan.adapter_count, plan.output_width, plan.max_rank)

    @property
    def plan(self) -> AdapterPlan:
        return self._plan

    @property
    def scratch(self) -> torch.Tensor:
        return self._workspace

    def _rows(self, tensor: torch.Tensor, name: str, rows: int, width: int) -> int:
        """The row stride of an operand (checked)."""

        if tensor.dtype is not self._plan.dtype or tensor.shape != (rows, width) or tensor.get_device() != self._index:
            raise ValueError(f"adapter {name} must be a {self._plan.dtype} tensor of shape {(rows, width)} on {self._device}")
        stride, column = tensor.stride()
        if (column != 1 and width > 1) or (stride < width and rows > 1):
            raise ValueError(f"adapter {name} must have contiguous, separate rows")
        return stride if rows > 1 else width

    def _batch(self, weights: AdapterWeights, adapter_ids: torch.Tensor, rows: int, fault_word: torch.Tensor | None) -> None:
        plan = self._plan
        if rows > plan.row_capacity:
            raise ValueError(f"{rows} adapter rows exceed the prepared capacity {plan.row_capacity}")
        if (
            weights.a.shape != self._pool_shape or weights.b.shape != self._output_shape
            or weights.a.dtype is not plan.dtype or weights.a.get_device() != self._index
        ):
            raise ValueError("adapter weights disagree with the prepared plan")
        if not weights.keeps_storage():
            raise ValueError("the storage of adapter weights was exchanged since their pool was made")
        if (
            adapter_ids.dtype is not torch.int32 or adapter_ids.shape != (rows,) or adapter_ids.get_device() != self._index
            or not adapter_ids.is_contiguous()
        ):
            raise ValueError(f"adapter ids must be a contiguous int32 tensor with one id for each of {rows} rows")
        if fault_word is not None and (
            fault_word.dtype is not torch.int32 or fault_word.numel() < 1 or fault_word.get_device() != self._index
        ):
            raise ValueError("an adapter fault word must be an int32 tensor on the workspace's device")
        if _native.current_device() != self._index:
            raise ValueError(f"adapters of {self._device} need it as the current device")

    def run_into(
        self,
        inputs: torch.Tensor,
        weights: AdapterWeights,
        *,
        adapter_ids: torch.Tensor,
        base: torch.Tensor | None,
        output: torch.Tensor,
        activation: Activation | None = None,
        fault_word: torch.Tensor | None = None,
    ) -> None:
        """Write ``base`` plus the rows' adapters, through ``activation`` if given, to ``output``.

        ``output`` may be ``base`` itself where there is no activation.  A gated activation takes
        INTERLEAVED Gate/Up columns and halves the width.  The fp32 sum is rounded once, at the store:
        the activation sees it unrounded, unlike a projection's fused one.  An id outside
        ``[-1, adapters)`` gives a row of NaN and ORs ``XP_FAULT_ADAPTER_OUT_OF_RANGE`` into ``fault_word``.
        """

        plan = self._plan
        if inputs.ndim != 2:
            raise ValueError("adapter inputs must be a matrix")
        rows = inputs.shape[0]
        self._batch(weights, adapter_ids, rows, fault_word)
        width = plan.output_width
        desc = None
        if activation is not None:
            desc = ctypes.byref(activation.descriptor())
            if activation.gate is not None:
                if width % 2:
                    raise ValueError("a gated activation needs an even number of (INTERLEAVED) columns")
                width //= 2
        ldx = self._rows(inputs, "inputs", rows, plan.input_width)
        ld_base = 0 if base is None else self._rows(base, "base", rows, plan.output_width)
        ld_out = self._rows(output, "output", rows, width)
        _native.call(
            "xp_adapter_apply", ctypes.byref(weights.descriptor), adapter_ids.data_ptr(), rows, inputs.data_ptr(), ldx,
            None if base is None else base.data_ptr(), ld_base, output.data_ptr(), ld_out, desc, self._scratch,
            self._scratch_bytes, None if fault_word is None else fault_word.data_ptr(), _native.current_stream(self._index),
        )

    def backward_into(
        self,
        inputs: torch.Tensor,
        grad_output: torch.Tensor,
        weights: AdapterWeights,
        *,
        adapter_ids: torch.Tensor,
        base: torch.Tensor | None = None,
        grad_inputs: torch.Tensor | None = None,
        grad_a: torch.Tensor | None = None,
        grad_b: torch.Tensor | None = None,
        fault_word: torch.Tensor | None = None,
    ) -> None:
        """Gradients of :meth:`run_into` without an activation.

        ``grad_inputs`` gets ``base`` (the gradient through the shared projection, default 0; it may be
        ``grad_inputs`` itself) plus the rows' adapters' part; ``grad_a`` and ``grad_b`` (asked for
        together, shaped and typed as the weights) are written whole: zero past an adapter's rank and
        for adapters without rows.
        """

        plan = self._plan
        if not plan.backward:
            raise ValueError("the adapter plan was prepared without backward")
        if inputs.ndim != 2:
            raise ValueError("adapter inputs must be a matrix")
        rows = inputs.shape[0]
        self._batch(weights, adapter_ids, rows, fault_word)
        if (grad_a is None) != (grad_b is None):
            raise ValueError("grad_a and grad_b are asked for together")
        if grad_a is not None:
            _require_pool(grad_a, "grad_a", plan.dtype, self._pool_shape, self._device)
            _require_pool(grad_b, "grad_b", plan.dtype, self._output_shape, self._device)
        ldx = self._rows(inputs, "inputs", rows, plan.input_width)
        ld_grad = self._rows(grad_output, "output gradient", rows, plan.output_width)
        ld_base = ld_grad_inputs = 0
        if grad_inputs is not None:
            ld_grad_inputs = self._rows(grad_inputs, "input gradient", rows, plan.input_width)
            if base is not None:
                ld_base = self._rows(base, "base gradient", rows, plan.input_width)
        elif base is not None:
            raise ValueError("a base gradient without an input gradient to add it to")
        _native.call(
            "xp_adapter_backward", ctypes.byref(weights.descriptor), adapter_ids.data_ptr(), rows, inputs.data_ptr(), ldx,
            grad_output.data_ptr(), ld_grad, None if base is None else base.data_ptr(), ld_base,
            None if grad_inputs is None else grad_inputs.data_ptr(), ld_grad_inputs,
            None if grad_a is None else grad_a.data_ptr(), None if grad_b is None else grad_b.data_ptr(), self._scratch,
            self._scratch_bytes, None if fault_word is None else fault_word.data_ptr(), _native.current_stream(self._index),
        )
