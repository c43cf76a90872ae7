"""FfnAgent operators over caller-owned storage: Activation, Gemm and Dense.

Mirrors the reference's operator layer (CrossPool checkout):

- ``Activation`` -- operators/activation.py:87-207 (``fused`` epilogue description,
  ``apply_into`` standalone activation);
- ``GemmPlan`` / ``Gemm`` -- operators/linear.py:28-257 (a prepared projection with its
  scratch, replayed with the current layer's values and bias);
- ``DenseExecutionPlan`` / ``Dense`` -- operators/dense.py:14-86 (i_proj, then the
  standalone activation when no epilogue could be fused -- CONCATENATED Gate/Up order --,
  then o_proj).

Every launch goes to the HIP library on the current torch stream and allocates nothing
(the plan's workspace holds all scratch), so a ``run_into`` can be captured into a graph.
Projections of bf16 payloads with aligned shapes, no bias and either no epilogue or the
gated SiLU epilogue over INTERLEAVED rows take ``xp_gemm_down`` / ``xp_gemm_gate_up_silu``;
every other projection -- fp16 and fp32 payloads, odd K or N, a bias, ReLU / GELU epilogues --
takes ``xp_projection_split``.

Training (no counterpart in the reference): ``Gemm.backward_into`` and, for a whole layer, ``Dense.run_into`` with
``projected`` and ``Dense.backward_into``, of plans prepared with ``backward``; ``crosspool_amd.muon`` updates the weights.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import TYPE_CHECKING

import torch

from crosspool_amd import _native
from crosspool_amd.execution import WorkspaceLayout
from crosspool_amd.ffn import GateTransform, GateUpOrder, GeluActivation, ReluActivation, SiluActivation
from crosspool_amd.weights import DenseFfnWeights, ProjectionWeights

if TYPE_CHECKING:
    from crosspool_amd.adapters import AdapterPlan, DenseAdapterWeights

ActivationSpec = SiluActivation | ReluActivation | GeluActivation

_DTYPE_CODES = {torch.bfloat16: _native.XP_DTYPE_BF16, torch.float16: _native.XP_DTYPE_F16,
                torch.float32: _native.XP_DTYPE_F32}
_ORDER_CODES = {GateUpOrder.CONCATENATED: _native.XP_GATE_UP_CONCATENATED,
                GateUpOrder.INTERLEAVED: _native.XP_GATE_UP_INTERLEAVED}


def _stream() -> ctypes.c_void_p:
    return _native.current_stream()


def _ptr(tensor: torch.Tensor | None) -> ctypes.c_void_p | None:
    return None if tensor is None else ctypes.c_void_p(tensor.data_ptr())


@dataclass(frozen=True, slots=True)
class TensorLayout:
    """Address-free shape, dtype and neutral fill value of one tensor (xpool.quantization.TensorLayout)."""

    shape: tuple[int, ...]
    dtype: torch.dtype
    zero_value: float = 0

    @property
    def nbytes(self) -> int:
        return math.prod(self.shape) * self.dtype.itemsize


@dataclass(frozen=True, slots=True)
class ProjectionLayout:
    """Unquantized projection: values ``[N, K]``, optional fp32 bias ``[N]`` and, for the
    i_proj of a gated layer, the physical Gate/Up row order (weights.py:52-92)."""

    values: TensorLayout
    bias: TensorLayout | None = None
    gate_up_order: GateUpOrder | None = None

    def zero_probe(self, device: torch.device) -> ProjectionWeights:
        """Shape-equivalent zero resources, as the Control Capture Probes (weights.py:66-87)."""

        values = torch.full(self.values.shape, self.values.zero_value, dtype=self.values.dtype, device=device)
        bias = None if self.bias is None else torch.full(self.bias.shape, self.bias.zero_value,
                                                         dtype=self.bias.dtype, device=device)
        return ProjectionWeights(values=values, bias=bias)

    @classmethod
    def of(cls, projection: ProjectionWeights, *, order: GateUpOrder | None = None) -> ProjectionLayout:
        bias = projection.bias
        return cls(
            values=TensorLayout(tuple(projection.values.shape), projection.values.dtype),
            bias=None if bias is None else TensorLayout(tuple(bias.shape), bias.dtype),
            gate_up_order=order,
        )


@dataclass(frozen=True, slots=True)
class Activation:
    """A layer's activation and optional Gate/Up combination (activation.py:87-96)."""

    function: ActivationSpec
    gate: GateTransform | None

    @property
    def supports_inplace(self) -> bool:
        """A standalone ungated activation may reuse its input (activation.py:94-97)."""

        return self.gate is None

    def descriptor(self) -> _native.ActivationDesc:
        function = self.function
        gate = self.gate
        desc = _native.ActivationDesc()
        desc.function = int(function.kind)
        desc.approximate_tanh = int(isinstance(function, GeluActivation) and function.approximate == "tanh")
        desc.alpha = float(function.alpha) if isinstance(function, SiluActivation) else 1.0
        desc.gated = int(gate is not None)
        desc.has_limit = int(gate is not None and gate.limit is not None)
        desc.limit = float(gate.limit) if gate is not None and gate.limit is not None else 0.0
        desc.up_offset = float(gate.up_offset) if gate is not None else 0.0
        return desc

    def fused(self, *, order: GateUpOrder | None) -> Activation | None:
        """The activation as a projection epilogue, or None when it cannot be one: a gated
        activation fuses only over adjacent (INTERLEAVED) Gate/Up rows (activation.py:112-131)."""

        if self.gate is not None and order is not GateUpOrder.INTERLEAVED:
            return None
        return self

    def apply_into(self, *, inputs: torch.Tensor, output: torch.Tensor, order: GateUpOrder | None) -> None:
        """Standalone activation into contiguous bf16 / fp16 storage (activation.py:175-207).

        Inputs already include the projection rounding.  Ungated input and output may be the
        same tensor; a gated input has twice the output width and needs separate storage.
        """

        if self.gate is not None and order is None:
            raise ValueError("gated activation requires a Gate/Up order")
        if inputs.dtype != output.dtype or inputs.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("activation payloads must share one bf16 or fp16 dtype")
        if not inputs.is_contiguous() or not output.is_contiguous():
            raise ValueError("activation payloads must be contiguous")
        width = output.shape[-1]
        rows = output.numel() // width if width else 0
        if inputs.numel() != output.numel() * (2 if self.gate is not None else 1):
            raise ValueError("gated inputs hold two values per output, ungated ones one")
        desc = self.descriptor()
        _native.call(
            "xp_activation", _ptr(inputs), _ptr(output), rows, width, _DTYPE_CODES[output.dtype],
            _ORDER_CODES.get(order, 0), ctypes.byref(desc), _stream(),
        )

    def backward_into(
        self,
        *,
        inputs: torch.Tensor,
        grad_output: torch.Tensor,
        grad_inputs: torch.Tensor,
        order: GateUpOrder | None,
    ) -> None:
        """Gradient of :meth:`apply_into`'s inputs, in their shape and order (no counterpart in the reference).

        A value clipped by the gate transform's limit gets none; one at the limit does, and NaN is not clipped:
        a NaN Gate makes both gradients of its pair NaN, a NaN Up the Gate's.  ``grad_inputs``
        may be ``inputs`` itself, and for an ungated activation ``grad_output`` itself.
        """

        if self.gate is not None and order is None:
            raise ValueError("gated activation requires a Gate/Up order")
        dtype = inputs.dtype
        if dtype not in (torch.bfloat16, torch.float16) or grad_output.dtype is not dtype or grad_inputs.dtype is not dtype:
            raise ValueError("activation payloads must share one bf16 or fp16 dtype")
        device = inputs.get_device()  # -1: not on a GPU
        if device < 0 or grad_output.get_device() != device or grad_inputs.get_device() != device:
            raise ValueError("activation payloads must share one GPU")
        if device != _native.current_device():
            raise ValueError(f"activation payloads of {inputs.device} need it as the current device")
        if not (inputs.is_contiguous() and grad_output.is_contiguous() and grad_inputs.is_contiguous()):
            raise ValueError("activation payloads must be contiguous")
        if grad_output.ndim < 1:
            raise ValueError("activation payloads must have rows")
        width = grad_output.shape[-1]
        wide = width if self.gate is None else 2 * width
        if inputs.shape != (*grad_output.shape[:-1], wide) or grad_inputs.shape != inputs.shape:
            raise ValueError("gated inputs hold two values per output, ungated ones one")
        rows = grad_output.numel() // width if width else 0
        desc = self.descriptor()
        _native.call(
            "xp_activation_backward", inputs.data_ptr(), grad_output.data_ptr(), grad_inputs.data_ptr(), rows, width,
            _DTYPE_CODES[dtype], 0 if order is None else _ORDER_CODES[order], ctypes.byref(desc),
            _native.current_stream(device),
        )


@dataclass(frozen=True, slots=True)
class GemmPlan:
    """Address-free operand layout, epilogue and scratch of one projection (linear.py:28-131)."""

    input_layout: TensorLayout
    weight_layout: ProjectionLayout
    output_layout: TensorLayout
    fused_activation: Activation | None
    workspace: WorkspaceLayout
    kernel: str  # "gate_up_silu" or "down" (xp_gemm_*) or "projection" (xp_projection_split)
    backward: bool = False

    @classmethod
    def prepare(
        cls,
        *,
        input_layout: TensorLayout,
        weight_layout: ProjectionLayout,
        result_layout: TensorLayout,
        activation: Activation | None,
        backward: bool = False,
    ) -> GemmPlan:
        """Choose the kernel and size its scratch; the fused epilogue keeps the projection
        rounding to the result dtype (linear.py:42-96).  ``backward``: the scratch of ``backward_into`` too
        (a projection without an activation)."""

        if backward and activation is not None:
            raise ValueError("the gradients of a projection with an activation are those of a Dense layer's backward pass")

        if len(input_layout.shape) != 2 or len(result_layout.shape) != 2 or len(weight_layout.values.shape) != 2:
            raise ValueError("GEMM input, weights and result must be matrices")
        rows, hidden = input_layout.shape
        width, reduction = weight_layout.values.shape
        if reduction != hidden:
            raise ValueError("GEMM weights disagree with the input width")
        dtype = input_layout.dtype
        if weight_layout.values.dtype is not dtype or result_layout.dtype is not dtype:
            raise ValueError("GEMM input, weights and result must share one payload dtype")
        if activation is not None and activation.gate is not None and weight_layout.gate_up_order is None:
            raise ValueError("gated GEMM preparation requires physical Gate/Up order")
        fused = None if activation is None else activation.fused(order=weight_layout.gate_up_order)
        gated_epilogue = fused is not None and fused.gate is not None
        output_width = width // 2 if gated_epilogue else width
        if result_layout.shape != (rows, output_width):
            raise ValueError(f"GEMM result must be {(rows, output_width)}")
        # xp_gemm_down and xp_gemm_gate_up_silu take bf16 rows of 16-byte multiples, no bias, and at
        # most 16384 columns on the side the C ABI treats as the hidden size (N for down, K for
        # gate_up).  xp_projection chooses among its own kernels and the tuned 16-bit ones.
        aligned = dtype is torch.bfloat16 and weight_layout.bias is None and hidden % 8 == 0 and width % 16 == 0
        if aligned and fused is None and width <= 16384:
            kernel = "down"
            scratch = _native.gemm_workspace_bytes_upto(rows, width, hidden, False)
        elif aligned and gated_epilogue and isinstance(fused.function, SiluActivation) and hidden <= 16384:
            kernel = "gate_up_silu"
            scratch = _native.gemm_workspace_bytes_upto(rows, width, hidden, True)
        else:
            kernel = "projection"
            scratch = _native.library().xp_projection_workspace_bytes(rows, width, hidden, _DTYPE_CODES[dtype])
        if backward:
            query = _native.library().xp_projection_backward_workspace_bytes
            needed = int(query(rows, width, hidden, _DTYPE_CODES.get(dtype, 0)))
            if needed == 0:
                raise ValueError("projection gradients take 1 to 2^24 rows, widths of 1 to 2^20 and bf16, fp16 or fp32 payloads")
            scratch = max(scratch, needed)  # a call of either kind uses it whole
        regions = ((torch.uint8, (scratch,)),) if scratch else ()
        return cls(
            input_layout=input_layout,
            weight_layout=weight_layout,
            output_layout=TensorLayout((rows, output_width), dtype),
            fused_activation=fused,
            workspace=WorkspaceLayout.from_regions(regions),
            kernel=kernel,
            backward=backward,
        )


def _row_stride(tensor: torch.Tensor, name: str, shape: tuple[int, int], dtype: torch.dtype, index: int) -> int:
    """The row stride of an operand of a training operator (checked)."""

    if tensor.shape != shape or tensor.dtype is not dtype or tensor.get_device() != index:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on cuda:{index}")
    stride, column = tensor.stride()
    if (column != 1 and shape[1] > 1) or (stride < shape[1] and shape[0] > 1):
        raise ValueError(f"{name} must have contiguous, separate rows")
    return stride if shape[0] > 1 else shape[1]


def _check_gradient(tensor: torch.Tensor | None, name: str, shape: tuple[int, ...], dtypes: tuple[torch.dtype, ...],
                    index: int) -> int | None:
    """The address of a weight's or bias's gradient (checked), or None."""

    if tensor is None:
        return None
    if tensor.shape != shape or tensor.dtype not in dtypes or tensor.get_device() != index or not tensor.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of shape {tuple(shape)} on cuda:{index}, {' or '.join(map(str, dtypes))}")
    return tensor.data_ptr()


def _check_projection(projection: ProjectionWeights, layout: ProjectionLayout, name: str, index: int) -> None:
    """Weights as they were prepared for, on the device of a training operator."""

    values = projection.values
    if values.shape != layout.values.shape or values.dtype is not layout.values.dtype or values.get_device() != index:
        raise ValueError(f"{name} weights disagree with the prepared layout")
    if (projection.bias is None) != (layout.bias is None):
        raise ValueError(f"{name} bias presence disagrees with the prepared layout")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two non-empty matrices of a training operator share addresses, the gaps between their rows among them."""

    (a_begin, a_end), (b_begin, b_end) = (
        (t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size()) for t in (a, b))
    return a_begin < b_end and b_begin < a_end


def _require_current(index: int) -> None:
    if _native.current_device() != index:
        raise ValueError(f"operands on cuda:{index} need it as the current device")


class Gemm:
    """Capture-time projection borrowing its plan and scratch (linear.py:134-257)."""

    def __init__(self, plan: GemmPlan, workspace: torch.Tensor) -> None:
        if workspace.device.type != "cuda":
            raise ValueError("GEMM scratch must reside on its execution device")
        self.plan = plan
        views = plan.workspace.views(workspace) if plan.workspace.nbytes else ()
        self.scratch = views[0] if views else None

    def run_into(self, inputs: torch.Tensor, projection: ProjectionWeights, *, output: torch.Tensor) -> None:
        """Write the prepared projection of ``inputs`` with the current layer's values and bias."""

        plan = self.plan
        rows, hidden = plan.input_layout.shape
        if inputs.shape[0] > rows or inputs.shape[1] != hidden or inputs.dtype is not plan.input_layout.dtype:
            raise ValueError("GEMM input disagrees with the prepared layout")
        if tuple(projection.values.shape) != plan.weight_layout.values.shape:
            raise ValueError("GEMM weights disagree with the prepared layout")
        if (projection.bias is None) != (plan.weight_layout.bias is None):
            raise ValueError("GEMM bias presence disagrees with the prepared layout")
        live = inputs.shape[0]
        width = projection.values.shape[0]
        scratch = _ptr(self.scratch)
        scratch_bytes = 0 if self.scratch is None else self.scratch.numel()
        if plan.kernel == "down":
            _native.call(
                "xp_gemm_down", _ptr(inputs), live, hidden, _ptr(projection.values), width, _ptr(output), None, live,
                scratch, scratch_bytes, _stream(),
            )
        elif plan.kernel == "gate_up_silu":
            function, gate = plan.fused_activation.function, plan.fused_activation.gate
            _native.call(
                "xp_gemm_gate_up_silu", _ptr(inputs), live, hidden, _ptr(projection.values), width // 2,
                _ptr(output), float(function.alpha), float(gate.limit or 0.0), float(gate.up_offset), scratch,
                scratch_bytes, _stream(),
            )
        else:
            desc = None if plan.fused_activation is None else plan.fused_activation.descriptor()
            _native.call(
                "xp_projection_split", _ptr(inputs), live, hidden, _ptr(projection.values), width,
                _ptr(projection.bias), _ptr(output), _DTYPE_CODES[inputs.dtype],
                None if desc is None else ctypes.byref(desc), scratch, scratch_bytes, _stream(),
            )


    def backward_into(
        self,
        inputs: torch.Tensor | None,
        grad_output: torch.Tensor,
        projection: ProjectionWeights,
        *,
        grad_inputs: torch.Tensor | None = None,
        grad_values: torch.Tensor | None = None,
        grad_bias: torch.Tensor | None = None,
        accumulate: bool = False,
    ) -> None:
        """Gradients of :meth:`run_into` without an activation (no counterpart in the reference), those that are asked for.

        ``grad_inputs`` gets ``grad_output @ values``, ``grad_values`` (of the payload dtype or fp32)
        ``grad_output.T @ inputs`` and ``grad_bias`` (fp32) the sum of ``grad_output``'s rows; ``accumulate`` adds the last
        two to what they hold.  Only ``grad_values`` reads ``inputs``, which may be None without it.  Rows may lie any stride
        up to 2^20 elements apart, but rows of whole 16 bytes on 16-byte boundaries.
        Without rows the weights' and the bias's gradients are zero.
        """

        plan = self.plan
        if not plan.backward:
            raise ValueError("the GEMM plan was prepared without backward")
        capacity, hidden = plan.input_layout.shape
        width = plan.output_layout.shape[1]
        dtype = plan.input_layout.dtype
        if grad_output.ndim != 2 or grad_output.shape[0] > capacity:
            raise ValueError("GEMM output gradient disagrees with the prepared layout")
        rows = grad_output.shape[0]
        index = self.scratch.get_device()
        _check_projection(projection, plan.weight_layout, "GEMM", index)
        _require_current(index)
        if grad_bias is not None and plan.weight_layout.bias is None:
            raise ValueError("a bias gradient of a projection without a bias")
        ld_grad = _row_stride(grad_output, "output gradient", (rows, width), dtype, index)
        if inputs is None and grad_values is not None:
            raise ValueError("the gradient of a projection's values needs its inputs")
        ld_inputs = hidden if inputs is None else _row_stride(inputs, "inputs", (rows, hidden), dtype, index)
        ld_grad_inputs = hidden
        if grad_inputs is not None:
            ld_grad_inputs = _row_stride(grad_inputs, "input gradient", (rows, hidden), dtype, index)
        values_at = _check_gradient(grad_values, "grad_values", (width, hidden), (dtype, torch.float32), index)
        bias_at = _check_gradient(grad_bias, "grad_bias", (width,), (torch.float32,), index)
        _native.call(
            "xp_projection_backward", None if inputs is None else inputs.data_ptr(), ld_inputs, rows, hidden,
            projection.values.data_ptr(), width, grad_output.data_ptr(), ld_grad, _DTYPE_CODES[dtype],
            None if grad_inputs is None else grad_inputs.data_ptr(),
            ld_grad_inputs, values_at, _DTYPE_CODES[dtype if grad_values is None else grad_values.dtype], bias_at,
            int(accumulate), capacity, self.scratch.data_ptr(), self.scratch.numel(), _native.current_stream(index),
        )


@dataclass(frozen=True, slots=True)
class DenseSignature:
    """Dense operator identity (execution.py:73-95 DenseFfnExecutionSignature): payload
    dtype and capacity, widths, activation and the two projection layouts."""

    payload_dtype: torch.dtype
    payload_row_capacity: int
    hidden_size: int
    local_intermediate_size: int
    activation: Activation
    i_proj: ProjectionLayout
    o_proj: ProjectionLayout

    @property
    def payload_shape(self) -> tuple[int, int]:
        return self.payload_row_capacity, self.hidden_size


@dataclass(frozen=True, slots=True)
class DenseAdapterLayout:
    """Adapter pools beside a Dense layer's projections: their adapters, and the largest rank of each
    projection's (None: that projection has no pool)."""

    adapter_count: int
    i_proj_rank: int | None = None
    o_proj_rank: int | None = None

    def __post_init__(self) -> None:
        if self.i_proj_rank is None and self.o_proj_rank is None:
            raise ValueError("a Dense adapter layout names a rank for at least one projection")


@dataclass(frozen=True, slots=True)
class DenseGradients:
    """Where a Dense layer's backward pass writes the gradients of its weights, each left out where None: values of
    the payload dtype or fp32 (both the same), biases fp32."""

    i_values: torch.Tensor | None = None
    o_values: torch.Tensor | None = None
    i_bias: torch.Tensor | None = None
    o_bias: torch.Tensor | None = None

    def __post_init__(self) -> None:
        if self.i_values is not None and self.o_values is not None and self.i_values.dtype is not self.o_values.dtype:
            raise ValueError("gradients of a Dense layer's values share one dtype")


@dataclass(frozen=True, slots=True)
class DenseExecutionPlan:
    """Two prepared projections and their shared intermediate storage (dense.py:14-52).

    With ``adapters`` the layer also takes low-rank adapters by row (``crosspool_amd.adapters``); an i_proj
    with a pool leaves the activation to the kernel that adds its adapters.  With ``backward`` it can be trained:
    its forward pass keeps the projected values, and ``Dense.backward_into`` gives the gradients.
    """

    signature: DenseSignature
    i_proj: GemmPlan
    o_proj: GemmPlan
    workspace: WorkspaceLayout
    adapters: DenseAdapterLayout | None = None
    i_proj_adapter: AdapterPlan | None = None
    o_proj_adapter: AdapterPlan | None = None
    backward: bool = False

    @classmethod
    def prepare(
        cls, signature: DenseSignature, *, adapters: DenseAdapterLayout | None = None, backward: bool = False
    ) -> DenseExecutionPlan:
        dtype = signature.payload_dtype
        capacity = signature.payload_row_capacity
        if backward and adapters is not None:
            raise ValueError("a Dense layer with adapters is trained through Gemm, Adapter and Activation")
        if (backward and dtype is torch.float32 and signature.activation.gate is not None
                and signature.i_proj.gate_up_order is not GateUpOrder.INTERLEAVED):
            raise ValueError("a gated fp32 Dense layer takes INTERLEAVED Gate/Up rows")
        activated = TensorLayout((capacity, signature.local_intermediate_size), dtype)
        adapted = adapters is not None and adapters.i_proj_rank is not None
        apart = signature.activation.fused(order=signature.i_proj.gate_up_order) is None
        gate = signature.activation.gate
        if adapted and apart and adapters.o_proj_rank is None and gate is not None and gate.limit is not None:
            # The limit would make a NaN row of an id out of range finite, and no later pool restores it.
            raise ValueError("a clipped gate over CONCATENATED columns takes i_proj adapters only beside o_proj adapters")
        activation = None if adapted else signature.activation
        fused = activation is not None and activation.fused(order=signature.i_proj.gate_up_order) is not None
        i_proj = GemmPlan.prepare(
            input_layout=TensorLayout(signature.payload_shape, dtype),
            weight_layout=signature.i_proj,
            result_layout=activated if fused else TensorLayout((capacity, signature.i_proj.values.shape[0]), dtype),
            activation=activation,
        )
        o_proj = GemmPlan.prepare(
            input_layout=activated, weight_layout=signature.o_proj,
            result_layout=TensorLayout(signature.payload_shape, dtype), activation=None,
        )
        regions = [(dtype, i_proj.output_layout.shape)]
        if i_proj.fused_activation is None and (adapted or not signature.activation.supports_inplace):
            regions.append((dtype, activated.shape))
        regions += [(torch.uint8, (i_proj.workspace.nbytes,)), (torch.uint8, (o_proj.workspace.nbytes,))]
        plans: list[AdapterPlan | None] = [None, None]
        if adapters is not None:
            from crosspool_amd.adapters import AdapterPlan

            for index, (rank, layout) in enumerate(
                ((adapters.i_proj_rank, signature.i_proj), (adapters.o_proj_rank, signature.o_proj))
            ):
                if rank is not None:
                    width, reduction = layout.values.shape
                    plans[index] = AdapterPlan.prepare(
                        row_capacity=capacity, adapter_count=adapters.adapter_count, max_rank=rank,
                        input_width=reduction, output_width=width, dtype=dtype,
                    )
            # One region serves both: their calls follow one another.
            regions.append((torch.uint8, (max(plan.workspace.nbytes for plan in plans if plan is not None),)))
        if backward:
            wide, hidden = signature.i_proj.values.shape
            code, lib = _DTYPE_CODES.get(dtype, 0), _native.library()
            needed = int(lib.xp_dense_backward_workspace_bytes(
                capacity, hidden, signature.local_intermediate_size, int(signature.activation.gate is not None), code))
            if needed == 0:
                raise ValueError("a Dense layer's backward pass takes 1 to 2^24 rows, widths of 1 to 2^20 and bf16, fp16 or fp32")
            needed = max(needed, int(lib.xp_projection_keep_workspace_bytes(capacity, wide, hidden, code)),
                         int(lib.xp_projection_keep_workspace_bytes(capacity, hidden, signature.local_intermediate_size, code)))
            regions.append((torch.uint8, (needed,)))
        return cls(signature, i_proj, o_proj, WorkspaceLayout.from_regions(tuple(regions)), adapters, *plans, backward)


class Dense:
    """Capture-time Dense computation over a prepared workspace (dense.py:55-86)."""

    def __init__(self, plan: DenseExecutionPlan, workspace: torch.Tensor) -> None:
        views = list(plan.workspace.views(workspace))
        self.plan = plan
        self.i_adapter = self.o_adapter = None
        self.training_scratch = views.pop() if plan.backward else None
        if plan.adapters is not None:
            from crosspool_amd.adapters import Adapter

            scratch = views.pop()
            self.i_adapter = None if plan.i_proj_adapter is None else Adapter(plan.i_proj_adapter, scratch)
            self.o_adapter = None if plan.o_proj_adapter is None else Adapter(plan.o_proj_adapter, scratch)
        self.projected = views[0]
        separate = plan.i_proj.fused_activation is None and (
            self.i_adapter is not None or not plan.signature.activation.supports_inplace
        )
        self.activated = views[1] if separate else self.projected
        self.i_proj = Gemm(plan.i_proj, views[-2])
        self.o_proj = Gemm(plan.o_proj, views[-1])

    def run_into(
        self,
        *,
        hidden_states: torch.Tensor,
        layer_weights: DenseFfnWeights,
        output: torch.Tensor,
        adapters: DenseAdapterWeights | None = None,
        adapter_ids: torch.Tensor | None = None,
        fault_word: torch.Tensor | None = None,
        projected: torch.Tensor | None = None,
    ) -> None:
        """Write the complete rank-local partial of ``hidden_states`` into ``output``.

        ``projected`` (of a plan prepared with ``backward``; contiguous ``[rows, i_proj width]`` of the payload dtype)
        gets the projected values that :meth:`backward_into` reads.  Its activation is that of the unrounded sums (of the kept
        values for CONCATENATED weights of 2 GiB and more), so outputs may differ in a last bit from those of a call without
        it; and a NaN Gate or Up is past no limit, as in the backward pass, where a call without it makes the limit of it.

        ``adapters`` (of a plan prepared for them) adds the low-rank adapters that ``adapter_ids`` (int32,
        one per row, -1: none) names to each projection; an id outside the pool gives a row of NaN and a
        bit in ``fault_word``.  With i_proj adapters the activation is that of
        ``Adapter.run_into``: rows without an adapter may differ in a last bit from those of a layer without
        pools, and a NaN that a limit hides there stays.
        """

        if (adapters is None) != (adapter_ids is None):
            raise ValueError("adapters and adapter ids come together")
        if adapters is not None:
            if (adapters.i_proj is None) != (self.i_adapter is None) or (adapters.o_proj is None) != (self.o_adapter is None):
                raise ValueError("Dense adapters disagree with the prepared plan")
        elif self.i_adapter is not None and self.plan.signature.payload_dtype is torch.float32:
            raise ValueError("an fp32 Dense layer prepared for i_proj adapters takes them in every call (id -1: none)")
        if projected is not None:
            self._run_keeping(hidden_states, layer_weights, output, projected)
            return
        rows = hidden_states.shape[0]
        projected = self.projected[:rows]
        self.i_proj.run_into(hidden_states, layer_weights.i_proj, output=projected)
        activated = self.activated[:rows]
        activation, order = self.plan.signature.activation, self.plan.signature.i_proj.gate_up_order
        pending = self.plan.i_proj.fused_activation is None
        if adapters is not None and adapters.i_proj is not None:
            fused = activation.fused(order=order)
            self.i_adapter.run_into(
                hidden_states, adapters.i_proj, adapter_ids=adapter_ids, base=projected,
                output=projected if fused is None else activated, activation=fused, fault_word=fault_word,
            )
            pending = fused is None
        if pending:
            activation.apply_into(inputs=projected, output=activated, order=order)
        self.o_proj.run_into(activated, layer_weights.o_proj, output=output)
        if adapters is not None and adapters.o_proj is not None:
            self.o_adapter.run_into(
                activated, adapters.o_proj, adapter_ids=adapter_ids, base=output[:rows], output=output[:rows],
                fault_word=fault_word,
            )

    def _trained(self, layer_weights: DenseFfnWeights, rows: int) -> int:
        """The device index of a training call (checked)."""

        signature = self.plan.signature
        if self.training_scratch is None:
            raise ValueError("the Dense plan was prepared without backward")
        if rows > signature.payload_row_capacity:
            raise ValueError(f"{rows} Dense rows exceed the prepared capacity {signature.payload_row_capacity}")
        index = self.training_scratch.get_device()
        _check_projection(layer_weights.i_proj, signature.i_proj, "i_proj", index)
        _check_projection(layer_weights.o_proj, signature.o_proj, "o_proj", index)
        _require_current(index)
        return index

    def _run_keeping(
        self, hidden_states: torch.Tensor, layer_weights: DenseFfnWeights, output: torch.Tensor, projected: torch.Tensor
    ) -> None:
        signature = self.plan.signature
        if hidden_states.ndim != 2:
            raise ValueError("hidden states must be a matrix")
        rows = hidden_states.shape[0]
        index = self._trained(layer_weights, rows)
        dtype, hidden, wide = signature.payload_dtype, signature.hidden_size, signature.i_proj.values.shape[0]
        ld_hidden = _row_stride(hidden_states, "hidden states", (rows, hidden), dtype, index)
        for name, tensor, shape in (("projected", projected, (rows, wide)), ("output", output, (rows, hidden))):
            _check_gradient(tensor, name, shape, (dtype,), index)
        if output.numel() and (_overlap(output, projected) or _overlap(output, hidden_states)):
            raise ValueError("a trained Dense layer's output must not overlap its hidden states and kept values")
        order = signature.i_proj.gate_up_order
        activated = self.activated[:rows]
        # The product works on pairs of Gate and Up rows in either order; halves of 2 GiB and more are past its offsets.
        fused = signature.activation.fused(order=order) is not None or wide * (hidden + 7) * dtype.itemsize < 1 << 31
        bias = layer_weights.i_proj.bias
        scratch = self.training_scratch
        desc = signature.activation.descriptor()
        _native.call(
            "xp_projection_keep", hidden_states.data_ptr(), ld_hidden, rows, hidden, layer_weights.i_proj.values.data_ptr(),
            wide, None if bias is None else bias.data_ptr(), projected.data_ptr(), wide,
            activated.data_ptr() if fused else None, _DTYPE_CODES[dtype], 0 if order is None else _ORDER_CODES[order],
            ctypes.byref(desc) if fused else None,
            signature.payload_row_capacity, scratch.data_ptr(), scratch.numel(), _native.current_stream(index),
        )
        if not fused:
            _native.call(
                "xp_kept_activation", projected.data_ptr(), activated.data_ptr(), rows, signature.local_intermediate_size,
                _DTYPE_CODES[dtype], _ORDER_CODES[order], ctypes.byref(desc), _native.current_stream(index),
            )
        width, bias = signature.local_intermediate_size, layer_weights.o_proj.bias
        # What the general projection kernel would compute (fp32; sums of no whole 64s) is mostly faster on the training
        # products' tiles (rows x width x hidden, us: fp16 777 x 2056 x 1032 14 against 25, fp32 494 x 11584 x 8288 711 against
        # 887; the other way round fp16 777 x 6152 x 4096 68 against 65, 512 rows 59 against 44).  Where rows are no whole 16
        # bytes the tiles' padded copies cost more than that for few rows.  Tiles / general, fp16, 777, 1024, 1500 and 4096
        # rows: 2053 x 1030 24 / 30, 30 / 32, 33 / 32, 55 / 71; 6145 x 2050 71 / 60, 94 / 68, 84 / 92, 180 / 276; 8003 x 4001
        # 105 / 102, 117 / 110, 162 / 171, 287 / 383.  fp32, 256, 512 and 777 rows: 31 / 23, 41 / 43, 54 / 69; 86 / 103,
        # 148 / 171, 216 / 274; 201 / 183, 310 / 348, 468 / 517.
        chunk = 16 // dtype.itemsize
        general = self.plan.o_proj.kernel == "projection" and (dtype is torch.float32 or width % 64 != 0)
        if not general or (width % chunk != 0 and rows < (512 if dtype is torch.float32 else 1280)):
            self.o_proj.run_into(activated, layer_weights.o_proj, output=output)
            return
        _native.call(
            "xp_projection_keep", activated.data_ptr(), width, rows, width, layer_weights.o_proj.values.data_ptr(), hidden,
            None if bias is None else bias.data_ptr(), output.data_ptr(), hidden, None, _DTYPE_CODES[dtype], 0, None,
            signature.payload_row_capacity, scratch.data_ptr(), scratch.numel(), _native.current_stream(index),
        )

    def backward_into(
        self,
        *,
        hidden_states: torch.Tensor | None = None,
        layer_weights: DenseFfnWeights,
        projected: torch.Tensor,
        grad_output: torch.Tensor,
        grad_hidden_states: torch.Tensor | None = None,
        gradients: DenseGradients | None = None,
        accumulate: bool = False,
    ) -> None:
        """Gradients of :meth:`run_into` of the same rows, weights and kept ``projected`` (no counterpart in the reference).

        ``grad_hidden_states`` and what ``gradients`` names are written; ``accumulate`` adds the weights' and biases'
        gradients to what they hold.  Only i_proj's gradient reads ``hidden_states``, which may be left out without it (a frozen
        layer).  The gradient of the projected values is rounded to the payload dtype between
        the products, as the activated values are; the biases' gradients sum unrounded values.  Clipped values
        get no gradient, as in :meth:`Activation.backward_into`.
        """

        signature = self.plan.signature
        if grad_output.ndim != 2:
            raise ValueError("a Dense layer's output gradient must be a matrix")
        rows = grad_output.shape[0]
        index = self._trained(layer_weights, rows)
        dtype, hidden, width = signature.payload_dtype, signature.hidden_size, signature.local_intermediate_size
        wide = signature.i_proj.values.shape[0]
        ld_hidden = hidden
        if hidden_states is not None:
            ld_hidden = _row_stride(hidden_states, "hidden states", (rows, hidden), dtype, index)
        ld_projected = _row_stride(projected, "projected", (rows, wide), dtype, index)
        ld_grad = _row_stride(grad_output, "output gradient", (rows, hidden), dtype, index)
        ld_grad_hidden = hidden
        if grad_hidden_states is not None:
            ld_grad_hidden = _row_stride(grad_hidden_states, "gradient of the hidden states", (rows, hidden), dtype, index)
        into = DenseGradients() if gradients is None else gradients
        if hidden_states is None and into.i_values is not None:
            raise ValueError("the gradient of an i_proj's values needs the hidden states")
        for name, bias, projection in (("i_proj", into.i_bias, signature.i_proj), ("o_proj", into.o_bias, signature.o_proj)):
            if bias is not None and projection.bias is None:
                raise ValueError(f"a bias gradient of an {name} without a bias")
        kinds = (dtype, torch.float32)
        i_values = _check_gradient(into.i_values, "i_proj gradient", (wide, hidden), kinds, index)
        o_values = _check_gradient(into.o_values, "o_proj gradient", (hidden, width), kinds, index)
        i_bias = _check_gradient(into.i_bias, "i_proj bias gradient", (wide,), (torch.float32,), index)
        o_bias = _check_gradient(into.o_bias, "o_proj bias gradient", (hidden,), (torch.float32,), index)
        kept = into.i_values if into.i_values is not None else into.o_values
        order = signature.i_proj.gate_up_order
        scratch = self.training_scratch
        desc = signature.activation.descriptor()
        _native.call(
            "xp_dense_backward", None if hidden_states is None else hidden_states.data_ptr(), ld_hidden, rows, hidden,
            layer_weights.i_proj.values.data_ptr(), layer_weights.o_proj.values.data_ptr(), width, projected.data_ptr(),
            ld_projected, grad_output.data_ptr(), ld_grad,
            _DTYPE_CODES[dtype], 0 if order is None else _ORDER_CODES[order], ctypes.byref(desc),
            None if grad_hidden_states is None else grad_hidden_states.data_ptr(), ld_grad_hidden, i_values, o_values,
            _DTYPE_CODES[dtype if kept is None else kept.dtype], i_bias, o_bias, int(accumulate),
            signature.payload_row_capacity, scratch.data_ptr(), scratch.numel(), _native.current_stream(index),
        )
