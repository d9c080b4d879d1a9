"""``linear`` for the experts of a mixture: the rows of ``x`` are sorted by expert, and the rows
``offsets[e] .. offsets[e + 1]`` are multiplied with the quantized weight of expert e.

The weight is a ``MatmulInputHandleRef`` of logical shape ``[E, N, K]``; ``offsets`` holds E + 1 ascending int32 or int64 on
the device, so a router's counts never come to the host.  An expert may have no rows; rows outside
``[offsets[0], offsets[E])`` are left as they were in every output."""
from __future__ import annotations

from .linear import Activation, _Call, backward_workspace_bytes, workspace_bytes  # noqa: F401
from .matmul_input import MatmulInputHandleRef
from .scheme import ElemType
from .tensor import ComputeClient, TensorHandleRef


class Prepared(_Call):
    """``launch`` with the argument marshalling done once."""

    def __init__(self, client: ComputeClient, input: TensorHandleRef, offsets: TensorHandleRef, weight: MatmulInputHandleRef,
                 output: TensorHandleRef, dtype: ElemType, bias: TensorHandleRef | None = None,
                 residual: TensorHandleRef | None = None, activation: Activation = Activation.Identity,
                 pre: TensorHandleRef | None = None, workspace: TensorHandleRef | None = None):
        super().__init__("qk_grouped_linear", (input, offsets), weight, lambda o: (o[0], o[1], int(activation), o[2], o[3]),
                         (bias, residual, output, pre), dtype, workspace, client)


class PreparedBackward(_Call):
    """``launch_backward`` with the argument marshalling done once."""

    def __init__(self, client: ComputeClient, grad_output: TensorHandleRef, offsets: TensorHandleRef, weight: MatmulInputHandleRef,
                 grad_input: TensorHandleRef | None, dtype: ElemType, pre: TensorHandleRef | None = None,
                 activation: Activation = Activation.Identity, grad_bias: TensorHandleRef | None = None,
                 grad_pre: TensorHandleRef | None = None, workspace: TensorHandleRef | None = None):
        super().__init__("qk_grouped_linear_backward", (grad_output, offsets), weight, lambda o: (int(activation), *o),
                         (pre, grad_input, grad_bias, grad_pre), dtype, workspace, client)


def launch(client: ComputeClient, input: TensorHandleRef, offsets: TensorHandleRef, weight: MatmulInputHandleRef,
           output: TensorHandleRef, dtype: ElemType, bias: TensorHandleRef | None = None, residual: TensorHandleRef | None = None,
           activation: Activation = Activation.Identity, pre: TensorHandleRef | None = None,
           workspace: TensorHandleRef | None = None) -> None:
    """``output[r] = act(input[r] W[e]^T + bias[e]) + residual[r]`` for the rows r of every expert e; ``bias`` is ``[E, N]``."""
    Prepared(client, input, offsets, weight, output, dtype, bias, residual, activation, pre, workspace)()


def launch_backward(client: ComputeClient, grad_output: TensorHandleRef, offsets: TensorHandleRef, weight: MatmulInputHandleRef,
                    grad_input: TensorHandleRef | None, dtype: ElemType, pre: TensorHandleRef | None = None,
                    activation: Activation = Activation.Identity, grad_bias: TensorHandleRef | None = None,
                    grad_pre: TensorHandleRef | None = None, workspace: TensorHandleRef | None = None) -> None:
    """Gradients of ``launch``, as ``linear.launch_backward`` per expert; ``grad_bias`` is ``[E, N]``, zero for an expert
    without rows."""
    PreparedBackward(client, grad_output, offsets, weight, grad_input, dtype, pre, activation, grad_bias, grad_pre, workspace)()
