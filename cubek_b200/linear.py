"""Products with quantized weights: ``y = act(x W^T + bias) + residual`` and its gradient.

The weight is the quantized matmul operand of the reference (``MatmulInputHandleRef::quantized``,
crates/cubek-matmul/src/base.rs:436-452) with logical shape ``[N, K]``, packed along K, as ``quantize`` writes it.  Its
value is, to the bit, what ``dequantize`` returns in the type of ``x`` (f16 or bf16); products are summed in f32 and ``y``
is rounded once.  ``grouped_linear`` is the same for the experts of a mixture."""
from __future__ import annotations

import enum

from . import _ffi
from .matmul_input import MatmulInputHandleRef
from .scheme import ElemType
from .tensor import ComputeClient, TensorHandleRef


class Activation(enum.IntEnum):
    """``Gelu`` is z Phi(z), ``GeluTanh`` its tanh form, ``Silu`` z / (1 + exp(-z))."""

    Identity = 0
    Relu = 1
    Gelu = 2
    GeluTanh = 3
    Silu = 4


def workspace_bytes(input: TensorHandleRef, weight: MatmulInputHandleRef, dtype: ElemType) -> int:
    """Device workspace of the forward call."""
    ti, tv = _ffi.c_tensors(input, weight.data)
    return _ffi.lib().qk_linear_workspace_bytes(ti.ref(), tv.ref(), _ffi.c_scheme(weight.scheme), int(dtype))


def backward_workspace_bytes(grad_output: TensorHandleRef, weight: MatmulInputHandleRef, dtype: ElemType,
                             activation: Activation = Activation.Identity, bias: bool = False,
                             grad_pre: TensorHandleRef | None = None) -> int:
    """Device workspace of the backward call; ``bias``: ``grad_bias`` is asked for; ``grad_pre``: what the call gets there."""
    tg, tv = _ffi.c_tensors(grad_output, weight.data)
    keep, pre = _ffi.optional(grad_pre)
    return _ffi.lib().qk_linear_backward_workspace_bytes(tg.ref(), tv.ref(), _ffi.c_scheme(weight.scheme), int(activation), int(bias),
                                                         pre, int(dtype))


class _Call:
    """One C call with its arguments marshalled once."""

    def __init__(self, name, required, weight, middle, optional, dtype, workspace, client):
        self._keep = _ffi.c_tensors(*required, weight.data, weight.scale)
        more = [_ffi.optional(t) for t in optional]
        self._more = [keep for keep, _ in more]
        refs = [ref for _, ref in more]
        self._scheme = _ffi.c_scheme(weight.scheme)
        ws = (workspace.handle, workspace.shape[0] * workspace.elem_size) if workspace else (None, 0)
        self._args = (*(k.ref() for k in self._keep), self._scheme, *middle(refs), int(dtype), *ws, client.stream)
        self._fn = getattr(_ffi.lib(), name)

    def __call__(self) -> None:
        status = self._fn(*self._args)
        if status:
            _ffi.check(status)


class Prepared(_Call):
    """``launch`` with the argument marshalling done once, for callers that run it again on the same buffers."""

    def __init__(self, client: ComputeClient, input: TensorHandleRef, weight: MatmulInputHandleRef, output: TensorHandleRef,
                 dtype: ElemType, bias: TensorHandleRef | None = None, residual: TensorHandleRef | None = None,
                 activation: Activation = Activation.Identity, pre: TensorHandleRef | None = None,
                 workspace: TensorHandleRef | None = None):
        super().__init__("qk_linear", (input,), weight, lambda o: (o[0], o[1], int(activation), o[2], o[3]),
                         (bias, residual, output, pre), dtype, workspace, client)


class PreparedBackward(_Call):
    """``launch_backward`` with the argument marshalling done once."""

    def __init__(self, client: ComputeClient, grad_output: TensorHandleRef, weight: MatmulInputHandleRef,
                 grad_input: TensorHandleRef | None, dtype: ElemType, pre: TensorHandleRef | None = None,
                 activation: Activation = Activation.Identity, grad_bias: TensorHandleRef | None = None,
                 grad_pre: TensorHandleRef | None = None, workspace: TensorHandleRef | None = None):
        super().__init__("qk_linear_backward", (grad_output,), weight, lambda o: (int(activation), *o),
                         (pre, grad_input, grad_bias, grad_pre), dtype, workspace, client)


def launch(client: ComputeClient, input: TensorHandleRef, weight: MatmulInputHandleRef, output: TensorHandleRef, dtype: ElemType,
           bias: TensorHandleRef | None = None, residual: TensorHandleRef | None = None,
           activation: Activation = Activation.Identity, pre: TensorHandleRef | None = None,
           workspace: TensorHandleRef | None = None) -> None:
    """``output = act(input W^T + bias) + residual``.

    ``input`` is ``[.., K]``, ``output`` and ``residual`` ``[.., N]`` (the residual may be the output itself), ``bias`` ``[N]``,
    all of type ``dtype``; ``pre``, if given, receives ``input W^T + bias`` for ``launch_backward``.  Enqueues on
    ``client.stream`` and returns."""
    Prepared(client, input, weight, output, dtype, bias, residual, activation, pre, workspace)()


def launch_backward(client: ComputeClient, grad_output: TensorHandleRef, weight: MatmulInputHandleRef,
                    grad_input: TensorHandleRef | None, dtype: ElemType, pre: TensorHandleRef | None = None,
                    activation: Activation = Activation.Identity, grad_bias: TensorHandleRef | None = None,
                    grad_pre: TensorHandleRef | None = None, workspace: TensorHandleRef | None = None) -> None:
    """Gradients of ``launch``: with ``dz = grad_output * act'(pre)``, ``grad_input = dz W``, ``grad_bias`` the column sums
    of ``dz`` and ``grad_pre`` = ``dz`` itself; those that are None are not computed.  The gradient of the residual is
    ``grad_output``; codes and scales are constants."""
    PreparedBackward(client, grad_output, weight, grad_input, dtype, pre, activation, grad_bias, grad_pre, workspace)()
