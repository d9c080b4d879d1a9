"""What the products with quantized weights refuse, each with its status, before any CUDA call is made."""
import pytest

from cubek_b200 import (ComputeClient, ElemType, LaunchError, QuantLevel, QuantPanic, QuantScheme, QuantStore, QuantValue, TensorHandleRef,
                        grouped_linear, linear)
from cubek_b200 import _ffi
from cubek_b200.linear import Activation
from cubek_b200.matmul_input import MatmulInputHandleRef

CLIENT = ComputeClient(0, 0)
Q4 = QuantScheme(value=QuantValue.Q4S, level=QuantLevel.block([32]))


def fake(shape, elem_size, addr=0x10000, strides=None):
    """A handle with a plausible address; the checks never dereference it."""
    return TensorHandleRef.from_raw_parts(addr, shape, elem_size, strides)


class Raw:
    """A weight operand without the host-side checks, so that the library's own are seen."""

    def __init__(self, data, scale, scheme):
        self.data, self.scale, self.scheme = data, scale, scheme


def weight(shape=(64, 64), scheme=Q4, data=None, scale=None):
    size = 4 if scheme.store == QuantStore.U32 else 1
    return Raw(data or fake(scheme.packed_shape(shape), size), scale or fake(scheme.scales_shape(shape), scheme.param.size), scheme)


def status(call, *args, **kw):
    with pytest.raises((QuantPanic, LaunchError)) as e:
        call(CLIENT, *args, **kw)
    return e.value.status


X, Y = fake((4, 64), 2), fake((4, 64), 2)
BF = ElemType.BF16


@pytest.mark.parametrize("want,kw", [
    (_ffi.QK_ERR_DTYPE, dict(dtype=ElemType.F32)),
    (_ffi.QK_ERR_DTYPE, dict(x=fake((4, 64), 4))),
    (_ffi.QK_ERR_DTYPE, dict(y=fake((4, 64), 4))),
    (_ffi.QK_ERR_SHAPE, dict(x=fake((4, 56), 2))),
    (_ffi.QK_ERR_SHAPE, dict(y=fake((4, 63), 2))),
    (_ffi.QK_ERR_SHAPE, dict(y=fake((5, 64), 2))),
    (_ffi.QK_ERR_SHAPE, dict(bias=fake((63,), 2))),
    (_ffi.QK_ERR_SHAPE, dict(bias=fake((1, 64), 2))),
    (_ffi.QK_ERR_SHAPE, dict(residual=fake((1, 64), 2))),
    (_ffi.QK_ERR_SHAPE, dict(pre=fake((4, 32), 2))),
    (_ffi.QK_ERR_LAYOUT, dict(x=fake((4, 64), 2, strides=(1, 4)))),
    (_ffi.QK_ERR_LAYOUT, dict(x=fake((4, 64), 2, strides=(0, 1)))),
    (_ffi.QK_ERR_LAYOUT, dict(y=fake((4, 64), 2, strides=(32, 1)))),
    (_ffi.QK_ERR_LAYOUT, dict(residual=fake((4, 64), 2, strides=(128, 2)))),
    (_ffi.QK_ERR_ALIGN, dict(x=fake((4, 64), 2, addr=0x10001))),
    (_ffi.QK_ERR_NULL, dict(x=fake((4, 64), 2, addr=0))),
    (_ffi.QK_ERR_NULL, dict(y=fake((4, 64), 2, addr=0))),
    (_ffi.QK_ERR_LAYOUT, dict(w=weight(data=fake((64, 8), 4, strides=(1, 64))))),
    (_ffi.QK_ERR_LAYOUT, dict(w=weight(data=fake((64, 8), 4, strides=(-8, 1))))),
    (_ffi.QK_ERR_DTYPE, dict(w=weight(data=fake((64, 8), 1)))),
    (_ffi.QK_ERR_SHAPE, dict(w=weight(data=fake((1, 64, 8), 4)))),
    (_ffi.QK_ERR_SHAPE, dict(w=weight(scale=fake((64, 3), 4)))),
    (_ffi.QK_ERR_SHAPE, dict(w=weight(scale=fake((128,), 4)))),
    (_ffi.QK_ERR_DTYPE, dict(w=weight(scale=fake((64, 2), 2)))),
    (_ffi.QK_ERR_SHAPE, dict(w=weight(scheme=QuantScheme(value=QuantValue.Q8S), scale=fake((2,), 4)))),
    (_ffi.QK_ERR_BLOCK_SIZE, dict(w=weight(scheme=QuantScheme(value=QuantValue.Q8S, level=QuantLevel.block([12]))))),
    (_ffi.QK_ERR_BLOCK_SIZE, dict(w=weight(scheme=QuantScheme(value=QuantValue.Q8S, level=QuantLevel.block([2]))))),
    (_ffi.QK_ERR_BLOCK_SIZE, dict(w=weight(scheme=QuantScheme(value=QuantValue.E4M3, store=QuantStore.Native, level=QuantLevel.block([20]))))),
    (_ffi.QK_ERR_UNSUPPORTED_SCHEME, dict(w=Raw(fake((64, 64), 1), fake((64, 2), 4), QuantScheme(value=QuantValue.Q4S, store=QuantStore.Native,
                                                                                              level=QuantLevel.block([32]))))),
    (_ffi.QK_ERR_UNSUPPORTED_SCHEME, dict(activation=9)),
    (_ffi.QK_ERR_UNSUPPORTED_SCHEME, dict(activation=-1)),
])
def test_forward(want, kw):
    kw = dict(kw)
    args = (kw.pop("x", X), kw.pop("w", None) or weight(), kw.pop("y", Y), kw.pop("dtype", BF))
    assert status(linear.launch, *args, **kw) == want


@pytest.mark.parametrize("want,kw", [
    (_ffi.QK_ERR_DTYPE, dict(dtype=ElemType.F32)),
    (_ffi.QK_ERR_SHAPE, dict(g=fake((4, 32), 2))),
    (_ffi.QK_ERR_SHAPE, dict(gx=fake((4, 32), 2))),
    (_ffi.QK_ERR_SHAPE, dict(grad_bias=fake((4,), 2))),
    (_ffi.QK_ERR_LAYOUT, dict(grad_bias=fake((64,), 2, strides=(0,)))),
    (_ffi.QK_ERR_NULL, dict(activation=Activation.Silu)),
    (_ffi.QK_ERR_WORKSPACE, dict(activation=Activation.Silu, pre=Y)),
    (_ffi.QK_ERR_WORKSPACE, dict(activation=Activation.Silu, pre=Y, workspace=fake((64,), 1))),
    (_ffi.QK_ERR_ALIGN, dict(activation=Activation.Silu, pre=Y, workspace=fake((1 << 20,), 1, addr=0x10004))),
    (_ffi.QK_ERR_WORKSPACE, dict(g=fake((1000, 64), 2), gx=fake((1000, 64), 2), grad_bias=fake((64,), 2))),
])
def test_backward(want, kw):
    kw = dict(kw)
    args = (kw.pop("g", Y), weight(), kw.pop("gx", X), kw.pop("dtype", BF))
    assert status(linear.launch_backward, *args, **kw) == want


def test_grouped():
    w = weight((3, 64, 64))
    off = fake((4,), 4)
    call = grouped_linear.launch
    assert status(call, X, fake((3,), 4), w, Y, BF) == _ffi.QK_ERR_SHAPE
    assert status(call, X, fake((4, 1), 4), w, Y, BF) == _ffi.QK_ERR_SHAPE
    assert status(call, X, fake((4,), 2), w, Y, BF) == _ffi.QK_ERR_DTYPE
    assert status(call, X, fake((4,), 4, strides=(2,)), w, Y, BF) == _ffi.QK_ERR_LAYOUT
    assert status(call, X, fake((4,), 4, addr=0), w, Y, BF) == _ffi.QK_ERR_NULL
    assert status(call, X, off, weight((64, 64)), Y, BF) == _ffi.QK_ERR_SHAPE
    assert status(call, X, off, w, Y, BF, bias=fake((64,), 2)) == _ffi.QK_ERR_SHAPE
    assert status(call, X, off, w, Y, BF, bias=fake((2, 64), 2)) == _ffi.QK_ERR_SHAPE
    assert status(call, X, off, w, Y, ElemType.F32) == _ffi.QK_ERR_DTYPE
    many = weight((1025, 8, 64))
    assert status(call, X, fake((1026,), 4), many, fake((4, 8), 2), BF) == _ffi.QK_ERR_TOO_LARGE
    back = grouped_linear.launch_backward
    assert status(back, Y, off, w, X, BF, grad_bias=fake((64,), 2)) == _ffi.QK_ERR_SHAPE
    assert status(back, Y, off, w, X, BF, grad_bias=fake((3, 64), 2, strides=(0, 1))) == _ffi.QK_ERR_LAYOUT
    assert status(back, Y, off, w, X, BF, grad_bias=fake((3, 64), 2, strides=(32, 1))) == _ffi.QK_ERR_LAYOUT
    assert status(back, Y, off, w, X, BF, activation=Activation.Relu) == _ffi.QK_ERR_NULL


def test_extents():
    wide = weight((8, 1 << 26))
    assert status(linear.launch, fake((1, 1 << 26), 2), wide, fake((1, 8), 2), BF) == _ffi.QK_ERR_TOO_LARGE
    tall = weight((1 << 26, 32))
    assert status(linear.launch, fake((1, 32), 2), tall, fake((1, 1 << 26), 2), BF) == _ffi.QK_ERR_TOO_LARGE
    assert status(linear.launch_backward, fake((1, 1 << 26), 2), tall, fake((1, 32), 2), BF) == _ffi.QK_ERR_TOO_LARGE
    with pytest.raises(LaunchError):   # an unaligned x needs the workspace
        linear.launch(CLIENT, fake((20, 64), 2, addr=0x10002), weight(), fake((20, 64), 2), BF)


def test_null_arguments():
    x, v, p = _ffi.c_tensors(X, fake((64, 8), 4), fake((64, 2), 4))
    s = _ffi.c_scheme(Q4)
    lib = _ffi.lib()
    full = [x.ref(), v.ref(), p.ref(), s, None, None, 0, x.ref(), None, int(BF), None, 0, None]
    for i in (0, 1, 2, 3, 7):
        args = list(full)
        args[i] = None
        assert lib.qk_linear(*args) == _ffi.QK_ERR_NULL
    full = [x.ref(), v.ref(), p.ref(), s, 0, None, x.ref(), None, None, int(BF), None, 0, None]
    for i in (0, 1, 2, 3):
        args = list(full)
        args[i] = None
        assert lib.qk_linear_backward(*args) == _ffi.QK_ERR_NULL
    assert lib.qk_grouped_linear(x.ref(), None, v.ref(), p.ref(), s, None, None, 0, x.ref(), None, int(BF), None, 0, None) != _ffi.QK_OK
    assert lib.qk_linear_backward_workspace_bytes(None, v.ref(), s, 0, 0, None, int(BF)) == 0
    assert lib.qk_linear_workspace_bytes(None, v.ref(), s, int(BF)) == 0


def test_nothing_to_do_is_no_error():
    linear.launch(CLIENT, fake((0, 64), 2), weight(), fake((0, 64), 2), BF)
    linear.launch(CLIENT, X, weight((0, 64)), fake((4, 0), 2), BF)
    linear.launch_backward(CLIENT, fake((0, 64), 2), weight(), fake((0, 64), 2), BF)
    linear.launch_backward(CLIENT, Y, weight(), None, BF)
    grouped_linear.launch(CLIENT, fake((0, 64), 2), fake((4,), 4), weight((3, 64, 64)), fake((0, 64), 2), BF)


def test_workspace_sizes():
    g = fake((1000, 512), 2)
    w = weight((512, 256))
    plain = linear.backward_workspace_bytes(g, w, BF)
    assert plain == 0
    staged = linear.backward_workspace_bytes(g, w, BF, activation=Activation.Silu)
    assert staged >= 1000 * 512 * 2
    assert linear.backward_workspace_bytes(g, w, BF, activation=Activation.Silu, grad_pre=g) == 0
    assert linear.backward_workspace_bytes(g, w, BF, bias=True) % 256 == 0
    handle = MatmulInputHandleRef.quantized(fake((3, 512, 32), 4), fake((3, 512, 8), 4), (3, 512, 256), Q4)
    assert grouped_linear.backward_workspace_bytes(g, handle, BF, activation=Activation.Silu) >= 1000 * 512 * 2
