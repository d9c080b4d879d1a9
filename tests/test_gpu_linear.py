"""``linear``: products with quantized weights and their gradients against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from cubek_b200 import (ComputeClient, ElemType, QuantLevel, QuantParam, QuantScheme, QuantStore, QuantValue, dequantize, linear,
                        quantize)
from cubek_b200 import _ffi
from cubek_b200.linear import Activation
from cubek_b200.matmul_input import MatmulInputHandleRef
from tests._cases import all_value_stores, scheme_id
from tests._linear import TORCH, H, Weight, check_backward, check_forward, filled, randn

pytestmark = pytest.mark.gpu

F16, BF16 = ElemType.F16, ElemType.BF16
Q4 = QuantScheme(value=QuantValue.Q4S, level=QuantLevel.block([32]))
Q8 = QuantScheme(value=QuantValue.Q8S, level=QuantLevel.block([128]))
FP4 = QuantScheme(value=QuantValue.E2M1, store=QuantStore.Native, level=QuantLevel.block([16]))


def workspace(nbytes):
    """Scratch that starts as NaN in every float type: nothing may be read before it is written."""
    return torch.full((max(nbytes, 16),), 0xFF, dtype=torch.uint8, device="cuda")


def forward(w: Weight, x, bias=None, residual=None, act=Activation.Identity, keep=True, handle=None, y=None):
    n = w.shape[-2]
    y = filled((*x.shape[:-1], n), w.elem) if y is None else y
    pre = filled((*x.shape[:-1], n), w.elem) if keep else None
    handle = handle or w.handle()
    opt = lambda t: None if t is None else H(t)  # noqa: E731
    ws = workspace(linear.workspace_bytes(H(x), handle, w.elem))
    linear.launch(ComputeClient.current(), H(x), handle, H(y), w.elem, bias=opt(bias), residual=opt(residual), activation=act, pre=opt(pre),
                  workspace=H(ws))
    return y, pre


def backward(w: Weight, g, pre=None, act=Activation.Identity, bias=True, keep=True, handle=None, gx=None):
    n, k = w.shape[-2:]
    gx = filled((*g.shape[:-1], k), w.elem) if gx is None else gx
    gb = filled((n,), w.elem) if bias else None
    gp = filled(g.shape, w.elem) if keep else None
    handle = handle or w.handle()
    opt = lambda t: None if t is None else H(t)  # noqa: E731
    ws = workspace(linear.backward_workspace_bytes(H(g), handle, w.elem, activation=act, bias=bias, grad_pre=opt(gp)))
    linear.launch_backward(ComputeClient.current(), H(g), handle, H(gx), w.elem, pre=opt(pre), activation=act, grad_bias=opt(gb),
                           grad_pre=opt(gp), workspace=H(ws))
    return gx, gb, gp


def no_device_error():
    import ctypes

    flag = ctypes.c_int(0)
    _ffi.check(_ffi.lib().qk_device_error(ctypes.byref(flag)))
    assert flag.value == 0


def case(rows, n, k, scheme, elem, seed=1):
    w = Weight((n, k), scheme, elem, seed)
    x = (randn((rows, k), elem, seed + 1).float() * (1.5 / max(k, 1) ** 0.5)).to(TORCH[elem])
    return w, x


def schemes():
    for v, store in all_value_stores():
        for level in (QuantLevel.Tensor, QuantLevel.block([16]), QuantLevel.block([32]), QuantLevel.block([64, 48])):
            param = QuantParam.F32 if level.is_tensor or level.block_size.as_slice() == (16,) else QuantParam.BF16
            yield QuantScheme(value=v, store=store, level=level, param=param)


@pytest.mark.parametrize("elem", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("scheme", list(schemes()), ids=scheme_id)
def test_every_format(scheme, elem):
    """Every value, store and level, few and many rows, sizes that are no multiples of a tile."""
    for rows in (3, 70):
        w, x = case(rows, 136, 208, scheme, elem)
        y, pre = forward(w, x)
        check_forward(y, pre, x, w.value, elem)
        g = randn((rows, 136), elem, 5)
        gx, gb, gp = backward(w, g)
        check_backward(gx, gb, gp, g, w.value, elem)
    no_device_error()


ROWS = [1, 2, 5, 8, 9, 16, 17, 31, 33, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300, 700]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("scheme,elem", [(Q4, BF16), (Q8, F16)], ids=["q4-bf16", "q8-f16"])
def test_rows(rows, scheme, elem):
    w, x = case(rows, 320, 512, scheme, elem)
    bias, res = randn((320,), elem, 7), randn((rows, 320), elem, 8)
    y, pre = forward(w, x, bias, res, Activation.Silu)
    check_forward(y, pre, x, w.value, elem, bias, res, Activation.Silu)
    g = randn((rows, 320), elem, 9)
    gx, gb, _ = backward(w, g, pre, Activation.Silu, keep=False)
    check_backward(gx, gb, None, g, w.value, elem, pre, Activation.Silu)
    no_device_error()


SIZES = [(1, 4), (1, 64), (2, 8), (3, 20), (63, 60), (64, 64), (65, 68), (127, 128), (128, 132), (129, 260), (130, 1000), (257, 516),
         (1000, 72), (511, 2052), (24, 6000)]


@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("rows", [1, 20, 150])
def test_sizes(rows, n, k):
    scheme = QuantScheme(value=QuantValue.Q8F, level=QuantLevel.block([32]))
    w, x = case(rows, n, k, scheme, BF16)
    y, pre = forward(w, x, act=Activation.Relu)
    check_forward(y, pre, x, w.value, BF16, act=Activation.Relu)
    g = randn((rows, n), BF16, 3)
    gx, gb, gp = backward(w, g, pre, Activation.Relu)
    check_backward(gx, gb, gp, g, w.value, BF16, pre, Activation.Relu)
    no_device_error()


@pytest.mark.parametrize("k", [1, 7, 33, 100, 255, 1025])
@pytest.mark.parametrize("value", [QuantValue.Q8S, QuantValue.E4M3])
@pytest.mark.parametrize("rows", [2, 40])
def test_odd_row_lengths(rows, value, k):
    """One-byte codes may have rows of any length: neither codes nor activations are aligned."""
    scheme = QuantScheme(value=value, store=QuantStore.Native)
    w, x = case(rows, 37, k, scheme, F16)
    y, pre = forward(w, x)
    check_forward(y, pre, x, w.value, F16)
    g = randn((rows, 37), F16, 4)
    gx, gb, gp = backward(w, g)
    check_backward(gx, gb, gp, g, w.value, F16)
    no_device_error()


@pytest.mark.parametrize("act", list(Activation))
@pytest.mark.parametrize("elem", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("bias,residual,keep", [(False, False, False), (True, False, True), (False, True, False), (True, True, True)])
@pytest.mark.parametrize("rows", [4, 90])
def test_epilogues(act, elem, bias, residual, keep, rows):
    w, x = case(rows, 161, 256, FP4, elem)
    x = x * 3
    b = randn((161,), elem, 2) if bias else None
    r = randn((rows, 161), elem, 3) if residual else None
    y, pre = forward(w, x, b, r, act, keep)
    check_forward(y, pre, x, w.value, elem, b, r, act)
    if keep:
        g = randn((rows, 161), elem, 4)
        gx, gb, gp = backward(w, g, pre, act, keep=not residual)
        check_backward(gx, gb, gp, g, w.value, elem, pre, act)
    no_device_error()


def test_gradient_against_differences():
    """The gradient of sum(g * y) along random directions, by central differences of the definition in 64 bits."""
    for act in Activation:
        if act == Activation.Relu:
            continue  # not differentiable at 0: its slope is tested exactly above
        w, x = case(33, 96, 128, Q4, BF16)
        b, g = randn((96,), BF16, 2), randn((33, 96), BF16, 3)
        from tests._linear import act64

        _, pre = forward(w, x, b, None, act)
        gx, gb, _ = backward(w, g, pre, act)
        f = lambda xs, bs: float((g.double() * act64(xs @ w.value.mT + bs, act)).sum())  # noqa: E731
        for seed in range(3):
            dx, db = randn((33, 128), BF16, 10 + seed).double(), randn((96,), BF16, 20 + seed).double()
            h = 1e-4
            slope = (f(x.double() + h * dx, b.double() + h * db) - f(x.double() - h * dx, b.double() - h * db)) / (2 * h)
            got = float((gx.double() * dx).sum() + (gb.double() * db).sum())
            # bf16 pre, dz and outputs: each term is off by at most about 3 half steps (slopes of second order included)
            size = float((gx.double() * dx).abs().sum() + (gb.double() * db).abs().sum())
            assert abs(got - slope) <= 4 * 2.0 ** -8 * size, (act, got, slope)


@pytest.mark.parametrize("rows", [1, 6, 100])
def test_strides(rows):
    """Column slices of wider matrices, padded codes, scales of other strides; what lies between is left alone."""
    n, k = 144, 192
    w, _ = case(rows, n, k, Q4, BF16)
    for pad in (8, 3):  # rows that start on 16 bytes, and on 2
        wide = randn((rows, k + 2 * pad), BF16, 5) * 0.1
        x = wide[:, pad:pad + k]
        out = filled((rows, n + pad + 5), BF16)
        resw = randn((rows, n + 11), BF16, 6)
        codes = torch.zeros(n, k // 8 + pad, dtype=torch.int32, device="cuda")
        codes[:, :k // 8] = w.dcodes
        scales = torch.zeros(k // 32, n, dtype=torch.float32, device="cuda").t()
        scales.copy_(w.dscales)
        handle = w.handle(codes[:, :k // 8], scales)
        before = out.clone()
        y, _ = forward(w, x, None, resw[:, 4:4 + n], Activation.Identity, True, handle, out[:, pad:pad + n])
        check_forward(y, None, x, w.value, BF16, None, resw[:, 4:4 + n])
        assert torch.equal(out[:, :pad].view(torch.int16), before[:, :pad].view(torch.int16))
        assert torch.equal(out[:, pad + n:].view(torch.int16), before[:, pad + n:].view(torch.int16))
        gw = randn((rows, n + 2 * pad), BF16, 7)
        gout = filled((rows, k + pad), BF16)
        gx, gb, gp = backward(w, gw[:, pad:pad + n], handle=handle, gx=gout[:, pad:pad + k])
        check_backward(gx, gb, gp, gw[:, pad:pad + n], w.value, BF16)
    no_device_error()


def test_leading_dims_and_in_place_residual():
    w, _ = case(1, 128, 64, Q4, F16)
    x = randn((3, 5, 64), F16, 3) * 0.2
    r = randn((3, 5, 128), F16, 4)
    y, pre = forward(w, x)
    check_forward(y.view(15, 128), pre.view(15, 128), x.view(15, 64), w.value, F16)
    out = r.clone()
    forward(w, x, residual=out, y=out, keep=False)
    check_forward(out.view(15, 128), None, x.view(15, 64), w.value, F16, None, r.view(15, 128))
    v = randn((64,), F16, 5)   # a single vector
    y1, _ = forward(w, v)
    check_forward(y1[None], None, v[None], w.value, F16)


def test_empty_sizes():
    """No rows, no features, an empty sum: act(bias) + residual; gradients of nothing are zero."""
    for rows, n, k in [(0, 16, 32), (4, 0, 32), (4, 16, 0), (40, 16, 0), (0, 0, 0)]:
        scheme = QuantScheme(value=QuantValue.Q8S)
        codes, scales = np.zeros((n, k // 4), np.uint32), np.ones(1, np.float32)
        w = Weight((n, k), scheme, BF16, 1, codes, scales)
        x, b, r = randn((rows, k), BF16, 2), randn((n,), BF16, 3), randn((rows, n), BF16, 4)
        y, pre = forward(w, x, b, r, Activation.Gelu)
        check_forward(y, pre, x, w.value, BF16, b, r, Activation.Gelu)
        g = randn((rows, n), BF16, 5)
        gx, gb, gp = backward(w, g, pre, Activation.Gelu)
        check_backward(gx, gb, gp, g, w.value, BF16, pre, Activation.Gelu)


@pytest.mark.parametrize("rows", [2, 40])
def test_infinities_and_nan_stay_in_their_rows(rows):
    """A NaN or infinity of x reaches its own row, one of a scale its own feature; padding never turns into one."""
    w, x = case(rows, 72, 72, Q4, BF16)
    x[0, 5], x[1, 71] = float("nan"), float("inf")
    y, _ = forward(w, x)
    want = x.double() @ w.value.mT
    assert torch.equal(torch.isnan(y[0]), torch.ones(72, dtype=torch.bool, device="cuda"))
    assert torch.equal(y[1].double().isinf() | y[1].isnan(), want[1].isinf() | want[1].isnan())
    check_forward(y[2:], None, x[2:], w.value, BF16)
    scales = w.scales.copy()
    scales[7, 2] = np.inf       # the block that ends inside the last tile
    codes = w.codes.copy()
    codes[7, 8] = 0x11111111    # no zero code in it: inf, not inf * 0
    v = Weight((72, 72), Q4, BF16, 1, codes, scales)
    xp = x.abs().nan_to_num(1.0, posinf=1.0)
    y, _ = forward(v, xp)
    assert bool((y[:, 7] == float("inf")).all())
    keep = [i for i in range(72) if i != 7]
    check_forward(y[:, keep], None, xp, v.value[keep], BF16)
    no_device_error()


def test_zero_and_far_scales():
    """Zero blocks, and scales whose products are subnormal or overflow in f16, as dequantize rounds them."""
    scheme = QuantScheme(value=QuantValue.Q8S, level=QuantLevel.block([32]))
    w, x = case(20, 64, 96, scheme, F16)
    scales = w.scales.copy()
    scales[3] = 0.0
    scales[4] = 2.0 ** -20
    scales[5] = 3e-8
    v = Weight((64, 96), scheme, F16, 1, w.codes, scales)
    y, _ = forward(v, x)
    check_forward(y, None, x, v.value, F16)
    assert bool((y[:, 3] == 0).all())


def test_repeated_calls_give_the_same_bits():
    w, x = case(300, 400, 1000, Q8, BF16)
    g = randn((300, 400), BF16, 2)
    first = None
    for _ in range(3):
        y, pre = forward(w, x, act=Activation.GeluTanh)
        out = (y, pre, *backward(w, g, pre, Activation.GeluTanh))
        if first is None:
            first = [t.clone() for t in out]
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(first, out))


def test_larger_problem():
    """Sizes of the library's weight set."""
    for rows in (1, 16, 333):
        w, x = case(rows, 1024, 4096, Q8, BF16)
        y, pre = forward(w, x)
        check_forward(y, pre, x, w.value, BF16)
        g = randn((rows, 1024), BF16, 2)
        gx, gb, gp = backward(w, g)
        check_backward(gx, gb, gp, g, w.value, BF16)
    no_device_error()


def test_rows_beyond_32_bit_offsets():
    """Outputs of more than 2^31 elements."""
    rows, n, k = 70000, 32768, 16
    scheme = QuantScheme(value=QuantValue.Q4S, level=QuantLevel.block([16]))
    w, x = case(rows, n, k, scheme, F16)
    y, _ = forward(w, x, keep=False)
    at = torch.tensor([0, 1, 65535, 65536, 69999], device="cuda")
    check_forward(y[at], None, x[at], w.value, F16)
    gx, gb, _ = backward(w, y, keep=False)
    check_backward(gx[at], None, None, y[at], w.value, F16)


def test_capture_and_replay_on_another_stream():
    """Two graphs that share one workspace, replayed in turn on new data."""
    act = Activation.Silu
    w, x = case(70, 200, 264, Q4, BF16)
    n = 200
    y, pre, gx, gb = filled((70, n), BF16), filled((70, n), BF16), filled((70, 264), BF16), filled((n,), BF16)
    g = randn((70, n), BF16, 3)
    handle = w.handle()
    ws = workspace(max(linear.workspace_bytes(H(x), handle, BF16), linear.backward_workspace_bytes(H(g), handle, BF16, activation=act, bias=True)))

    def fwd():
        linear.launch(ComputeClient.current(), H(x), handle, H(y), BF16, activation=act, pre=H(pre), workspace=H(ws))

    def bwd():
        linear.launch_backward(ComputeClient.current(), H(g), handle, H(gx), BF16, pre=H(pre), activation=act, grad_bias=H(gb), workspace=H(ws))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fwd()
        bwd()
    torch.cuda.synchronize()
    graphs = []
    for call in (fwd, bwd):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append(graph)
    for seed in (11, 12):
        x.copy_(randn((70, 264), BF16, seed).float() * 0.1)
        g.copy_(randn((70, n), BF16, seed + 5))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        check_forward(y, pre, x, w.value, BF16, act=act)
        check_backward(gx, gb, None, g, w.value, BF16, pre, act)


def test_quantize_linear_backward_run_together():
    """A block as a model has it: weights quantized by the library, up projection, activation, down projection added to the
    residual stream, and the gradient back through both; each step against the definition on the step's own inputs."""
    elem, hidden, inner, rows = BF16, 256, 704, 50
    client = ComputeClient.current()
    weights = []
    for shape, seed in (((inner, hidden), 1), ((hidden, inner), 2)):
        full = randn(shape, elem, seed) * 0.05
        codes = torch.empty(Q4.packed_shape(shape), dtype=torch.int32, device="cuda")
        scales = torch.empty(Q4.scales_shape(shape), dtype=torch.float32, device="cuda")
        quantize.launch_dynamic(client, H(full), H(codes), H(scales), Q4, elem)
        restored = torch.empty_like(full)
        dequantize.launch_ref(client, H(codes), H(restored), H(scales), Q4, elem)
        handle = MatmulInputHandleRef.quantized(H(codes), H(scales), shape, Q4)
        weights.append((handle, restored.double(), codes, scales))
    (up, up64, *_), (down, down64, *_) = weights
    x, b = randn((rows, hidden), elem, 3), randn((inner,), elem, 4)
    h, pre, y = filled((rows, inner), elem), filled((rows, inner), elem), filled((rows, hidden), elem)
    linear.launch(client, H(x), up, H(h), elem, bias=H(b), activation=Activation.Gelu, pre=H(pre))
    linear.launch(client, H(h), down, H(y), elem, residual=H(x))
    check_forward(h, pre, x, up64, elem, b, None, Activation.Gelu)
    check_forward(y, None, h, down64, elem, None, x)
    g = randn((rows, hidden), elem, 5)
    gh, gx, gb = filled((rows, inner), elem), filled((rows, hidden), elem), filled((inner,), elem)
    linear.launch_backward(client, H(g), down, H(gh), elem)
    ws = workspace(linear.backward_workspace_bytes(H(gh), up, elem, activation=Activation.Gelu, bias=True))
    linear.launch_backward(client, H(gh), up, H(gx), elem, pre=H(pre), activation=Activation.Gelu, grad_bias=H(gb), workspace=H(ws))
    check_backward(gh, None, None, g, down64, elem)
    check_backward(gx, gb, None, gh, up64, elem, pre, Activation.Gelu)
