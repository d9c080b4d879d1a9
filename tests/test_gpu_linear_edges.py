"""``linear`` and ``grouped_linear`` at values and sizes far from the ordinary ones."""
import numpy as np
import pytest
import torch

from cubek_b200 import ComputeClient, QuantLevel, QuantParam, QuantScheme, QuantStore, QuantValue, grouped_linear, linear
from cubek_b200.linear import Activation
from cubek_b200.matmul_input import MatmulInputHandleRef
from tests._linear import H, Weight, check_backward, check_forward, filled, randn
from tests.test_gpu_linear import BF16, F16, backward, forward, no_device_error

pytestmark = pytest.mark.gpu

ROWS = [3, 40, 300]   # one for each kernel


def q8(n, k, store, elem, scales, low=-127, high=128, param=QuantParam.F32, seed=1):
    """A weight of random 8-bit codes in blocks of 32, one scale for each row."""
    scheme = QuantScheme(value=QuantValue.Q8S, store=store, level=QuantLevel.block([32]), param=param)
    codes = np.random.default_rng(seed).integers(low, high, (n, k)).astype(np.int8)
    codes[:, :3] = [1, 0, -1] if low < 0 else 1
    full = np.repeat(np.resize(np.asarray(scales, np.float32), n)[:, None], k // 32, 1)
    return Weight((n, k), scheme, elem, seed, codes.view(np.uint32) if store == QuantStore.U32 else codes, np.ascontiguousarray(full))


@pytest.mark.parametrize("store", [QuantStore.U32, QuantStore.Native])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("k", [192, 160])
def test_large_scales_of_8_bit_codes(rows, store, k):
    """Scales of which no multiple of 2^15 is a finite f32: the weight is code times scale all the same, and zero for code 0."""
    w = q8(80, k, store, BF16, [2e34, -2e34, 1.0, 1.04e34, -2.0 ** 116])
    assert bool(w.value.isfinite().all())
    x = (randn((rows, k), BF16, 2).float() * 0.1).bfloat16()
    x[:, :3] = 1.0
    y, pre = forward(w, x)
    check_forward(y, pre, x, w.value, BF16)
    g = (randn((rows, 80), BF16, 3).float() * 0.1).bfloat16()
    gx, gb, gp = backward(w, g)
    check_backward(gx, gb, gp, g, w.value, BF16)
    no_device_error()


@pytest.mark.parametrize("store", [QuantStore.U32, QuantStore.Native])
@pytest.mark.parametrize("rows", ROWS)
def test_largest_scale_of_8_bit_codes(rows, store):
    """The largest bf16 as a scale: codes 1, 0 and -1 stay finite."""
    w = q8(72, 64, store, BF16, [float(torch.finfo(torch.bfloat16).max)], -1, 2)
    x = (randn((rows, 64), BF16, 2).float() * 2.0 ** -10).bfloat16()
    y, pre = forward(w, x)
    check_forward(y, pre, x, w.value, BF16)
    assert bool(y.isfinite().all())
    g = (randn((rows, 72), BF16, 3).float() * 2.0 ** -10).bfloat16()
    gx, gb, gp = backward(w, g)
    check_backward(gx, gb, gp, g, w.value, BF16)


@pytest.mark.parametrize("elem,scale", [(BF16, float("inf")), (BF16, float("-inf")), (F16, float("inf")), (F16, 7e4), (F16, -1e3)])
@pytest.mark.parametrize("rows", ROWS)
def test_overflowing_scales_of_8_bit_codes(rows, elem, scale):
    """Infinite scales, scales that round to an infinite f16, and products that do: infinities of the code's sign."""
    w = q8(64, 64, QuantStore.U32, elem, [1.0], 1, 128)
    scales, codes = w.scales.copy(), w.codes.copy()
    scales[5] = scale
    codes[5] = 0x7F7F7F7F if abs(scale) == 1e3 else codes[5]   # 127 * 1000 is past the largest f16
    codes[9, 3] = 0x01000101   # a zero code: 0 * inf is no number, as dequantize has it
    scales[9] = scale
    v = Weight((64, 64), w.scheme, elem, 1, codes, scales)
    x = (randn((rows, 64), elem, 2).float().abs() * 0.01 + 0.01).to(torch.float16 if elem == F16 else torch.bfloat16)
    y, _ = forward(v, x)
    assert bool((y[:, 5] == (float("inf") if scale > 0 else float("-inf"))).all())
    if abs(scale) != 1e3:
        assert bool(v.value[9].isnan().any()) and bool(y[:, 9].isnan().all())
    keep = [i for i in range(64) if i not in (5, 9)]
    check_forward(y[:, keep], None, x, v.value[keep], elem)
    no_device_error()


@pytest.mark.parametrize("rows,n,k", [(4, 0, 32), (40, 0, 64), (300, 0, 64), (0, 16, 32), (4, 16, 0)])
def test_empty_sizes_with_the_workspace_that_is_asked_for(rows, n, k):
    """What the queries call enough is enough: nothing at all where they say zero."""
    scheme = QuantScheme(value=QuantValue.Q8S)
    w = Weight((n, k), scheme, BF16, 1, np.zeros((n, k // 4), np.uint32), np.ones(1, np.float32))
    g, pre = randn((rows, n), BF16, 2), randn((rows, n), BF16, 3)
    gx, gb = filled((rows, k), BF16), filled((n,), BF16)
    size = linear.backward_workspace_bytes(H(g), w.handle(), BF16, activation=Activation.Gelu, bias=True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
    linear.launch_backward(ComputeClient.current(), H(g), w.handle(), H(gx), BF16, pre=H(pre), activation=Activation.Gelu, grad_bias=H(gb),
                           workspace=None if ws is None else H(ws))
    check_backward(gx, gb, None, g, w.value, BF16, pre, Activation.Gelu)


@pytest.fixture
def released():
    """Large buffers go back to the device after the test."""
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n", [1, 8])
def test_most_rows(n, released):
    """2^31 - 512 rows, the most that are taken: the last ones are as right as the first."""
    rows, k = 2 ** 31 - 512, 8
    w = Weight((n, k), QuantScheme(value=QuantValue.Q8S, store=QuantStore.Native), BF16, 1)
    at = torch.tensor([0, 1, 511, 512, 2 ** 30 + 5, rows - 513, rows - 2, rows - 1], device="cuda")
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[at] = randn((8, k), BF16, 2)
    y = torch.full((rows, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    linear.launch(ComputeClient.current(), H(x), w.handle(), H(y), BF16)
    check_forward(y[at], None, x[at], w.value, BF16)
    assert bool((y[2 ** 30 + 6:2 ** 30 + 600] == 0).all()) and bool((y[-500:-2] == 0).all())
    if n == 8:   # rows of one element start on no 16 bytes: their gradient would copy them
        gx = torch.full((rows, k), float("nan"), dtype=torch.bfloat16, device="cuda")
        linear.launch_backward(ComputeClient.current(), H(y), w.handle(), H(gx), BF16)
        check_backward(gx[at], None, None, y[at], w.value, BF16)
    no_device_error()


@pytest.mark.parametrize("rows", [20, 60, 1000])
def test_offsets_that_overlap(rows):
    """Descending offsets that name rows twice: the first expert has them, whatever the timing."""
    w = Weight((5, 72, 96), QuantScheme(value=QuantValue.Q4S, level=QuantLevel.block([32])), BF16, 1)
    x = (randn((rows, 96), BF16, 2).float() * 0.2).bfloat16()
    half = rows // 2
    off = torch.tensor([0, half, 0, half + 5, 3, rows], dtype=torch.int32, device="cuda")
    owner = [(0, 0, half), (2, half, half + 5), (4, half + 5, rows)]   # expert, its rows
    for _ in range(3):
        y = filled((rows, 72), BF16)
        grouped_linear.launch(ComputeClient.current(), H(x), H(off), w.handle(), H(y), BF16)
        for e, lo, hi in owner:
            check_forward(y[lo:hi], None, x[lo:hi], w.value[e], BF16)
    no_device_error()


def test_a_sum_of_the_longest_extent(released):
    """2^26 - 1 terms on the path of unaligned rows of codes, where a step takes longest: no wait may end before the sum does."""
    rows, n, k = 160, 16, (1 << 26) - 1
    scheme = QuantScheme(value=QuantValue.Q8S, store=QuantStore.Native)
    codes = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    scale = torch.full((1,), 0.5, device="cuda")
    x = torch.zeros(rows, k + 1, dtype=torch.bfloat16, device="cuda")[:, :k]
    at = torch.tensor([0, 1, 63, 64, (1 << 25) + 7, k - 1], device="cuda")
    codes[:, at] = torch.randint(-127, 128, (n, 6), device="cuda", dtype=torch.int8)
    x[:, at] = randn((rows, 6), BF16, 3)
    y = filled((rows, n), BF16)
    linear.launch(ComputeClient.current(), H(x), MatmulInputHandleRef.quantized(H(codes), H(scale), (n, k), scheme), H(y), BF16)
    torch.cuda.synchronize()
    no_device_error()
    check_forward(y, None, x[:, at], codes[:, at].double() * 0.5, BF16)


@pytest.mark.parametrize("rows", [160, 333, 700])
@pytest.mark.parametrize("n", [72, 264])
def test_few_tiles_and_a_long_sum(rows, n):
    """Many rows of few features: tiles that fill little of the machine, whose contraction is split instead."""
    k = 16384
    w = Weight((n, k), QuantScheme(value=QuantValue.Q4S, level=QuantLevel.block([32])), BF16, 1)
    x = (randn((rows, k), BF16, 2).float() * 0.01).bfloat16()
    bias = randn((n,), BF16, 3)
    y, pre = forward(w, x, bias, act=Activation.Silu)
    check_forward(y, pre, x, w.value, BF16, bias, act=Activation.Silu)
    v = Weight((k, n), QuantScheme(value=QuantValue.Q4S, level=QuantLevel.block([8])), BF16, 1)
    g = (randn((rows, k), BF16, 4).float() * 0.01).bfloat16()
    gx, gb, gp = backward(v, g)
    check_backward(gx, gb, gp, g, v.value, BF16)
    no_device_error()


def test_few_tiles_of_experts_and_a_long_sum():
    w = Weight((3, 72, 16384), QuantScheme(value=QuantValue.Q4S, level=QuantLevel.block([32])), BF16, 1)
    counts = [200, 0, 300]
    x = (randn((500, 16384), BF16, 2).float() * 0.01).bfloat16()
    off = torch.tensor([0, 200, 200, 500], dtype=torch.int32, device="cuda")
    y = filled((500, 72), BF16)
    grouped_linear.launch(ComputeClient.current(), H(x), H(off), w.handle(), H(y), BF16)
    lo = 0
    for e, c in enumerate(counts):
        check_forward(y[lo:lo + c], None, x[lo:lo + c], w.value[e], BF16)
        lo += c
    no_device_error()


@pytest.mark.parametrize("act", [Activation.Gelu, Activation.GeluTanh, Activation.Silu])
def test_slopes_at_far_values(act):
    """Far from zero the slope is one or zero, also where squares and cubes of the pre-activation are no finite f32."""
    w = Weight((64, 64), QuantScheme(value=QuantValue.Q8S), BF16, 1)
    far = torch.tensor([1e3, 1e10, 1e13, 1.7e19, 2e19, 1e20, 1e30, 3e38], device="cuda").bfloat16()
    pre = torch.cat([far, -far]).repeat(4).expand(20, 64).contiguous()
    g = randn((20, 64), BF16, 2)
    _, gb, gp = backward(w, g, pre, act)
    assert torch.equal(gp, torch.where(pre > 0, g, torch.zeros_like(g)))
    want = torch.where(pre > 0, g, torch.zeros_like(g)).double()
    assert bool(((gb.double() - want.sum(0)).abs() <= 36 * 2.0 ** -23 * want.abs().sum(0) * 1.01 + 2.0 ** -8 * want.sum(0).abs()).all())
    y = torch.zeros(20, 64, dtype=torch.bfloat16, device="cuda")
    bias = pre[0].contiguous()
    out, _ = forward(w, y, bias, act=act)
    assert torch.equal(out, torch.where(pre > 0, pre, torch.zeros_like(pre)))


@pytest.mark.parametrize("n", [64, 37])
def test_relu_passes_nothing_where_it_is_flat(n):
    """An infinite or undefined incoming gradient (an overflown loss scale) stays out of the places where ReLU is flat."""
    w = Weight((n, 64), QuantScheme(value=QuantValue.Q8S), F16, 1)
    pre, g = randn((50, n), F16, 2), randn((50, n), F16, 3)
    flat = ~(pre > 0)
    flat[:, 0], pre[:, 0] = True, 0.0
    g = torch.where(flat & (torch.arange(n, device="cuda") % 3 == 0), torch.full_like(g, float("inf")), g)
    g = torch.where(flat & (torch.arange(n, device="cuda") % 3 == 1), torch.full_like(g, float("nan")), g)
    gx, gb, gp = backward(w, g, pre, Activation.Relu)
    clean = torch.where(flat, torch.zeros_like(g), g)
    check_backward(gx, gb, gp, clean, w.value, F16, pre, Activation.Relu)


def test_most_experts_with_unaligned_codes():
    """1024 experts on the tiles for many rows, with rows of 8-bit codes that start anywhere: the most shared memory a call takes."""
    e, n, k = 1024, 16, 33
    scheme = QuantScheme(value=QuantValue.Q8S, store=QuantStore.Native, level=QuantLevel.block([8]))
    w = Weight((e, n, k), scheme, BF16, 1)
    counts = torch.tensor([(i * 37) % 321 for i in range(e)])
    rows = int(counts.sum())
    off = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32).cuda()
    x = randn((rows, 40), BF16, 2)[:, :k]
    y = filled((rows, n), BF16)
    grouped_linear.launch(ComputeClient.current(), H(x), H(off), w.handle(), H(y), BF16)
    owner = torch.repeat_interleave(torch.arange(e), counts).cuda()
    x64 = x.double()[:, :, None]
    want = torch.bmm(w.value[owner], x64)[:, :, 0]
    tol = (k + 16) * 2.0 ** -23 * torch.bmm(w.value[owner].abs(), x64.abs())[:, :, 0]
    assert bool(((y.double() - want).abs() <= 1.01 * tol + 2.0 ** -8 * want.abs() + 2.0 ** -134).all())
    no_device_error()
