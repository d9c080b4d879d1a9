"""``linear`` and ``grouped_linear`` with many rows: tiles of 512 rows, every format, sizes around their edges, concurrent calls."""
import pytest
import torch

from cubek_b200 import ComputeClient, QuantLevel, QuantParam, QuantScheme, QuantValue, grouped_linear, linear
from cubek_b200.linear import Activation
from tests._cases import scheme_id
from tests._linear import H, Weight, check_backward, check_forward, filled, randn
from tests.test_gpu_grouped_linear import offsets_of, run
from tests.test_gpu_linear import BF16, F16, Q4, Q8, backward, case, forward, no_device_error, schemes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("elem", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("scheme", list(schemes()), ids=scheme_id)
def test_every_format(scheme, elem):
    """K of whole steps and of none (576, 528); rows of outputs on 32 and on 16 bytes."""
    for n, k in ((320, 576), (136, 528)):
        w, x = case(530, n, k, scheme, elem)
        bias = randn((n,), elem, 6)
        y, pre = forward(w, x, bias, act=Activation.Silu)
        check_forward(y, pre, x, w.value, elem, bias, act=Activation.Silu)
        g = randn((530, n), elem, 5)
        gx, gb, gp = backward(w, g, pre, Activation.Silu)
        check_backward(gx, gb, gp, g, w.value, elem, pre, Activation.Silu)
    no_device_error()


@pytest.mark.parametrize("rows", [159, 160, 161, 255, 256, 257, 288, 384, 385, 511, 512, 513, 640, 769, 1025, 1600])
@pytest.mark.parametrize("n", [16, 129, 384])
def test_rows(rows, n):
    w, x = case(rows, n, 320, Q4, BF16)
    res = randn((rows, n), BF16, 8)
    y, pre = forward(w, x, None, res, Activation.Relu)
    check_forward(y, pre, x, w.value, BF16, None, res, Activation.Relu)
    g = randn((rows, n), BF16, 9)
    gx, gb, _ = backward(w, g, pre, Activation.Relu, keep=False)
    check_backward(gx, gb, None, g, w.value, BF16, pre, Activation.Relu)
    no_device_error()


@pytest.mark.parametrize("param", list(QuantParam))
@pytest.mark.parametrize("level", [QuantLevel.block([8]), QuantLevel.block([24]), QuantLevel.block([16]), QuantLevel.block([255, 64]),
                                   QuantLevel.block([3, 128]), QuantLevel.block([248])], ids=lambda v: "x".join(map(str, v.block_size.as_slice())))
@pytest.mark.parametrize("rows", [3, 50, 300])
def test_blocks(rows, level, param):
    """Block extents that divide nothing, scales of every type."""
    scheme = QuantScheme(value=QuantValue.Q8S, level=level, param=param)
    w, x = case(rows, 272, 448, scheme, BF16)
    y, pre = forward(w, x)
    check_forward(y, pre, x, w.value, BF16)
    g = randn((rows, 272), BF16, 9)
    gx, gb, gp = backward(w, g)
    check_backward(gx, gb, gp, g, w.value, BF16)
    no_device_error()


@pytest.mark.parametrize("counts", [[700, 0, 300, 129], [512, 513, 1, 511], [160] * 6, [0, 1300], [2000, 1, 1, 1]],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("n,k", [(136, 160), (200, 1028), (33, 64)])
def test_experts(counts, n, k):
    scheme = QuantScheme(value=QuantValue.Q8F, level=QuantLevel.block([32]), param=QuantParam.F16)
    w = Weight((len(counts), n, k), scheme, BF16, 1)
    run(w, counts, sum(counts) + 5, first=3, act=Activation.GeluTanh, bias=True, residual=True)


def test_most_experts():
    """1024 experts, few and many rows."""
    w = Weight((1024, 16, 64), QuantScheme(value=QuantValue.Q4S, level=QuantLevel.block([32])), F16, 1)
    for per in (1, 20):
        counts = [(i * 7) % (2 * per + 1) for i in range(1024)]
        x = randn((sum(counts), 64), F16, 2) * 0.2
        off = offsets_of(counts)
        y = filled((sum(counts), 16), F16)
        grouped_linear.launch(ComputeClient.current(), H(x), H(off), w.handle(), H(y), F16)
        e = torch.repeat_interleave(torch.arange(1024, device="cuda"), torch.tensor(counts, device="cuda"))
        want = torch.bmm(w.value[e], x.double()[:, :, None])[:, :, 0]
        tol = (64 + 16) * 2.0 ** -23 * torch.bmm(w.value[e].abs(), x.double().abs()[:, :, None])[:, :, 0]
        assert bool(((y.double() - want).abs() <= 1.001 * tol + 2.0 ** -11 * want.abs() + 2.0 ** -25).all())
    no_device_error()


def test_one_expert_has_all_rows_of_many():
    """The average says few rows, one expert has them all."""
    w = Weight((64, 80, 96), Q4, BF16, 1)
    run(w, [0] * 40 + [400] + [0] * 23, 400, bias=True)


def test_two_streams_at_once():
    """Calls of every kernel overlap on two streams; each has buffers of its own."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    jobs = []
    for i, rows in enumerate((900, 40, 4, 700)):
        for s in (0, 1):
            w, x = case(rows, 528, 1024, Q8 if i % 2 else Q4, BF16, seed=10 * i + s)
            g = randn((rows, 528), BF16, 3)
            jobs.append((s, w, x, g, filled((rows, 528), BF16), filled((rows, 1024), BF16)))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, w, x, g, y, gx in jobs:
            client = ComputeClient(0, streams[s].cuda_stream)
            linear.launch(client, H(x), w.handle(), H(y), BF16)
            linear.launch_backward(client, H(g), w.handle(), H(gx), BF16)
    torch.cuda.synchronize()
    for s, w, x, g, y, gx in jobs:
        check_forward(y, None, x, w.value, BF16)
        check_backward(gx, None, None, g, w.value, BF16)
    no_device_error()


def test_nan_and_infinity():
    """A NaN row of x reaches its own row, an infinite scale its own feature, with padding in every direction."""
    w, x = case(300, 80, 96, Q4, BF16)
    x[5, 95] = float("nan")
    y, _ = forward(w, x)
    assert bool(y[5].isnan().all())
    keep = [i for i in range(300) if i != 5]
    check_forward(y[keep], None, x[keep], w.value, BF16)
    scales, codes = w.scales.copy(), w.codes.copy()
    scales[79, 2] = float("inf")
    codes[79, 8:] = 0x11111111
    v = Weight((80, 96), Q4, BF16, 1, codes, scales)
    xp = x.abs().nan_to_num(1.0)
    y, _ = forward(v, xp)
    assert bool((y[:, 79] == float("inf")).all())
    check_forward(y[:, :79], None, xp, v.value[:79], BF16)


def test_captured_with_other_row_counts():
    """Graphs of the pair kernel replayed on new data, twice each, in turn."""
    w, x = case(600, 256, 256, Q8, F16)
    y, gx = filled((600, 256), F16), filled((600, 256), F16)
    g = randn((600, 256), F16, 2)
    forward(w, x)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        linear.launch(ComputeClient.current(), H(x), w.handle(), H(y), F16)
    with torch.cuda.graph(graphs[1]):
        linear.launch_backward(ComputeClient.current(), H(y), w.handle(), H(gx), F16)
    for seed in (1, 2):
        x.copy_(randn((600, 256), F16, seed) * 0.05)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        check_forward(y, None, x, w.value, F16)
        check_backward(gx, None, None, y, w.value, F16)
