"""``grouped_linear``: the rows of each expert against the definition in 64 bits, ragged and empty experts included."""
import pytest
import torch

from cubek_b200 import ComputeClient, ElemType, QuantLevel, QuantScheme, QuantStore, QuantValue, grouped_linear
from cubek_b200.linear import Activation
from tests._linear import TORCH, H, Weight, check_backward, check_forward, filled, randn
from tests.test_gpu_linear import BF16, F16, FP4, Q4, Q8, no_device_error, workspace

pytestmark = pytest.mark.gpu


def offsets_of(counts, first=0, dtype=torch.int32):
    return torch.tensor([first] + [first + sum(counts[:i + 1]) for i in range(len(counts))], dtype=dtype, device="cuda")


def run(w: Weight, counts, rows, first=0, act=Activation.Identity, bias=False, residual=False, dtype=torch.int32, seed=3):
    """Forward and backward, all outputs checked expert by expert, rows outside the experts unchanged."""
    e, n, k = w.shape
    elem = w.elem
    x = (randn((rows, k), elem, seed).float() * (1.5 / k ** 0.5)).to(TORCH[elem])
    x[:first] = float("nan")           # rows of no expert are not even read into others
    x[first + sum(counts):] = float("nan")
    b = randn((e, n), elem, seed + 1) if bias else None
    r = randn((rows, n), elem, seed + 2) if residual else None
    off = offsets_of(counts, first, dtype)
    y, pre, gx, gp = filled((rows, n), elem), filled((rows, n), elem), filled((rows, k), elem), filled((rows, n), elem)
    gb = filled((e, n), elem)
    untouched = [t.clone() for t in (y, pre, gx, gp)]
    client, handle = ComputeClient.current(), w.handle()
    opt = lambda t: None if t is None else H(t)  # noqa: E731
    ws = workspace(grouped_linear.workspace_bytes(H(x), handle, elem))
    grouped_linear.launch(client, H(x), H(off), handle, H(y), elem, bias=opt(b), residual=opt(r), activation=act, pre=H(pre), workspace=H(ws))
    g = randn((rows, n), elem, seed + 3)
    ws = workspace(grouped_linear.backward_workspace_bytes(H(g), handle, elem, activation=act, bias=True, grad_pre=H(gp)))
    grouped_linear.launch_backward(client, H(g), H(off), handle, H(gx), elem, pre=H(pre), activation=act, grad_bias=H(gb), grad_pre=H(gp),
                                   workspace=H(ws))
    # the same through the staged dz
    gx2 = filled((rows, k), elem)
    ws = workspace(grouped_linear.backward_workspace_bytes(H(g), handle, elem, activation=act, bias=False))
    grouped_linear.launch_backward(client, H(g), H(off), handle, H(gx2), elem, pre=H(pre), activation=act, workspace=H(ws))
    lo = first
    for i, c in enumerate(counts):
        s = slice(lo, lo + c)
        lo += c
        check_forward(y[s], pre[s], x[s], w.value[i], elem, None if b is None else b[i], None if r is None else r[s], act)
        check_backward(gx[s], gb[i], gp[s], g[s], w.value[i], elem, pre[s], act)
        assert torch.equal(gx2[s].view(torch.int16), gx[s].view(torch.int16))
    for t, u in zip((y, pre, gx, gp), untouched):
        for s in (slice(0, first), slice(lo, rows)):
            assert torch.equal(t[s].view(torch.int16), u[s].view(torch.int16))
    no_device_error()


COUNTS = [[5], [0], [1, 1], [0, 7, 0], [3, 0, 0, 9, 1], [64, 128, 1, 0], [300, 2, 17, 129], [0, 0, 0, 0, 0, 0, 0, 40], [256, 256],
          [33] * 16]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("scheme,elem", [(Q4, BF16), (FP4, F16)], ids=["q4-bf16", "fp4-f16"])
def test_ragged(counts, scheme, elem):
    w = Weight((len(counts), 136, 160), scheme, elem, 1)
    run(w, counts, sum(counts), act=Activation.Silu, bias=True, residual=True)


@pytest.mark.parametrize("n,k", [(1, 4), (65, 68), (128, 64), (129, 300), (300, 1028)])
def test_sizes(n, k):
    scheme = QuantScheme(value=QuantValue.Q8F, level=QuantLevel.block([32]))
    w = Weight((4, n, k), scheme, BF16, 1)
    run(w, [10, 0, 70, 3], 90, first=2)


@pytest.mark.parametrize("scheme", [
    QuantScheme(value=QuantValue.Q8S), QuantScheme(value=QuantValue.Q2S, level=QuantLevel.block([16])),
    QuantScheme(value=QuantValue.E4M3, store=QuantStore.Native, level=QuantLevel.block([32, 32])),
    QuantScheme(value=QuantValue.E5M2, store=QuantStore.Native, level=QuantLevel.block([64])),
    QuantScheme(value=QuantValue.E2M1, level=QuantLevel.block([8]))])
@pytest.mark.parametrize("elem", [F16, BF16], ids=["f16", "bf16"])
def test_formats(scheme, elem):
    w = Weight((3, 96, 128), scheme, elem, 1)
    run(w, [2, 50, 9], 64, first=1, act=Activation.GeluTanh, bias=True, dtype=torch.int64)


def test_many_experts_few_rows():
    w = Weight((128, 64, 64), Q8, BF16, 1)
    counts = [1 if i % 5 == 0 else 0 for i in range(128)]
    run(w, counts, sum(counts), bias=True)


def test_one_expert_takes_all():
    w = Weight((8, 256, 512), Q4, BF16, 1)
    run(w, [0, 0, 0, 1500, 0, 0, 0, 0], 1500, act=Activation.Relu, bias=True)


def test_wrong_offsets_stay_inside_the_tensors():
    """Offsets past the rows, negative or descending: the rows they leave are computed, nothing else is touched."""
    w = Weight((3, 64, 64), Q4, BF16, 1)
    x = randn((20, 64), BF16, 2) * 0.2
    for off, spans in (([-5, 4, 400, 30], [(0, 4), (4, 20), None]), ([8, 2, 6, 6], [None, (2, 6), None])):
        y = filled((20, 64), BF16)
        before = y.clone()
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        grouped_linear.launch(ComputeClient.current(), H(x), H(o), w.handle(), H(y), BF16)
        seen = torch.zeros(20, dtype=torch.bool)
        for i, s in enumerate(spans):
            if s:
                check_forward(y[s[0]:s[1]], None, x[s[0]:s[1]], w.value[i], BF16)
                seen[s[0]:s[1]] = True
        assert torch.equal(y[~seen].view(torch.int16), before[~seen].view(torch.int16))
    no_device_error()


def test_expert_strides():
    """Experts that lie apart in memory, and one weight shared by all (stride 0)."""
    w = Weight((3, 64, 64), Q4, F16, 1)
    x = randn((30, 64), F16, 2) * 0.2
    off = offsets_of([10, 5, 15])
    for shared in (False, True):
        codes = torch.zeros(3, 2, 64, 8, dtype=torch.int32, device="cuda")
        codes[:, 1] = w.dcodes
        data = w.dcodes[:1].expand(3, 64, 8) if shared else codes[:, 1]
        scale = w.dscales[:1].expand(3, 64, 2) if shared else w.dscales
        y = filled((30, 64), F16)
        grouped_linear.launch(ComputeClient.current(), H(x), H(off), w.handle(data, scale), H(y), F16)
        for i, s in enumerate((slice(0, 10), slice(10, 15), slice(15, 30))):
            check_forward(y[s], None, x[s], w.value[0 if shared else i], F16)


def test_mixture_layer_run_together():
    """Tokens sorted by expert, up projection with activation, down projection, and the gradient back through both, replayed
    from a graph with other counts: the offsets are read on the device."""
    elem, e, hidden, inner, rows = BF16, 4, 128, 320, 96
    up, down = Weight((e, inner, hidden), Q4, elem, 1), Weight((e, hidden, inner), Q4, elem, 2)
    act = Activation.Silu
    x = randn((rows, hidden), elem, 3) * 0.1
    off = offsets_of([24, 24, 24, 24])
    h, pre, y = filled((rows, inner), elem), filled((rows, inner), elem), filled((rows, hidden), elem)
    g = randn((rows, hidden), elem, 4)
    gh, gx = filled((rows, inner), elem), filled((rows, hidden), elem)
    ws = workspace(grouped_linear.backward_workspace_bytes(H(gh), up.handle(), elem, activation=act))

    def step():
        c = ComputeClient.current()
        grouped_linear.launch(c, H(x), H(off), up.handle(), H(h), elem, activation=act, pre=H(pre))
        grouped_linear.launch(c, H(h), H(off), down.handle(), H(y), elem)
        grouped_linear.launch_backward(c, H(g), H(off), down.handle(), H(gh), elem)
        grouped_linear.launch_backward(c, H(gh), H(off), up.handle(), H(gx), elem, pre=H(pre), activation=act, workspace=H(ws))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for counts in ([10, 0, 80, 6], [96, 0, 0, 0], [1, 2, 3, 90]):
        off.copy_(offsets_of(counts))
        graph.replay()
        torch.cuda.synchronize()
        lo = 0
        for i, c in enumerate(counts):
            s = slice(lo, lo + c)
            lo += c
            check_forward(h[s], pre[s], x[s], up.value[i], elem, act=act)
            check_forward(y[s], None, h[s], down.value[i], elem)
            check_backward(gh[s], None, None, g[s], down.value[i], elem)
            check_backward(gx[s], None, None, gh[s], up.value[i], elem, pre[s], act)
    no_device_error()
