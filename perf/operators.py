"""The products with quantized weights, as cases to measure and to compare.

Two operators, each with its gradient:

* ``linear``   y = act(x W^T + b) + r, W [N, K] held in one of the library's quantized formats.
* ``grouped``  the same for E experts, W [E, N, K]; the rows of x are sorted by expert, expert e has the
  rows offsets[e] .. offsets[e + 1], any number of them.

W is by definition the tensor that ``dequantize`` returns in the type of x: code times scale, the scale in the type
of x, rounded to the type of x.  The gradient is that of x, of b and (a copy of the incoming one, so not computed) of r;
codes are integers and have none.

A case's ``pass`` is "forward", "backward" (the pre-activation of an earlier forward pass is an input) or "train"
(forward that keeps the pre-activation, then backward).  With ``own`` false ``run`` computes the plain form with
elementary torch operations, else it calls the library.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BITS = {"q8s": 8, "q4s": 4, "q2s": 2, "e4m3": 8, "e5m2": 8, "e2m1": 4}
TOP = {"q8s": 127.0, "q4s": 7.0, "q2s": 1.0, "e4m3": 448.0, "e5m2": 57344.0, "e2m1": 6.0}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _case(name, op, way, rows, n, k, value, store, block, param, dtype, act="none", bias=False, residual=False, experts=1, skew=0.0):
    return {"name": name, "op": op, "pass": way, "rows": rows, "n": n, "k": k, "experts": experts, "value": value, "store": store,
            "block": block, "param": param, "dtype": dtype, "act": act, "bias": bias, "residual": residual, "skew": skew}


def listed():
    return [
        # one token through an attention output projection, 4-bit weights: latency counts
        _case("one_token", "linear", "forward", 1, 4096, 4096, "q4s", "u32", "32", "f32", "bf16", residual=True),
        # a decoding batch through a feed-forward up projection
        _case("decode_batch", "linear", "forward", 16, 14336, 4096, "q8s", "u32", "128", "f32", "bf16", act="silu"),
        # a few dozen rows, no size a multiple of a tile, fp4 weights of a half-precision model
        _case("odd_sizes", "linear", "forward", 77, 1111, 1000, "e2m1", "native", "16", "f16", "f16", act="gelu", bias=True),
        # a prompt through the up projection
        _case("prompt_up", "linear", "forward", 4096, 14336, 4096, "q8s", "u32", "128", "f32", "bf16", act="silu", bias=True),
        # a prompt through the down projection, added to the residual stream
        _case("prompt_down", "linear", "forward", 2048, 4096, 14336, "e2m1", "native", "16", "f16", "f16", residual=True),
        # one layer of a training step on frozen 4-bit weights
        _case("train_step", "linear", "train", 2048, 4096, 4096, "q4s", "u32", "32", "bf16", "bf16", act="gelu_tanh", bias=True),
        # the gradient of a large layer, one scale per tensor
        _case("backward_up", "linear", "backward", 4096, 14336, 4096, "q8s", "u32", "tensor", "f32", "bf16", act="silu", bias=True),
        # a decoding batch of 8 tokens with 2 experts each
        _case("experts_decode", "grouped", "forward", 16, 14336, 4096, "q4s", "u32", "32", "bf16", "bf16", act="silu", experts=8),
        # a middling batch over many small experts, uneven, rows of an odd length in memory
        _case("experts_ragged", "grouped", "forward", 1003, 1500, 1028, "q8s", "u32", "64", "f32", "f16", act="relu", bias=True, experts=16, skew=1.0),
        # prompts through the experts' up projections
        _case("experts_prompt", "grouped", "forward", 8192, 14336, 4096, "q4s", "u32", "32", "bf16", "bf16", act="silu", experts=8, skew=0.5),
        # one layer of a training step on frozen experts
        _case("experts_train", "grouped", "train", 4096, 4096, 2048, "q8s", "u32", "128", "f32", "bf16", act="gelu_tanh", bias=True, experts=8, skew=0.5),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["linear", "grouped"])
    way = rng.choice(["forward", "forward", "backward", "train"])
    value, store = rng.choice([("q8s", "u32"), ("q4s", "u32"), ("q2s", "u32"), ("q8s", "native"), ("e2m1", "native"), ("e4m3", "native"), ("e5m2", "native")])
    block = rng.choice(["tensor", "16", "32", "64", "128", "64x64", "128x128"])
    if value == "q2s" and block == "tensor":
        block = "64"
    experts = rng.choice([2, 4, 8, 16, 32, 64]) if op == "grouped" else 1
    step = {"q8s": 4, "q4s": 8, "q2s": 16, "e2m1": 2}.get(value, 1) if (value, store) != ("q8s", "native") else 1
    n = log(64, 14336)
    k = log(64, 14336) // step * step
    if rng.random() < 0.5:  # half of the cases have the round sizes that models have
        n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
    while experts * n * k > 8 * 14336 * 4096:
        experts //= 2
    rows = log(1, 8192)
    if way == "train":
        rows = min(rows, 4096)
    rows = max(1, min(rows, int(8192 * 14336 * 4096 * 0.5 / (n * k))))
    dtype = rng.choice(["bf16", "f16"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    return {"op": op, "pass": way, "rows": rows, "n": n, "k": k, "experts": experts, "value": value, "store": store, "block": block,
            "param": rng.choice(["f32", dtype]), "dtype": dtype, "act": act, "bias": rng.random() < 0.5,
            "residual": way == "forward" and rng.random() < 0.5, "skew": rng.choice([0.0, 0.5, 1.0]) if op == "grouped" else 0.0}


def _block(case):
    """Block extents along n and k; None per tensor."""
    if case["block"] == "tensor":
        return None
    dims = [int(d) for d in case["block"].split("x")]
    return (1, dims[0]) if len(dims) == 1 else tuple(dims)


def _pack(codes, bits):
    """Codes of ``bits`` bits (0 .. 2^bits - 1, int32) packed along the last dim into int32 words."""
    per = 32 // bits
    c = codes.view(*codes.shape[:-1], codes.shape[-1] // per, per)
    words = c[..., 0].clone()
    for i in range(1, per):
        words |= c[..., i] << (bits * i)
    return words


def _quantized(case, gen):
    """Codes and scales of random weights N(0, 0.02), as the library's quantize leaves them; one expert at a time."""
    n, k, value, bits = case["n"], case["k"], case["value"], BITS[case["value"]]
    blk = _block(case)
    pdt, xdt = DTYPES[case["param"]], DTYPES[case["dtype"]]
    tiny = 2.0 ** -13 if value == "e5m2" and (case["param"] == "f16" or case["dtype"] == "f16") else 1.0  # e5m2's scale stays a normal f16
    all_codes, all_scales = [], []
    for _ in range(case["experts"]):
        w = torch.randn(n, k, device="cuda", generator=gen) * 0.02
        if blk is None:
            s = (torch.full((1, 1), 0.1, device="cuda") / (TOP[value] * tiny)).to(pdt)
            full = s.to(xdt).float()
        else:
            bn, bk = blk
            wp = torch.nn.functional.pad(w.abs(), (0, -k % bk, 0, -n % bn))
            s = (wp.view(wp.shape[0] // bn, bn, wp.shape[1] // bk, bk).amax((1, 3)) / (TOP[value] * tiny)).to(pdt)
            full = s.to(xdt).float().repeat_interleave(bn, 0)[:n].repeat_interleave(bk, 1)[:, :k]
        q = (w / full).clamp(-TOP[value], TOP[value])
        if value in ("q8s", "q4s", "q2s"):
            c = q.round().to(torch.int32)
            c = c.to(torch.int8) if case["store"] == "native" else _pack(c & ((1 << bits) - 1), bits)
        elif value == "e2m1":
            mag = torch.bucketize(q.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")).to(torch.uint8)
            nib = mag | ((q < 0).to(torch.uint8) << 3)
            c = nib[:, 0::2] | (nib[:, 1::2] << 4)
        else:
            c = q.to(torch.float8_e4m3fn if value == "e4m3" else torch.float8_e5m2).view(torch.uint8)
        all_codes.append(c)
        all_scales.append(s)
    if case["op"] == "linear":
        return all_codes[0], all_scales[0].view(-1) if blk is None else all_scales[0]
    codes = torch.stack(all_codes)
    return codes, all_scales[0].view(-1) if blk is None else torch.stack(all_scales)


def _counts(case, gen):
    """Rows of each expert: tokens choose experts at random, the popular ones by ``skew``."""
    e = case["experts"]
    weight = torch.exp(torch.randn(e, device="cuda", generator=gen) * case["skew"])
    chosen = torch.multinomial(weight, case["rows"], replacement=True, generator=gen)
    return torch.bincount(chosen, minlength=e)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, n, k, e = case["rows"], case["n"], case["k"], case["experts"]
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    s["codes"], s["scales"] = _quantized(case, gen)
    lead = (e,) if case["op"] == "grouped" else ()
    if case["op"] == "grouped":
        counts = _counts(case, gen)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["most"] = int(counts.max())  # the plain form pads every expert to this many rows
    if case["pass"] != "backward":
        s["x"] = torch.randn(t, k, device="cuda", generator=gen).to(dt)
        s["bias"] = (torch.randn(*lead, n, device="cuda", generator=gen) * 0.5).to(dt) if case["bias"] else None
        s["residual"] = torch.randn(t, n, device="cuda", generator=gen).to(dt) if case["residual"] else None
        s["y"] = torch.empty(t, n, device="cuda", dtype=dt)
    if case["pass"] != "forward":
        s["grad"] = torch.randn(t, n, device="cuda", generator=gen).to(dt)
        s["grad_x"] = torch.empty(t, k, device="cuda", dtype=dt)
        s["grad_bias"] = torch.empty(*lead, n, device="cuda", dtype=dt) if case["bias"] else None
        s["pre"] = None
        if case["act"] != "none":  # for "train" a buffer that the forward pass fills
            s["pre"] = torch.randn(t, n, device="cuda", generator=gen).to(dt) if case["pass"] == "backward" else torch.empty(t, n, device="cuda", dtype=dt)
    return s


# ---- plain form ---------------------------------------------------------------------------------------------------------

def _values(codes, case):
    """The numbers that the stored codes stand for, f32 [.., n, k]."""
    value, bits = case["value"], BITS[case["value"]]
    if value in ("e4m3", "e5m2"):
        return codes.view(torch.float8_e4m3fn if value == "e4m3" else torch.float8_e5m2).float()
    if value == "e2m1":
        nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
        return torch.tensor(FP4, device=codes.device)[nib.int()]
    if case["store"] == "native":
        return codes.float()
    shift = torch.arange(0, 32, bits, device=codes.device, dtype=torch.int32)
    field = (codes.unsqueeze(-1) << (32 - bits - shift)) >> (32 - bits)  # sign extended
    return field.flatten(-2).float()


def _weights(s):
    """W in f32: code times scale, each as ``dequantize`` has it in the type of x."""
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    q = _values(s["codes"], case)
    scale = s["scales"].to(dt).float()
    blk = _block(case)
    if blk is not None:
        bn, bk = blk
        if bn > 1:
            scale = scale.repeat_interleave(bn, -2)[..., :case["n"], :]
        scale = scale.repeat_interleave(bk, -1)[..., :case["k"]]
    return (q * scale).to(dt).float()


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z / (1 + torch.exp(-z)) if act == "silu" else z


def _slope(z, act):
    """Derivative of ``_act``."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)
    sig = 1 / (1 + torch.exp(-z))
    return sig * (1 + z * (1 - sig))


def _expert_of(s):
    rows = torch.arange(s["case"]["rows"], device="cuda")
    return torch.searchsorted(s["offsets"].long(), rows, right=True) - 1, rows


def _product(s, a, w):
    """a [T, c] times the weights [.., c, f] of each row's expert, f32."""
    if s["case"]["op"] == "linear":
        return a @ w
    e, rows = _expert_of(s)
    at = rows - s["offsets"].long()[e]
    padded = a.new_zeros(s["case"]["experts"], s["most"], a.shape[1])
    padded[e, at] = a
    return torch.bmm(padded, w)[e, at]


def _forward(s, w):
    case = s["case"]
    z = _product(s, s["x"].float(), w.mT)
    if s["bias"] is not None:
        z = z + (s["bias"].float() if case["op"] == "linear" else s["bias"].float()[_expert_of(s)[0]])
    y = _act(z, case["act"])
    return (y if s["residual"] is None else y + s["residual"].float()).to(DTYPES[case["dtype"]]), z


def _backward(s, w, z):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    dz = s["grad"].float()
    if case["act"] != "none":
        dz = dz * _slope(z, case["act"])
    out = {"grad_x": _product(s, dz, w).to(dt)}
    if case["bias"]:
        if case["op"] == "linear":
            out["grad_bias"] = dz.sum(0).to(dt)
        else:
            out["grad_bias"] = dz.new_zeros(case["experts"], case["n"]).index_add_(0, _expert_of(s)[0], dz).to(dt)
    return out


def _plain(s):
    case = s["case"]
    w = _weights(s)
    if case["pass"] == "backward":
        return _backward(s, w, None if s["pre"] is None else s["pre"].float())
    y, z = _forward(s, w)
    return {"y": y} if case["pass"] == "forward" else {"y": y, **_backward(s, w, z)}


# ---- the library's operators ----------------------------------------------------------------------------------------------

def _plan(s):
    """The prepared calls that a user's program keeps beside its buffers: checks of arguments and workspaces, done once."""
    from cubek_b200 import (ComputeClient, ElemType, QuantLevel, QuantParam, QuantScheme, QuantStore, QuantValue, TensorHandleRef,
                            grouped_linear, linear)
    from cubek_b200.linear import Activation
    from cubek_b200.matmul_input import MatmulInputHandleRef

    case = s["case"]
    handle = lambda t: None if t is None else TensorHandleRef.from_torch(t)  # noqa: E731
    value = {"q8s": QuantValue.Q8S, "q4s": QuantValue.Q4S, "q2s": QuantValue.Q2S, "e4m3": QuantValue.E4M3, "e5m2": QuantValue.E5M2,
             "e2m1": QuantValue.E2M1}[case["value"]]
    param = {"f32": QuantParam.F32, "f16": QuantParam.F16, "bf16": QuantParam.BF16}[case["param"]]
    elem = {"f16": ElemType.F16, "bf16": ElemType.BF16}[case["dtype"]]
    act = {"none": Activation.Identity, "relu": Activation.Relu, "gelu": Activation.Gelu, "gelu_tanh": Activation.GeluTanh,
           "silu": Activation.Silu}[case["act"]]
    level = QuantLevel.Tensor if case["block"] == "tensor" else QuantLevel.block([int(d) for d in case["block"].split("x")])
    scheme = QuantScheme(value=value, param=param, store=QuantStore.U32 if case["store"] == "u32" else QuantStore.Native, level=level)
    grouped = case["op"] == "grouped"
    shape = ((case["experts"],) if grouped else ()) + (case["n"], case["k"])
    weight = MatmulInputHandleRef.quantized(handle(s["codes"]), handle(s["scales"]), shape, scheme)
    client = ComputeClient.current()
    at = (handle(s["offsets"]),) if grouped else ()
    mod = grouped_linear if grouped else linear
    calls = []
    if case["pass"] != "backward":
        size = mod.workspace_bytes(handle(s["x"]), weight, elem)
        s["work"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        calls.append(mod.Prepared(client, handle(s["x"]), *at, weight, handle(s["y"]), elem, bias=handle(s["bias"]), residual=handle(s["residual"]),
                                  activation=act, pre=handle(s.get("pre")), workspace=handle(s["work"])))
    if case["pass"] != "forward":
        size = mod.backward_workspace_bytes(handle(s["grad"]), weight, elem, activation=act, bias=case["bias"])
        s["work_back"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        calls.append(mod.PreparedBackward(client, handle(s["grad"]), *at, weight, handle(s["grad_x"]), elem, pre=handle(s["pre"]), activation=act,
                                          grad_bias=handle(s["grad_bias"]), workspace=handle(s["work_back"])))
    return calls


def _own(s):
    if "plan" not in s:
        s["plan"] = _plan(s)
    for call in s["plan"]:
        call()
    out = {"y": s["y"]} if "y" in s else {}
    if "grad_x" in s:
        out["grad_x"] = s["grad_x"]
        if s["grad_bias"] is not None:
            out["grad_bias"] = s["grad_bias"]
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------

def work(case):
    t, n, k, e = case["rows"], case["n"], case["k"], case["experts"]
    busy = e * (1 - (1 - 1 / e) ** t) if case["op"] == "grouped" and e > 1 else 1.0  # experts with rows
    blk = _block(case)
    per = {"f32": 4, "f16": 2, "bf16": 2}[case["param"]]
    weights = busy * n * k * BITS[case["value"]] / 8 + (per if blk is None else busy * -(-n // blk[0]) * -(-k // blk[1]) * per)
    size, product, total, flops = 2, 2.0 * t * n * k, 0.0, 0.0
    if case["pass"] != "backward":
        total += weights + size * (t * k + t * n * (2 if case["residual"] else 1) + (busy * n if case["bias"] else 0))
        flops += product
    if case["pass"] != "forward":
        total += weights + size * (t * n * (2 if case["act"] != "none" else 1) + t * k + (e * n if case["bias"] else 0))
        total += size * t * n if case["pass"] == "train" and case["act"] != "none" else 0  # the kept pre-activation is written too
        flops += product
    return {"bytes": total, "flops": flops}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------

def _table(case):
    """What every byte (8-bit values) or nibble / pair of bits stands for, f64."""
    value = case["value"]
    if value == "e2m1":
        return [(-1.0) ** (c >> 3) * ((c & 1) * 0.5 if (c >> 1 & 3) == 0 else (1 + (c & 1) * 0.5) * 2.0 ** ((c >> 1 & 3) - 1)) for c in range(16)]
    if value in ("e4m3", "e5m2"):
        m = 3 if value == "e4m3" else 2
        bias = 7 if value == "e4m3" else 15
        out = []
        for c in range(256):
            ex, fr = c >> m & (1 << (7 - m)) - 1, c & (1 << m) - 1
            v = fr * 2.0 ** (1 - bias - m) if ex == 0 else (1 + fr / (1 << m)) * 2.0 ** (ex - bias)
            if value == "e4m3" and c & 127 == 127:
                v = math.nan
            if value == "e5m2" and ex == 31:
                v = math.nan if fr else math.inf
            out.append(-v if c >> 7 else v)
        return out
    b = BITS[value]
    return [float(c - (1 << b) if c >> (b - 1) else c) for c in range(1 << b)]


def exact(case, seed):
    s = prepare(case, seed)
    f64, dt = torch.float64, DTYPES[case["dtype"]]
    n, k, e, b = case["n"], case["k"], case["experts"], BITS[case["value"]]
    grouped = case["op"] == "grouped"
    bounds = s["offsets"].tolist() if grouped else [0, case["rows"]]
    table = torch.tensor(_table(case), dtype=f64, device="cuda")
    blk = _block(case)
    y = torch.empty(case["rows"], n, dtype=f64, device="cuda")
    gx = torch.empty(case["rows"], k, dtype=f64, device="cuda")
    gb = torch.zeros(e, n, dtype=f64, device="cuda")
    for i in range(e):
        rows = slice(bounds[i], bounds[i + 1])
        if rows.start == rows.stop:
            continue
        raw = (s["codes"][i] if grouped else s["codes"]).contiguous().view(torch.uint8)  # little endian: fields in order from the low bits
        fields = torch.stack([raw >> sh & (1 << b) - 1 for sh in range(0, 8, b)], -1).reshape(n, k)
        w = table[fields.long()]
        del fields
        scale = (s["scales"][i] if grouped and blk else s["scales"]).to(dt).to(f64)
        if blk is None:
            w *= scale.reshape(())
        else:
            w *= scale[torch.arange(n, device="cuda") // blk[0]][:, torch.arange(k, device="cuda") // blk[1]]
        w = w.to(dt).to(f64)
        z = s["pre"][rows].to(f64) if case["pass"] == "backward" and s["pre"] is not None else None
        if case["pass"] != "backward":
            z = s["x"][rows].to(f64) @ w.T
            if case["bias"]:
                z += (s["bias"][i] if grouped else s["bias"]).to(f64)
            half = 0.5 * (1 + torch.erf(z / 2 ** 0.5))
            y[rows] = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0.0), "gelu": lambda: z * half, "silu": lambda: z * torch.sigmoid(z),
                       "gelu_tanh": lambda: z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z))}[case["act"]]()
            if case["residual"]:
                y[rows] += s["residual"][rows].to(f64)
        if case["pass"] != "forward":
            dz = s["grad"][rows].to(f64)
            if case["act"] == "relu":
                dz = torch.where(z > 0, dz, 0.0)
            elif case["act"] == "gelu":
                dz = dz * (0.5 * torch.erfc(-z / 2 ** 0.5) + z * torch.exp(-z * z / 2) * (0.5 / math.pi) ** 0.5)
            elif case["act"] == "silu":
                dz = dz * (torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z))
            elif case["act"] == "gelu_tanh":
                u = 2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)
                dz = dz * (torch.sigmoid(u) + z * torch.sigmoid(u) * torch.sigmoid(-u) * 2 * (2 / math.pi) ** 0.5 * (1 + 0.134145 * z * z))
            gx[rows] = dz @ w
            gb[i] = dz.sum(0)
        del w
    out = {"y": y} if case["pass"] != "backward" else {}
    if case["pass"] != "forward":
        out["grad_x"] = gx
        if case["bias"]:
            out["grad_bias"] = gb if grouped else gb[0]
    return out
