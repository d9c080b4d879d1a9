"""Shared by the tests of the products with quantized weights: inputs, the 64-bit reference and its error bounds.

W is the oracle's dequantized weight in the type F of x (u = half a step of F, relative).  The kernel's f32 sum of c products
differs from the exact one by at most (c + 16) 2^-23 S with S = sum |a_i w_i| (each addition, also one that truncates, is off
by at most 2^-23 of a partial sum, and those are bounded by S); the activations change z by at most 1.13 |dz| and cost a few
f32 roundings (2^-20 covers exp, the division and the polynomial); then one rounding to F: u |y|, and half the smallest
subnormal of F."""
from __future__ import annotations

import math

import numpy as np
import torch

from cubek_b200 import ElemType, QuantScheme, TensorHandleRef
from cubek_b200.linear import Activation
from cubek_b200.matmul_input import MatmulInputHandleRef
from oracle import oracle as O
from tests._util import NP_FLOAT, to_device

H = TensorHandleRef.from_torch
TORCH = {ElemType.F16: torch.float16, ElemType.BF16: torch.bfloat16}
HALF_STEP = {ElemType.F16: 2.0 ** -11, ElemType.BF16: 2.0 ** -8}
TINY = {ElemType.F16: 2.0 ** -25, ElemType.BF16: 2.0 ** -134}
LIPSCHITZ = 1.13  # of gelu and silu; 1 for the others


class Weight:
    """A random weight of logical shape [N, K] or [E, N, K], quantized by the oracle, on the device."""

    def __init__(self, shape, scheme: QuantScheme, elem: ElemType, seed: int, codes=None, scales=None):
        rng = np.random.default_rng(seed)
        w = rng.standard_normal(shape).astype(np.float32)
        if codes is None:
            codes, scales = O.quantize_dynamic(w, scheme)
        self.scheme, self.elem, self.shape = scheme, elem, tuple(shape)
        self.codes, self.scales = codes, scales
        self.dcodes, self.dscales = to_device(codes), to_device(scales)
        if codes.size == 0:   # NumPy's strides of an empty array are zeros
            self.dcodes = torch.empty(codes.shape, dtype=self.dcodes.dtype, device="cuda")
        self.value = to_device(O.dequantize(codes, scales, scheme, NP_FLOAT[elem])).double()   # [.., N, K]

    def handle(self, data=None, scale=None) -> MatmulInputHandleRef:
        return MatmulInputHandleRef.quantized(H(self.dcodes if data is None else data), H(self.dscales if scale is None else scale),
                                              self.shape, self.scheme)


def randn(shape, elem: ElemType, seed: int) -> torch.Tensor:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=gen).to(TORCH[elem])


def filled(shape, elem: ElemType) -> torch.Tensor:
    """An output buffer of a bit pattern that no result has, so that unwritten elements are seen."""
    t = torch.empty(*shape, device="cuda", dtype=TORCH[elem])
    t.view(torch.uint8).fill_(0xA5)
    return t


def act64(z, act):
    if act == Activation.Relu:
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == Activation.Gelu:
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    if act == Activation.GeluTanh:
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z) if act == Activation.Silu else z


def slope64(z, act):
    if act == Activation.Relu:
        return (z > 0).double()
    if act == Activation.Gelu:
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == Activation.GeluTanh:
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == Activation.Silu:
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def sum_bound(a, w):
    """Bound of the error of the f32 sums of a [rows, c] times w [c, f]."""
    return (a.shape[-1] + 16) * 2.0 ** -23 * (a.abs() @ w.abs())


def check_forward(y, pre, x, w, elem, bias=None, residual=None, act=Activation.Identity):
    """y [rows, N] (and pre) against the definition, w [N, K] in 64 bits."""
    u, x64 = HALF_STEP[elem], x.double()
    z = x64 @ w.mT
    off = sum_bound(x64, w.mT)
    if bias is not None:
        z = z + bias.double()
        off = off + 2.0 ** -23 * z.abs()
    want = act64(z, act)
    tol = LIPSCHITZ * off + 2.0 ** -20 * z.abs()
    if residual is not None:
        want = want + residual.double()
        tol = tol + 2.0 ** -23 * want.abs()
    assert_within(y, want, (1 + u) * tol + u * want.abs() + TINY[elem], "y")
    if pre is not None:
        assert_within(pre, z, (1 + u) * off + u * z.abs() + TINY[elem], "pre")


def check_backward(gx, gb, gp, g, w, elem, pre=None, act=Activation.Identity):
    u, dz = HALF_STEP[elem], g.double()
    approx = torch.zeros_like(dz)
    rounded = 0.0
    if act != Activation.Identity:
        z = pre.double()
        dz = dz * slope64(z, act)
        # exp and erfc to a few f32 steps, times factors of up to |z|^3 / 2 where 1 - sigmoid(..) cancels
        approx = g.double().abs() * (1 + z.abs() ** 3) * 2.0 ** -20
        rounded = u
    if gp is not None:
        assert_within(gp, dz, approx * (1 + u) + u * dz.abs() + TINY[elem], "grad_pre")
    if gx is not None:
        want = dz @ w
        tol = sum_bound(dz, w) * (1 + u) + (approx * (1 + u) + rounded * dz.abs() + TINY[elem] * (rounded > 0)) @ w.abs()
        assert_within(gx, want, (1 + u) * tol + u * want.abs() + TINY[elem], "grad_input")
    if gb is not None:
        want = dz.sum(0)
        tol = (dz.shape[0] + 16) * 2.0 ** -23 * dz.abs().sum(0) + approx.sum(0)
        assert_within(gb, want, (1 + u) * tol + u * want.abs() + TINY[elem], "grad_bias")


def assert_within(got, want, tol, what):
    got = got.double()
    off = (got - want).abs()
    bad = ~(off <= tol)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} elements off; first at {i}: got {float(got[i])!r}, "
                             f"want {float(want[i])!r} within {float(tol[i])!r}")
