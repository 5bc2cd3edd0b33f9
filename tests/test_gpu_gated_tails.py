"""gated_linear's activations far from zero, where they or their slopes are small: to a few roundings of themselves, not of 1.

One row of a single value 1 makes g the weight itself, y act(g) with u = 1, and dw's first half dy u act'(g). Tolerances in u = 2^-24
of the value: GELU's erfc is good for 16 of its steps (32 u), its argument -g / sqrt(2) for 2 u, which its slope turns into 2 (g^2 + 1) u,
and what multiplies it for 6 u; exp's argument g^2 / 2 is off by u of itself twice, and exp by 4 u. The logistic's exp(-g) has an exact
argument: 4 u, and 12 for what follows. Then half a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def call(g, act, dtype):
    """y and the gradient of g for values g of the type"""
    from yggdrasil_amd import ops
    w = torch.stack([g, torch.ones_like(g)])[:, :, None].cuda().requires_grad_()
    y = ops.gated_linear(torch.ones(1, 1, dtype=dtype, device="cuda"), w, act)
    dw, = torch.autograd.grad(y.sum(), w)
    return y.detach()[0].cpu(), dw[0, :, 0].cpu()


def near(got, ref, tol):
    half = torch.finfo(got.dtype).eps / 2
    room = tol + half * (ref.abs() + tol) + LEAST[got.dtype]
    err = (got.double() - ref).abs()
    assert (err <= room).all(), float((err / room).max())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gelu(dtype):
    g = torch.linspace(-12.0, 12.0, 4001).to(dtype)
    y, slope = call(g, "gelu", dtype)
    v = g.double()
    phi, bell = 0.5 * torch.special.erfc(-v * math.sqrt(0.5)), torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    near(y, v * phi, (v * phi).abs() * U * (42 + 2 * v * v))
    near(slope, phi + v * bell, U * (phi * (42 + 2 * v * v) + (v * bell).abs() * (12 + v * v)))
