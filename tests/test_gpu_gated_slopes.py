"""The logistic's slope p (1 - p) in gated_linear's gradient, far on both sides of zero: to a few roundings of itself.

One row of a single value 1 makes g the weight itself, and dw's first half dy u act'(g) with dy = u = 1. exp(-g) is good for 4 u
(u = 2^-24), the sum, the quotient and the products for 8 more. Then half a step of the type, or of its smallest."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


@pytest.mark.parametrize("dtype", list(LEAST), ids=str)
def test_sigmoid(dtype):
    from yggdrasil_amd import ops
    g = torch.linspace(-80.0, 80.0, 4001).to(dtype)
    w = torch.stack([g, torch.ones_like(g)])[:, :, None].cuda().requires_grad_()
    y = ops.gated_linear(torch.ones(1, 1, dtype=dtype, device="cuda"), w, "sigmoid")
    dw, = torch.autograd.grad(y.sum(), w)
    v = g.double()
    for got, ref in ((y.detach()[0], torch.sigmoid(v)), (dw[0, :, 0], torch.sigmoid(v) * torch.sigmoid(-v))):
        tol = 12 * U * ref.abs()
        room = tol + torch.finfo(dtype).eps / 2 * (ref.abs() + tol) + LEAST[dtype]
        err = (got.double().cpu() - ref).abs()
        assert (err <= room).all(), float((err / room).max())
