"""What gated_linear keeps of its projections for the backward pass: f32, or its upper 24 bits for 16-bit types. With a single row
whose first value is 1 the first column of dw is dg and du themselves, rounded once to the type, so that a projection kept in fewer
bits shows. And the same gradients every time.

Tolerances: g and u are kept to 2^-16 of themselves (f32: exactly) after their sum's own p (2^-22 (8 + 2 sqrt(K)) times the root of
the products' squares); of dg that is dy times the error of u times act', and times u times that of g times act'' (at most 0.8), with a few roundings
in f32 (16 cover the activation's); of du dy times 1.13 times g's. Then half a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def act_of(name, g):
    if name == "gelu":
        phi = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
        return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    p = torch.sigmoid(g)
    return (g * p, p + g * p * torch.sigmoid(-g)) if name == "silu" else (p, p * torch.sigmoid(-g))


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N, K", [(4000, 64), (1003, 200), (5001, 33)])
def test_projections_are_kept_in_24_bits(N, K, dtype, act):
    from yggdrasil_amd import ops
    r = torch.Generator().manual_seed(N)
    x = torch.randn(1, K, generator=r)
    x[0, 0] = 1.0
    x, w = x.to(dtype), (torch.randn(2, N, K, generator=r) * 1.5 / math.sqrt(K)).to(dtype)
    dy = (2 + torch.rand(1, N, generator=r)).to(dtype)
    xg, wg = x.cuda(), w.cuda().requires_grad_()
    got, = torch.autograd.grad(ops.gated_linear(xg, wg, act), wg, dy.cuda())
    x, w, dy = x.double(), w.double(), dy.double()
    g, u = x @ w[0].t(), x @ w[1].t()
    a, slope = act_of(act, g)
    keep = 0.0 if dtype == torch.float32 else 2.0 ** -16
    tg, tu = (2.0 ** -22 * (8 + 2 * math.sqrt(K)) * (x ** 2 @ (v ** 2).t()).sqrt() for v in w)
    eg, eu = tg + keep * (g.abs() + tg), tu + keep * (u.abs() + tu)
    half = torch.finfo(dtype).eps / 2
    for d, t, out in ((dy * u * slope, dy.abs() * (eu * (slope.abs() + 0.8 * eg) + 0.8 * eg * u.abs() + 16 * U * u.abs()), got[0]),
                      (dy * a, dy.abs() * (1.13 * eg + 16 * U * (1 + g.abs())), got[1])):
        err = (out[:, 0].double().cpu() - d[0]).abs()
        room = (t + half * (d.abs() + t) + 2.0 ** -25)[0]
        assert (err <= room).all(), float((err / room).max())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, N, K", [(1, 300, 64), (70, 500, 333), (1001, 2003, 1000), (2048, 2048, 1024)])
def test_the_same_every_time(M, N, K, dtype):
    from yggdrasil_amd import ops
    r = torch.Generator("cuda").manual_seed(M)
    x, w, dy = (torch.randn(s, generator=r, device="cuda").to(dtype) for s in ((M, K), (2, N, K), (M, N)))
    x, w = x.requires_grad_(), (w / math.sqrt(K)).requires_grad_()

    def once():
        y = ops.gated_linear(x, w, "gelu")
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))
    want = once()
    for _ in range(5):
        filled = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(4)]    # what later allocations hold
        del filled
        assert all(torch.equal(a, b) for a, b in zip(once(), want))
