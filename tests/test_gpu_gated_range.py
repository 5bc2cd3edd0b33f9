"""gated_linear's gradients where dg = dy u act'(g) and du = dy act(g) leave float16's range, above and below, though what comes of
them does not; and where rows or columns of them differ by many powers of two.

Tolerances, with h half a step of the type: those of g and u (sums of K products in f32, p(K, s) = 2^-22 (8 + 2 sqrt(K)) s with s^2 the
squares' sum; kept in 24 bits, 2^-16 of themselves, in f32 whole) times dy, the other factor and the activation's slopes (act' at most
1.13, act'' at most 0.8); dg and du are rounded to the type: h of themselves, or in float16 half a step of its smallest, 2^-25, where the
row's (for dx) or column's (for dw) largest is 2^-3 or more as it is, or brought to 2^14: 2^-22 of that. Then each sum's own p and half a step of the
result's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
ACTS = ["silu", "gelu", "sigmoid"]


def act_of(name, g):
    if name == "gelu":
        phi = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
        return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    p = torch.sigmoid(g)
    return (g * p, p + g * p * torch.sigmoid(-g)) if name == "silu" else (p, p * torch.sigmoid(-g))


def near(got, ref, tol, name):
    assert got.shape == ref.shape, name
    half = torch.finfo(got.dtype).eps / 2
    err = (got.detach().double().cpu() - ref).abs()
    room = tol + half * (ref.abs() + tol) + LEAST[got.dtype]
    assert (err <= room).all(), (name, float((err / room).max()))


def p(terms, squares):
    return 2.0 ** -22 * (8 + 2 * math.sqrt(terms)) * squares.sqrt()


def gradients(x, w, dy, act):
    """dg, du, and dx and dw with their tolerances, in 64 bits."""
    (M, K), N = x.shape, w.shape[1]
    h, half = torch.finfo(x.dtype).eps / 2, x.dtype == torch.float16
    keep = 0.0 if x.dtype == torch.float32 else 2.0 ** -16
    x, w, dy = x.double(), w.double(), dy.double()
    g, u = x @ w[0].t(), x @ w[1].t()
    a, slope = act_of(act, g)
    tg, tu = p(K, x ** 2 @ (w[0] ** 2).t()), p(K, x ** 2 @ (w[1] ** 2).t())
    eg, eu = tg + keep * (g.abs() + tg), tu + keep * (u.abs() + tu)
    dg, du = dy * u * slope, dy * a
    rg = dy.abs() * (eu * (slope.abs() + 0.8 * eg) + 0.8 * eg * u.abs() + 16 * U * u.abs()) + 1.01 * h * dg.abs()
    ru = dy.abs() * (1.13 * eg + 16 * U * (1 + g.abs())) + 1.01 * h * du.abs()
    both = torch.cat([dg, du], 1).abs()
    row = 2.0 ** -22 * both.amax(1, keepdim=True) if half else 0.0
    dx = dg @ w[0] + du @ w[1]
    tx = (rg + row) @ w[0].abs() + (ru + row) @ w[1].abs() + 1.1 * p(2 * N, dg ** 2 @ w[0] ** 2 + du ** 2 @ w[1] ** 2)
    dw, tw = [], []
    for d, r in ((dg, rg), (du, ru)):
        column = 2.0 ** -22 * d.abs().amax(0, keepdim=True) if half else 0.0
        dw.append(d.t() @ x)
        tw.append((r + column).t() @ x.abs() + 1.1 * p(M, (d ** 2).t() @ x ** 2))
    return dg, du, (dx, tx), (torch.stack(dw), torch.stack(tw))


SIZES = [(1, 5, 9), (7, 33, 40), (40, 70, 64), (300, 256, 264), (500, 1003, 203), (1100, 1000, 520)]
# scales of x, Wg, Wu and dy; which gradient they leave in range
REACH = {"large dx": (100.0, 0.016, 3.0, 300.0), "large dw": (2.0 ** -7, 100.0, 4e4, 150.0),
         "tiny dx": (2.0 ** -12, 2.0 ** 12, 2.0 ** 6, 2.0 ** -20), "tiny dw": (2.0 ** 9, 2.0 ** -9, 2.0 ** -15, 2.0 ** -20)}


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M, N, K", SIZES)
@pytest.mark.parametrize("reach", list(REACH))
def test_float16(reach, M, N, K, act):
    from yggdrasil_amd import ops
    sx, sg, su, sy = REACH[reach]
    r = torch.Generator().manual_seed(M)
    x = (sx * torch.randn(M, K, generator=r)).half()
    w = torch.randn(2, N, K, generator=r) / math.sqrt(K)
    w = torch.stack([sg * w[0], su * w[1]]).clamp(-6e4, 6e4).half()
    dy = (sy * torch.randn(M, N, generator=r)).half()
    dg, du, dx, dw = gradients(x, w, dy, act)
    if reach[:5] == "large":
        assert M < 40 or (dg.abs() > 65520).any()
    else:
        assert float((dg.abs() < 2.0 ** -25).float().mean()) > 0.5
    ref, tol = dx if reach[-2:] == "dx" else dw
    assert float(ref.abs().max()) < 65504 and float(ref.abs().max()) > 2.0 ** -18
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    got = torch.autograd.grad(ops.gated_linear(xg, wg, act), (xg, wg), dy.cuda())
    near(got[reach[-2:] == "dw"], ref, tol, reach)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M, N, K", SIZES)
@pytest.mark.parametrize("along", [0, 1])
def test_rows_and_columns_of_many_sizes(along, M, N, K, dtype):
    """dy's rows, or its columns, from 2^-18 to 2^7 in size; a row and a column of zeros."""
    from yggdrasil_amd import ops
    r = torch.Generator().manual_seed(M + along)
    x, w = torch.randn(M, K, generator=r).to(dtype), (torch.randn(2, N, K, generator=r) * 1.5 / math.sqrt(K)).to(dtype)
    dy = torch.randn(M, N, generator=r)
    size = 2.0 ** torch.randint(-18, 8, (dy.shape[along],), generator=r)
    dy = (dy * (size[:, None] if along == 0 else size)).to(dtype)
    dy[M // 2], dy[:, N // 2] = 0, 0
    _, _, dx, dw = gradients(x, w, dy, "silu")
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    got = torch.autograd.grad(ops.gated_linear(xg, wg), (xg, wg), dy.cuda())
    near(got[0], *dx, "dx")
    near(got[1], *dw, "dw")
    assert not got[0][M // 2].any() and not got[1][:, N // 2].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M, N, K", SIZES[2:])
def test_values_that_are_not_finite(M, N, K, dtype):
    """An infinity or a NaN of dy stays in its row of dx and its columns' rows of dw, and the others are as they were."""
    from yggdrasil_amd import ops
    r = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, K, generator=r).to(dtype), (torch.randn(2, N, K, generator=r) * 1.5 / math.sqrt(K)).to(dtype)
    dy = torch.randn(M, N, generator=r).to(dtype)
    _, _, dx, dw = gradients(x, w, dy, "silu")
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    dy[3, 5], dy[9, 11] = math.inf, math.nan
    got = torch.autograd.grad(ops.gated_linear(xg, wg), (xg, wg), dy.cuda())
    for t, bad, (ref, tol) in ((got[0], torch.tensor([3, 9]), dx), (got[1].transpose(0, 1), torch.tensor([5, 11]), (dw[0].transpose(0, 1), dw[1].transpose(0, 1)))):
        assert not t[bad.cuda()].isfinite().any()
        good = torch.ones(len(t), dtype=torch.bool)
        good[bad] = False
        near(t[good.cuda()], ref[good], tol[good], "others")


@pytest.mark.parametrize("N, K", [(5, 9), (300, 264), (4096, 777)])
def test_no_rows(N, K):
    from yggdrasil_amd import ops
    x, w = (torch.zeros(s, dtype=torch.float16, device="cuda", requires_grad=True) for s in ((0, K), (2, N, K)))
    dx, dw = torch.autograd.grad(ops.gated_linear(x, w).sum(), (x, w))
    assert dx.shape == (0, K) and dw.shape == w.shape and not dw.any()


@pytest.mark.parametrize("M, N, K", [(1, 300, 256), (300, 200, 264), (2048, 4096, 64), (500, 1003, 203)])
def test_streams_and_graphs(M, N, K):
    """Rows of other sizes in each replay: the largest of the one before must not stay."""
    from yggdrasil_amd import ops

    def make(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        x, w, dy = (torch.randn(s, generator=g, device="cuda") for s in ((M, K), (2, N, K), (M, N)))
        return x.half(), (w / math.sqrt(K)).half(), (dy * 2.0 ** torch.randint(-12, 9, (M, 1), generator=g, device="cuda")).half()

    def both(leaves, dy):
        y = ops.gated_linear(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    x, w, dy = make(0)
    leaves = [t.requires_grad_() for t in (x, w)]
    want = both(leaves, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(leaves, dy)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del want, got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(leaves, dy)
    for k in range(4):
        new = make(10 + k)
        with torch.no_grad():
            for t, v in zip((x, w, dy), new):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        want = both([t.requires_grad_() for t in new[:2]], new[2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want)), k
