"""gated_linear and its gradients against the formula in 64 bits: every type and activation, sizes from one on, ones that end inside a
tile or off an alignment, those where another kernel takes over.

Tolerances, with h half a step of the inputs' type and p(I, s) = 2^-22 (8 + 2 sqrt(I)) s for a sum of I products in f32 whose squares
sum to s^2 (each addition rounds a partial sum of about that size): g and u are off by p; y by act'(g) of g's error (at most 1.13)
times u and act(g) of u's, with a few roundings in f32 (16 of them cover the activation's). Backwards g and u are first rounded to
their type, which moves u by h u and act' by at most 0.8 (its own slope) h g, act by 1.13 h g; dg and du are rounded again: their errors
times the other factor, summed, bound what the products are off by, then p. Each output takes half a step of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["silu", "gelu", "sigmoid"]
U = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def make(M, N, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(M, K, generator=g).to(dtype), (torch.randn(2, N, K, generator=g) * 1.5 / math.sqrt(K)).to(dtype),
            torch.randn(M, N, generator=g).to(dtype))


def act_of(name, g):
    if name == "gelu":
        phi = torch.special.ndtr(g)
        return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    p = torch.sigmoid(g)
    return (g * p, p + g * p * (1 - p)) if name == "silu" else (p, p * (1 - p))


def near(got, ref, tol, name):
    assert got.shape == ref.shape, name
    half = torch.finfo(got.dtype).eps / 2
    err = (got.detach().double().cpu() - ref).abs()
    room = tol + half * (ref.abs() + tol) + LEAST[got.dtype]
    assert (err <= room).all(), (name, float((err / room).max()))


def p(terms, squares):
    return 2.0 ** -22 * (8 + 2 * math.sqrt(terms)) * squares.sqrt()


def check(x, w, dy, act, device=None, train=True):
    from yggdrasil_amd import ops
    dev = [t.cuda() for t in (x, w)] if device is None else device
    if train:
        xg, wg = [t.detach().requires_grad_() for t in dev]
    else:
        xg, wg = dev
    y = ops.gated_linear(xg, wg, act)
    assert y.dtype == x.dtype and y.is_contiguous()
    M, K = x.shape
    N = w.shape[1]
    x64, w64, dy64 = x.double(), w.double(), dy.double()
    g, u = x64 @ w64[0].t(), x64 @ w64[1].t()
    a, slope = act_of(act, g)
    tg, tu = p(K, x64 ** 2 @ (w64[0] ** 2).t()), p(K, x64 ** 2 @ (w64[1] ** 2).t())
    near(y, a * u, 1.13 * tg * (u.abs() + tu) + a.abs() * tu + 16 * U * (1 + g.abs()) * u.abs(), "y")
    if not train:
        return
    dx, dw = torch.autograd.grad(y, (xg, wg), dy.cuda())
    assert dx.dtype == x.dtype and dw.dtype == x.dtype
    h, least = torch.finfo(x.dtype).eps / 2, LEAST[x.dtype]
    eg, eu = tg + h * (g.abs() + tg) + least, tu + h * (u.abs() + tu) + least
    dg, du = dy64 * u * slope, dy64 * a
    rg = dy64.abs() * (eu * (slope.abs() + eg) + 0.8 * eg * u.abs() + 16 * U * u.abs()) + h * dg.abs() * 1.01 + least
    ru = dy64.abs() * (1.13 * eg + 16 * U * (1 + g.abs())) + h * du.abs() * 1.01 + least
    near(dx, dg @ w64[0] + du @ w64[1], rg @ w64[0].abs() + ru @ w64[1].abs() + p(2 * N, dg ** 2 @ w64[0] ** 2 + du ** 2 @ w64[1] ** 2) * 1.1,
         "dx")
    near(dw, torch.stack([dg.t() @ x64, du.t() @ x64]),
         torch.stack([r.t() @ x64.abs() + p(M, (d ** 2).t() @ x64 ** 2) * 1.1 for d, r in ((dg, rg), (du, ru))]), "dw")


SHAPES = [(1, 1, 1), (1, 8, 16), (2, 3, 5), (7, 17, 33), (16, 32, 64), (17, 33, 100), (40, 64, 8), (33, 100, 72), (64, 130, 256), (65, 63, 129),
          (129, 65, 1000), (200, 256, 264), (3, 520, 1030), (300, 129, 40)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_shapes(M, N, K, dtype, act):
    check(*make(M, N, K, dtype, seed=M + N), act)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, N, K", [(4100, 2056, 136), (2050, 4104, 72), (1030, 1100, 2040), (2000, 1001, 203), (16, 5000, 1024), (12, 4097, 511),
                                     (6150, 1100, 515), (1500, 1003, 1000)])
def test_large(M, N, K, dtype):
    """Whole and cut tiles of each kernel."""
    check(*make(M, N, K, dtype, seed=M), "silu")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_few_rows(dtype):
    """A served batch: one row to more than a tile."""
    for M in (1, 2, 5, 15, 16, 17, 31, 48, 65):
        check(*make(M, 200, 320, dtype, seed=M), "gelu", train=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, N, K", [(32, 4100, 136), (33, 2048, 520), (70, 1500, 72), (100, 1300, 1031), (256, 1024, 264), (250, 1000, 96),
                                     (512, 1020, 200), (17, 8200, 40), (64, 8190, 64)])
def test_few_tiles(M, N, K, dtype):
    """Batches between a tile's rows and many: each form of the kernel without a tile in LDS, and where they end."""
    check(*make(M, N, K, dtype, seed=N), "silu", train=M == 100)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_off_an_alignment_and_strides(dtype):
    x, w, dy = make(70, 96, 160, dtype, seed=1)
    for at in (1, 3):
        wide_x = torch.zeros(70, 200, dtype=dtype, device="cuda")
        wide_x[:, at:at + 160] = x.cuda()
        flat = torch.zeros(w.numel() + 8, dtype=dtype, device="cuda")
        flat[at:at + w.numel()] = w.cuda().reshape(-1)
        check(x, w, dy, "silu", (wide_x[:, at:at + 160], flat[at:at + w.numel()].view(w.shape)))
    check(x, w, dy, "silu", (x.t().contiguous().t().cuda(), w.transpose(1, 2).contiguous().transpose(1, 2).cuda()))


def test_leading_axes_and_no_rows():
    from yggdrasil_amd import ops
    x, w, dy = (t.cuda() for t in make(24, 40, 32, torch.float32, seed=2))
    whole = ops.gated_linear(x, w)
    assert torch.equal(ops.gated_linear(x.view(2, 3, 4, 32), w), whole.view(2, 3, 4, 40))
    assert torch.equal(ops.gated_linear(x[0], w)[None], ops.gated_linear(x[:1], w))
    e, w = torch.zeros(0, 5, 32, device="cuda", requires_grad=True), w.requires_grad_()
    y = ops.gated_linear(e, w)
    assert y.shape == (0, 5, 40)
    dx, dw = torch.autograd.grad(y.sum(), (e, w))
    assert dx.shape == e.shape and not dw.any()
    # sizes whose operands would be laid out anew, had they rows
    e, w = (torch.zeros(s, dtype=torch.bfloat16, device="cuda", requires_grad=True) for s in ((0, 777), (2, 4096, 777)))
    assert not torch.autograd.grad(ops.gated_linear(e, w).sum(), w)[0].any()


@pytest.mark.parametrize("act", ACTS)
def test_far_values(act):
    """Gates far from zero on both sides: the activation ends in 0, 1 or the gate itself, and its slope in 0 or 1."""
    from yggdrasil_amd import ops
    at = torch.tensor([-3e4, -200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 200.0, 3e4], device="cuda")[:, None].requires_grad_()
    w = torch.ones(2, 1, 1, device="cuda")
    w[1] = 0.5
    y = ops.gated_linear(at, w, act)
    ref = at.detach().double().cpu().requires_grad_()
    want = act_of(act, ref)[0] * ref * 0.5
    assert torch.allclose(y.detach().cpu().double(), want.detach(), rtol=1e-5, atol=1e-6)
    dx, = torch.autograd.grad(y.sum(), at)
    rx, = torch.autograd.grad(want.sum(), ref)
    assert torch.allclose(dx.cpu().double(), rx, rtol=1e-5, atol=1e-5)
    x = torch.ones(3, 4, device="cuda")
    x[1, 2] = math.nan
    y = ops.gated_linear(x, torch.ones(2, 5, 4, device="cuda"), act)
    assert y[1].isnan().all() and not y[::2].isnan().any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_some_gradients_alone(dtype):
    from yggdrasil_amd import ops
    x, w, dy = (t.cuda() for t in make(150, 90, 60, dtype, seed=3))
    leaves = [t.requires_grad_() for t in (x, w)]
    y = ops.gated_linear(*leaves)
    whole = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(whole, again))
    for i, leaf in enumerate(leaves):
        assert torch.equal(torch.autograd.grad(y, leaf, dy, retain_graph=True)[0], whole[i])
        others = [t.detach().requires_grad_(k == i) for k, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(ops.gated_linear(*others), others[i], dy)[0], whole[i])


@pytest.mark.parametrize("act", ACTS)
def test_against_differences(act):
    """With steps of 2^-6 a difference is off by 2^-12 times a third derivative of a few, and by roundings of 2^-24 over the step."""
    from yggdrasil_amd import ops
    x, w, dy = (t.cuda() for t in make(5, 7, 9, torch.float32, seed=4))
    leaves = [t.requires_grad_() for t in (x, w)]
    grads = torch.autograd.grad(ops.gated_linear(*leaves, act), leaves, dy)
    with torch.no_grad():
        for i, (leaf, grad) in enumerate(zip(leaves, grads)):
            for k in range(0, leaf.numel(), 4):
                ends = []
                for step in (2.0 ** -6, -2.0 ** -6):
                    moved = leaf.clone()
                    moved.view(-1)[k] += step
                    ends.append((ops.gated_linear(*[moved if j == i else t for j, t in enumerate(leaves)], act).double() * dy.double()).sum())
                assert abs((ends[0] - ends[1]) * 32 - grad.view(-1)[k].double()) < 2e-2


@pytest.mark.parametrize("M, N, K", [(1, 300, 256), (300, 200, 264), (2048, 4096, 64)])
def test_streams_and_graphs(M, N, K):
    from yggdrasil_amd import ops
    x, w, dy = (t.cuda() for t in make(M, N, K, torch.bfloat16, seed=5))
    leaves = [t.requires_grad_() for t in (x, w)]

    def both(leaves, dy):
        y = ops.gated_linear(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    want = both(leaves, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(leaves, dy)
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del want, got
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both(leaves, dy)
    for k in range(3):
        new = make(M, N, K, torch.bfloat16, seed=40 + k)
        with torch.no_grad():
            for t, v in zip((x, w, dy), new):
                t.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        fresh = [v.cuda() for v in new]
        want = both([t.requires_grad_() for t in fresh[:2]], fresh[2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(kept, want)), k


def test_refusals():
    from yggdrasil_amd import ops
    x, w = torch.zeros(3, 8, device="cuda"), torch.zeros(2, 5, 8, device="cuda")
    for bad in (lambda: ops.gated_linear(x, w[0]), lambda: ops.gated_linear(x, w[:1]), lambda: ops.gated_linear(x, w[..., :7]),
                lambda: ops.gated_linear(x.half(), w), lambda: ops.gated_linear(x, w.cpu()), lambda: ops.gated_linear(x, w, "relu"),
                lambda: ops.gated_linear(x, w, 0), lambda: ops.gated_linear(x, w[:, :0]), lambda: ops.gated_linear(x.double(), w.double()),
                lambda: ops.gated_linear(x[:, :0], w[..., :0]), lambda: ops.gated_linear(x, None)):
        with pytest.raises(ValueError):
            bad()
    x.requires_grad_()
    g, = torch.autograd.grad(ops.gated_linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ops.gated_linear(fwd.make_dual(x.detach(), torch.ones_like(x)), w)
