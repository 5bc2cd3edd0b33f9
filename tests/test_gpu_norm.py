"""layer_norm and its gradients against the formula in 64 bits: every type, rows from one value to those wider than a workgroup's
registers, weights of either type, rows off an alignment and apart.

Tolerances, with u = 2^-24 a rounding in f32 and D the most additions that a value of a row goes through on its way into a sum (32 in
a lane or n / 1024 of a wide row, 16 over lanes and waves): the mean is off by dm <= D u mean|x|, the variance by (D + 6) u of
itself and dm^2, so 1 / sqrt by half of that and 3 u of itself, z by that and by dm / sd. The sums over q and q z bring D u of their
magnitudes' means; dw and db bring the additions over the rows. Then half a step of the output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def make(rows, n, dtype, wide=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    w_type = torch.float32 if wide else dtype
    x = (torch.randn(rows, n, generator=g) * (0.2 + torch.rand(n, generator=g)) + torch.randn(rows, 1, generator=g)).to(dtype)
    w, b = (1 + 0.3 * torch.randn(n, generator=g)).to(w_type), torch.randn(n, generator=g).to(w_type)
    return x, w, b, torch.randn(rows, n, generator=g).to(dtype)


def near(got, ref, tol):
    assert got.shape == ref.shape
    half = torch.finfo(got.dtype).eps / 2
    err = (got.detach().double().cpu() - ref).abs()
    room = tol + half * (ref.abs() + tol) + LEAST[got.dtype]
    assert (err <= room).all(), float((err / room).max())


def check(x, w, b, dy, eps=1e-5, device_x=None):
    from yggdrasil_amd import ops
    xg = (x.cuda() if device_x is None else device_x).detach().requires_grad_()
    wg, bg = (None if t is None else t.cuda().requires_grad_() for t in (w, b))
    y = ops.layer_norm(xg, wg, bg, eps)
    n, rows = x.shape[-1], x[..., 0].numel()
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    x64, dy64 = x.double().reshape(-1, n), dy.double().reshape(-1, n)
    w64 = torch.ones(n).double() if w is None else w.double()
    b64 = torch.zeros(n).double() if b is None else b.double()
    D = 48 + n / 1024
    m = x64.mean(-1, keepdim=True)
    var = ((x64 - m) ** 2).mean(-1, keepdim=True)
    rs = 1 / torch.sqrt(var + eps)
    z = (x64 - m) * rs
    dm = D * U * x64.abs().mean(-1, keepdim=True) + U * m.abs()
    rel = 0.5 * ((D + 6) * U + dm ** 2 * rs ** 2) + 3 * U
    dz = z.abs() * (rel + 2 * U) + dm * rs
    near(y.reshape(-1, n), z * w64 + b64, w64.abs() * dz + 2 * U * ((z * w64).abs() + b64.abs()))
    given = [t for t in (xg, wg, bg) if t is not None]
    grads = list(torch.autograd.grad(y, given, dy.cuda()))
    assert [g.dtype for g in grads] == [t.dtype for t in given]
    q = w64 * dy64
    s1, s2 = q.mean(-1, keepdim=True), (q * z).mean(-1, keepdim=True)
    d1 = (D + 2) * U * q.abs().mean(-1, keepdim=True)
    d2 = (D + 3) * U * (q * z).abs().mean(-1, keepdim=True) + (q.abs() * dz).mean(-1, keepdim=True)
    dx = (q - s1 - z * s2) * rs
    tol = rs * (6 * U * (q.abs() + s1.abs() + (z * s2).abs()) + d1 + z.abs() * d2 + (s2.abs() + d2) * dz) + rel * dx.abs()
    near(grads.pop(0).reshape(-1, n), dx, tol)
    R = 64 + rows / 256
    if w is not None:
        near(grads.pop(0), (dy64 * z).sum(0), R * U * (dy64 * z).abs().sum(0) + (dy64.abs() * dz).sum(0))
    if b is not None:
        near(grads.pop(0), dy64.sum(0), R * U * dy64.abs().sum(0))


SIZES = [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 129, 255, 256, 257, 500, 512, 513, 1000, 1023, 1024, 1025, 2047,
         2048, 2049, 4095, 4096, 4100, 5003, 8192, 8193, 16384, 16385, 20000, 32768, 33000]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", SIZES)
def test_sizes(n, dtype):
    for rows, wide in ((1, True), (5, False), (70, True)):
        check(*make(rows, n, dtype, wide, seed=n + rows))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows, n", [(20000, 8), (9001, 40), (5000, 200), (2100, 1000), (1500, 2100), (700, 9000)])
def test_more_rows_than_workgroups(rows, n, dtype):
    check(*make(rows, n, dtype, seed=rows))


@pytest.mark.parametrize("n", [131072, 100001])
def test_widest(n):
    for dtype in DTYPES:
        check(*make(3, n, dtype, seed=1))


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_without_weight_or_bias(which, dtype):
    for wide in (True, False):
        x, w, b, dy = make(33, 300, dtype, wide, seed=3)
        check(x, w if which == "weight" else None, b if which == "bias" else None, dy)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_apart_and_off_an_alignment(dtype):
    x, w, b, dy = make(37, 515, dtype, seed=4)
    whole = torch.full((37, 600), 9.0, dtype=dtype, device="cuda")
    for at in (0, 1, 3, 8):
        part = whole[:, at:at + 515]
        part.copy_(x)
        check(x, w, b, dy, device_x=part)
    check(x, w, b, dy, device_x=x.t().contiguous().t().cuda())
    assert (whole[:, -70:] == 9.0).all()


def test_leading_axes_and_no_rows():
    from yggdrasil_amd import ops
    x, w, b, dy = make(24, 130, torch.float32, seed=5)
    check(x.reshape(2, 3, 4, 130), w, b, dy.reshape(2, 3, 4, 130))
    check(x[0], w, b, dy[0])
    e, w, b = torch.zeros(0, 3, 130, device="cuda", requires_grad=True), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    y = ops.layer_norm(e, w, b)
    assert y.shape == e.shape
    g = torch.autograd.grad(y.sum(), (e, w, b))
    assert g[0].shape == e.shape and not g[1].any() and not g[2].any()


def test_far_from_zero_and_constant_rows():
    """A mean that is thousands of deviations, a row of one value (variance 0), no eps, rows of an infinity or NaN."""
    from yggdrasil_amd import ops
    x, w, b, dy = make(40, 700, torch.float32, seed=6)
    x = x + 3000.0
    x[1] = 5.0
    check(x, w, b, dy)
    x[2, 3], x[3, 4] = math.inf, math.nan
    y = ops.layer_norm(x.cuda(), w.cuda(), b.cuda())
    assert y[2:4].isnan().all() and not y[:2].isnan().any() and not y[4:].isnan().any()
    assert ops.layer_norm(torch.full((1, 9), 2.0, device="cuda"), eps=0.0).isnan().all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", [48, 500, 3000, 40000])
def test_some_gradients_alone(n, dtype):
    """Each input's gradient by itself equals the one of all together, and comes out the same every time."""
    from yggdrasil_amd import ops
    x, w, b, dy = (t.cuda() for t in make(60, n, dtype, seed=7))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ops.layer_norm(*leaves)
    whole = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for i, leaf in enumerate(leaves):
        assert torch.equal(torch.autograd.grad(y, leaf, dy, retain_graph=True)[0], whole[i])
        others = [t.detach().requires_grad_(k == i) for k, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(ops.layer_norm(*others), others[i], dy)[0], whole[i])
    only_bias = b.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x.detach(), None, only_bias), only_bias, dy)[0], whole[2])


def test_against_differences():
    """The gradients against differences of the operator itself: with steps of 2^-6 the difference's own error is of third order,
    2^-12 times third derivatives of a few, and roundings in y bring 2^-24 / 2^-6 times the values."""
    from yggdrasil_amd import ops
    x, w, b, dy = (t.cuda() for t in make(4, 24, torch.float32, seed=8))
    x = x * 2
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
    with torch.no_grad():
        for i, (leaf, grad) in enumerate(zip(leaves, grads)):
            for k in range(0, leaf.numel(), 5):
                ends = []
                for step in (2.0 ** -6, -2.0 ** -6):
                    moved = leaf.clone()
                    moved.view(-1)[k] += step
                    args = [moved if j == i else t for j, t in enumerate(leaves)]
                    ends.append((ops.layer_norm(*args).double() * dy.double()).sum())
                assert abs((ends[0] - ends[1]) / 2.0 ** -5 - grad.view(-1)[k].double()) < 2e-2


@pytest.mark.parametrize("rows, n", [(1, 256), (300, 2048), (6, 40000)])
def test_streams_and_graphs(rows, n):
    from yggdrasil_amd import ops
    x, w, b, dy = (t.cuda() for t in make(rows, n, torch.bfloat16, seed=9))
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def both():
        y = ops.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del want, got
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    for k in range(3):
        new = make(rows, n, torch.bfloat16, seed=20 + k)
        with torch.no_grad():
            for t, v in zip((x, w, b, dy), new):
                t.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        fresh = [v.cuda() for v in new]
        own = [t.requires_grad_() for t in fresh[:3]]
        y = ops.layer_norm(*own)
        want = (y, *torch.autograd.grad(y, own, fresh[3]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(kept, want)), k


def test_refusals():
    from yggdrasil_amd import ops
    x, w = torch.zeros(3, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x, w[:7]), lambda: ops.layer_norm(x, w.cpu()),
                lambda: ops.layer_norm(x, w.half()), lambda: ops.layer_norm(x.half(), w, w.half()), lambda: ops.layer_norm(x, eps=-1.0),
                lambda: ops.layer_norm(x, eps=math.nan), lambda: ops.layer_norm(x, eps="a"), lambda: ops.layer_norm(x[:, :0]),
                lambda: ops.layer_norm(x, w[None]), lambda: ops.layer_norm(torch.zeros(1, ops.MOST_INNER + 1, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    x.requires_grad_()
    g, = torch.autograd.grad(ops.layer_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ops.layer_norm(fwd.make_dual(x.detach(), torch.ones_like(x)), w)
