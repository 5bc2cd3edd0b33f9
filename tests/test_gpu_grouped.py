"""grouped_matmul and its gradients against products in 64 bits: every type, expert loads from none to all rows, sizes that
end inside a tile or off an alignment, rows in their own order, bad offsets.

Tolerance: an output is a sum of I products, each exact to a rounding in f32 and added in f32, so it is off by at most
2^-24 (I + 1) sum |a b|, and by far less in the mean: sqrt(I) roundings of random sign, each of a partial sum that is about
the root of the sum of squares of the products. Held here to 2^-22 (8 + 2 sqrt(I)) times that root, then half a step of the
output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def loads(kind, M, E, g):
    """Rows of each expert."""
    if kind == "even":
        leaves = torch.arange(M) % E
    elif kind == "one":
        leaves = torch.full((M,), E // 2)
    elif kind == "ends":
        leaves = torch.where(torch.arange(M) % 2 == 0, 0, E - 1)
    else:
        p = 1.0 / (1 + torch.arange(E, dtype=torch.double))
        leaves = torch.multinomial(p[torch.randperm(E, generator=g)], M, replacement=True, generator=g) if M else torch.zeros(0)
    return leaves.long()


def make(M, E, N, K, dtype, kind="ragged", ordered=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    leaves = loads(kind, M, E, g)
    if ordered:
        leaves = leaves[torch.randperm(M, generator=g)]
    else:
        leaves = leaves.sort().values
    x = torch.randn(M, K, generator=g).to(dtype)
    w = (torch.randn(E, N, K, generator=g) / math.sqrt(K)).to(dtype)
    dy = torch.randn(M, N, generator=g).to(dtype)
    return leaves, x, w, dy


def near(got, ref, a2, terms):
    """a2: sum of squares of the products of each output."""
    half = torch.finfo(got.dtype).eps / 2
    least = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[got.dtype]
    tol = 2.0 ** -23 * (8 + 2 * math.sqrt(terms)) * 2 * a2.sqrt()
    err = (got.detach().double().cpu() - ref).abs()
    assert (err <= tol + half * (ref.abs() + tol) + least).all(), float((err - tol - half * ref.abs()).max())


def check(leaves, x, w, dy, ordered, train=True):
    from yggdrasil_amd import ops
    E, N, K = w.shape
    M = len(x)
    dev = [v.cuda() for v in (x, w, dy)]
    xg, wg, dyg = dev
    if train:
        xg.requires_grad_()
        wg.requires_grad_()
    offsets, order = ops.group_rows(leaves.cuda(), E)
    y = ops.grouped_matmul(xg, wg, offsets, order if ordered else None)
    x64, w64, dy64 = x.double(), w.double(), dy.double()
    ref, sq = torch.zeros(M, N, dtype=torch.double), torch.zeros(M, N, dtype=torch.double)
    rx, sx = torch.zeros(M, K, dtype=torch.double), torch.zeros(M, K, dtype=torch.double)
    rw, sw = torch.zeros(E, N, K, dtype=torch.double), torch.zeros(E, N, K, dtype=torch.double)
    most = 1
    for e in torch.unique(leaves).tolist():
        if not 0 <= e < E:
            continue
        i = (leaves == e).nonzero()[:, 0]
        most = max(most, len(i))
        ref[i] = x64[i] @ w64[e].t()
        sq[i] = x64[i] ** 2 @ (w64[e] ** 2).t()
        if train:
            rx[i] = dy64[i] @ w64[e]
            sx[i] = dy64[i] ** 2 @ w64[e] ** 2
            rw[e] = dy64[i].t() @ x64[i]
            sw[e] = (dy64[i] ** 2).t() @ x64[i] ** 2
    assert y.dtype == x.dtype
    near(y, ref, sq, K)
    if train:
        dx, dw = torch.autograd.grad(y, (xg, wg), dyg)
        assert dx.dtype == x.dtype and dw.dtype == x.dtype
        near(dx, rx, sx, N)
        near(dw, rw, sw, most)
    return y


SHAPES = [(1, 1, 1, 1), (1, 4, 8, 16), (7, 3, 5, 3), (40, 16, 8, 64), (100, 300, 8, 128), (64, 5, 17, 33), (200, 4, 64, 256),
          (130, 9, 100, 72), (300, 2, 129, 200), (513, 3, 256, 136), (700, 2, 264, 520), (33, 2, 300, 1000), (1000, 8, 40, 24)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, E, N, K", SHAPES)
def test_shapes(M, E, N, K, dtype):
    for ordered in (False, True):
        leaves, x, w, dy = make(M, E, N, K, dtype, ordered=ordered, seed=M + N)
        check(leaves, x, w, dy, ordered)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kind", ["even", "one", "ends"])
@pytest.mark.parametrize("M, E, N, K", [(96, 32, 16, 64), (520, 6, 144, 96), (257, 3, 256, 512)])
def test_loads(M, E, N, K, kind, dtype):
    """Even loads, one expert that takes all rows, experts without a row between the first and the last."""
    leaves, x, w, dy = make(M, E, N, K, dtype, kind, True)
    check(leaves, x, w, dy, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_more_experts_than_rows(dtype):
    leaves, x, w, dy = make(50, 5000, 8, 32, dtype, ordered=True)
    check(leaves, x, w, dy, True)
    leaves, x, w, dy = make(3, 70, 96, 160, dtype)
    check(leaves, x, w, dy, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("M", [2000, 4500])
def test_tall(M, dtype):
    """Long groups: sums over thousands of rows in the weights' gradient, several tiles an expert."""
    leaves, x, w, dy = make(M, 3, 200, 264, dtype, ordered=True)
    check(leaves, x, w, dy, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_of_no_expert_are_zero(dtype):
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(90, 4, 24, 40, dtype, ordered=True)
    leaves[::3] = -1
    leaves[1::9] = 4
    y = check(leaves, x, w, dy, True)
    assert (y[::3] == 0).all()
    # offsets that end before the rows do: rows past the end
    offsets = torch.tensor([0, 10, 10, 20, 30], dtype=torch.int32, device="cuda")
    z = ops.grouped_matmul(x.cuda(), w.cuda(), offsets)
    assert (z[30:] == 0).all() and (z[:30] != 0).any()
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    dx, dw = torch.autograd.grad(ops.grouped_matmul(xg, wg, offsets), (xg, wg), dy.cuda())
    assert (dx[30:] == 0).all() and (dw[1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N, K", [(16, 64), (200, 328)])
def test_values_that_are_not_finite_stay_in_their_rows(N, K, dtype):
    """A NaN or an infinity in one row reaches that row's outputs and its expert's gradient alone."""
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(150, 3, N, K, dtype, "even")
    x[10, 3] = math.nan
    x[70, 0] = math.inf
    e = {int(leaves[10]), int(leaves[70])}
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    offsets, _ = ops.group_rows(leaves.cuda(), 3)
    y = ops.grouped_matmul(xg, wg, offsets)
    rows = [i for i in range(150) if i not in (10, 70)]
    assert torch.isfinite(y[rows]).all() and not torch.isfinite(y[10]).any() and not torch.isfinite(y[70]).any()
    dx, dw = torch.autograd.grad(y, (xg, wg), dy.cuda())
    assert torch.isfinite(dx).all()
    for k in range(3):
        assert torch.isfinite(dw[k]).all() == (k not in e)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, N, K", [(60, 8, 32), (400, 160, 192)])
def test_bad_offsets_and_orders_stay_in_bounds(M, N, K, dtype):
    """Offsets past the rows, falling or negative ones, an order with entries that are no rows: no access out of bounds (the
    kernels clamp the offsets and skip such entries), and the call ends."""
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(M, 4, N, K, dtype)
    bad = [[0, M + 50, 2 * M, 1 << 30, (1 << 31) - 1], [0, -5, M // 2, -(1 << 31), M], [5, 4, 3, 2, 1], [M, M, M, M, M]]
    order = torch.randperm(M, dtype=torch.int32)
    order[::7] = M + 3
    order[3::11] = -1
    for o in bad:
        for r in (None, order.cuda()):
            xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
            y = ops.grouped_matmul(xg, wg, torch.tensor(o, dtype=torch.int32, device="cuda"), r)
            torch.autograd.grad(y, (xg, wg), dy.cuda())
            torch.cuda.synchronize()


def test_strided_and_shared_inputs():
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(60, 4, 24, 40, torch.float32)
    offsets, _ = ops.group_rows(leaves.cuda(), 4)
    want = ops.grouped_matmul(x.cuda(), w.cuda(), offsets)
    wide = torch.zeros(60, 80, device="cuda")
    wide[:, ::2] = x.cuda()
    assert torch.equal(ops.grouped_matmul(wide[:, ::2], w.cuda(), offsets), want)
    wt = w.transpose(1, 2).contiguous().cuda()
    assert torch.equal(ops.grouped_matmul(x.cuda(), wt.transpose(1, 2), offsets), want)
    # one matrix for every expert, one row for all: their gradients are sums
    shared = w[:1].cuda().requires_grad_()
    one = x[:1].cuda().requires_grad_()
    y = ops.grouped_matmul(one.expand(60, 40), shared.expand(4, 24, 40), offsets)
    y.sum().backward()
    ref = torch.ones(24, 1, dtype=torch.double) * 60 * x[0].double()
    assert ((shared.grad[0].double().cpu() - ref).abs() <= 2.0 ** -20 * ref.abs() + 1e-30).all()
    ref = 60 * w[0].double().sum(0)
    assert ((one.grad[0].double().cpu() - ref).abs() <= 2.0 ** -19 * 60 * w[0].double().abs().sum(0)).all()
    e = ops.grouped_matmul(torch.empty(0, 40, device="cuda"), w.cuda(), torch.zeros(5, dtype=torch.int32, device="cuda"))
    assert e.shape == (0, 24)
    xe, we = torch.empty(0, 40, device="cuda", requires_grad=True), w.cuda().requires_grad_()
    ops.grouped_matmul(xe, we, torch.zeros(5, dtype=torch.int32, device="cuda")).sum().backward()
    assert (we.grad == 0).all()


def test_only_the_gradients_asked_for():
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(30, 4, 8, 16, torch.float32)
    offsets, _ = ops.group_rows(leaves.cuda(), 4)
    wg = w.cuda().requires_grad_()
    y = ops.grouped_matmul(x.cuda(), wg, offsets)
    y.backward(dy.cuda())
    assert wg.grad.shape == w.shape
    xg = x.cuda().requires_grad_()
    ops.grouped_matmul(xg, w.cuda(), offsets).backward(dy.cuda())
    assert xg.grad.shape == x.shape


def test_gradient_against_differences():
    """Central differences of the product in 64 bits: the function is linear in x and in w, so they are exact but for
    rounding; the kernel's own error is that of the sums above."""
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(40, 5, 12, 20, torch.float32, ordered=True)
    offsets, order = ops.group_rows(leaves.cuda(), 5)
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    dx, dw = torch.autograd.grad(ops.grouped_matmul(xg, wg, offsets, order), (xg, wg), dy.cuda())

    def f(a, b):
        return float((torch.einsum("mk,mnk->mn", a, b[leaves]) * dy.double()).sum())
    for s in range(4):
        g = torch.Generator().manual_seed(s)
        vx, vw = torch.randn(x.shape, generator=g).double(), torch.randn(w.shape, generator=g).double()
        for v, d, at in ((vx, dx, lambda h: f(x.double() + h * vx, w.double())),
                         (vw, dw, lambda h: f(x.double(), w.double() + h * vw))):
            want, got = (at(1e-3) - at(-1e-3)) / 2e-3, float((d.double().cpu() * v).sum())
            assert abs(got - want) <= 1e-4 * (1 + abs(want))


def test_same_result_every_time():
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(3000, 6, 72, 136, torch.bfloat16, ordered=True)
    offsets, order = ops.group_rows(leaves.cuda(), 6)
    runs = []
    for _ in range(3):
        xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        y = ops.grouped_matmul(xg, wg, offsets, order)
        runs.append((y.detach(), *torch.autograd.grad(y, (xg, wg), dy.cuda())))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


@pytest.mark.parametrize("M, E, N, K", [(24, 40, 8, 32), (500, 4, 160, 192)])
def test_streams_and_graphs(M, E, N, K):
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(M, E, N, K, torch.bfloat16)
    xg, wg = x.cuda(), w.cuda()
    offsets, order = ops.group_rows(leaves.cuda(), E)
    want = ops.grouped_matmul(xg, wg, offsets, order)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.grouped_matmul(xg, wg, offsets, order)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.grouped_matmul(xg, wg, offsets, order)
    for k in range(4):
        l2, x2, w2, _ = make(M, E, N, K, torch.bfloat16, seed=k + 5)
        o2, r2 = ops.group_rows(l2.cuda(), E)
        for a, b in ((xg, x2), (wg, w2), (offsets, o2), (order, r2)):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        want = ops.grouped_matmul(x2.cuda(), w2.cuda(), o2, r2)
        torch.cuda.synchronize()
        assert torch.equal(out, want), k


def test_group_rows():
    from yggdrasil_amd import ops
    leaves = torch.tensor([3, 0, 3, -1, 1, 9, 0], device="cuda")
    offsets, order = ops.group_rows(leaves, 5)
    assert offsets.tolist() == [0, 2, 3, 3, 5, 5] and order.tolist() == [1, 6, 4, 0, 2, 3, 5]
    assert offsets.dtype == order.dtype == torch.int32
    offsets, order = ops.group_rows(torch.empty(0, dtype=torch.int64, device="cuda"), 2)
    assert offsets.tolist() == [0, 0, 0] and order.numel() == 0


def test_refusals():
    from yggdrasil_amd import ops
    x, w = torch.zeros(6, 8, device="cuda"), torch.zeros(3, 4, 8, device="cuda")
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    ops.grouped_matmul(x, w, off)
    for a in ((x[0], w, off), (x, w[0], off), (x, w.half(), off), (x, w[:, :, :7], off), (x, w, off[:3]), (x, w, off.long()),
              (x, w, off.cpu()), (x, w, off, torch.zeros(5, dtype=torch.int32, device="cuda")),
              (x, w, off, torch.zeros(6, dtype=torch.int64, device="cuda")), (x.double(), w.double(), off), (x, w.cpu(), off),
              (x, w[:, :0], off), (x, w[:0], off[:1])):
        with pytest.raises(ValueError):
            ops.grouped_matmul(*a)
    with pytest.raises(ValueError):
        ops.group_rows(torch.zeros(3, device="cuda"), 2)
    with pytest.raises(ValueError):
        ops.group_rows(torch.zeros(3, dtype=torch.int32, device="cuda"), 0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, E, N, K, ordered", [
    (8192, 8, 2048, 2056, True), (5000, 16, 1528, 2040, False), (9000, 2, 4096, 264, True), (16384, 1, 2048, 1000, True),
    (3000, 16, 1000, 1000, True), (2500, 9, 1027, 2049, True), (1200, 8, 2101, 2051, True)])
def test_large_tiles(M, E, N, K, ordered, dtype):
    """Products large enough for the largest tiles, with rows of no expert, ends inside a tile and a step, more rows of one
    expert than a workgroup holds numbers of; against products in 64 bits on the GPU, to the tolerances above."""
    from yggdrasil_amd import ops
    g = torch.Generator("cuda").manual_seed(M + N)
    leaves = torch.randint(E, (M,), device="cuda", generator=g)
    leaves[torch.rand(M, device="cuda", generator=g) < 0.3] = E // 2
    leaves[:5] = -1
    if not ordered:
        leaves = torch.where(leaves < 0, E, leaves).sort().values
    offsets, order = ops.group_rows(leaves, E)
    x = torch.randn(M, K, device="cuda", generator=g).to(dtype).requires_grad_()
    w = (torch.randn(E, N, K, device="cuda", generator=g) / math.sqrt(K)).to(dtype).requires_grad_()
    dy = torch.randn(M, N, device="cuda", generator=g).to(dtype)
    y = ops.grouped_matmul(x, w, offsets, order if ordered else None)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x, w = x.detach(), w.detach()
    for e in range(-1, E):
        i = ((leaves < 0) | (leaves >= E) if e < 0 else leaves == e).nonzero()[:, 0]
        if e < 0:
            assert (y[i] == 0).all() and (dx[i] == 0).all()
            continue
        a, b, c = x[i].double(), w[e].double(), dy[i].double()
        bt, ct = b.t().contiguous(), c.t().contiguous()
        near(y[i], (a @ bt).cpu(), (a ** 2 @ bt ** 2).cpu(), K)
        near(dx[i], (c @ b).cpu(), (c ** 2 @ b ** 2).cpu(), N)
        near(dw[e], (ct @ a).cpu(), (ct ** 2 @ a ** 2).cpu(), max(len(i), 1))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N, K", [(8, 64), (20, 48), (64, 200), (33, 70)])
def test_long_experts_of_small_matrices(N, K, dtype):
    """Experts of 256 rows and more beside short ones, their first places on, before and after multiples of 256."""
    sizes = [256, 255, 1, 0, 257, 511, 0, 30, 1024, 16, 17, 700, 0]
    leaves = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes))
    g = torch.Generator().manual_seed(N)
    for ordered in (False, True):
        M = len(leaves)
        mine = leaves[torch.randperm(M, generator=g)] if ordered else leaves
        x, dy = torch.randn(M, K, generator=g).to(dtype), torch.randn(M, N, generator=g).to(dtype)
        w = (torch.randn(len(sizes), N, K, generator=g) / math.sqrt(K)).to(dtype)
        check(mine, x, w, dy, ordered)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, E, N, K", [(1, 3, 70, 1300), (7, 45, 200, 2111), (20, 9, 150, 1024), (63, 2, 90, 2056), (200, 100, 300, 513)])
def test_few_rows(M, E, N, K, dtype):
    """Few rows an expert and long reductions, at and off an alignment of 16 bytes."""
    leaves, x, w, dy = make(M, E, N, K, dtype, ordered=True, seed=M)
    check(leaves, x, w, dy, True)


@pytest.mark.parametrize("at", [1, 2, 4])
def test_operands_off_their_alignment(at):
    """x, w and dy that begin `at` elements into their storage, at sizes whose rows would be aligned."""
    from yggdrasil_amd import ops
    M, E, N, K = 2100, 4, 520, 2048
    leaves, x, w, dy = make(M, E, N, K, torch.bfloat16, "even", True)
    offsets, order = ops.group_rows(leaves.cuda(), E)

    def off(t):
        flat = torch.zeros(t.numel() + at, dtype=t.dtype, device="cuda")
        flat[at:] = t.reshape(-1).cuda()
        return flat[at:].view(t.shape)
    runs = []
    for f in (lambda t: t.cuda(), off):
        a, b = f(x).requires_grad_(), f(w).requires_grad_()
        y = ops.grouped_matmul(a, b, offsets, order)
        runs.append((y.detach(), *torch.autograd.grad(y, (a, b), f(dy))))
    for p, q in zip(*runs):      # another order of the same sums in f32, then the type's rounding
        assert ((p.double() - q.double()).abs() <= 2.0 ** -7 * q.double().abs() + 2.0 ** -10).all()


def test_second_derivatives_are_refused():
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(12, 3, 8, 16, torch.float32)
    offsets, _ = ops.group_rows(leaves.cuda(), 3)
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = ops.grouped_matmul(xg, wg, offsets)
    gx, gw = torch.autograd.grad(y, (xg, wg), dy.cuda(), create_graph=True)
    for g in (gx, gw):
        with pytest.raises(RuntimeError, match="second derivative"):
            g.sum().backward(retain_graph=True)


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwd
    from yggdrasil_amd import ops
    leaves, x, w, dy = make(12, 3, 8, 16, torch.float32)
    offsets, _ = ops.group_rows(leaves.cuda(), 3)
    x, w, dy = x.cuda(), w.cuda(), dy.cuda()
    with fwd.dual_level():
        for a, b in ((fwd.make_dual(x, x), w), (x, fwd.make_dual(w, w)), (fwd.make_dual(x, x)[:, ::2], w[:, :, ::2])):
            with pytest.raises(RuntimeError, match="forward"):
                ops.grouped_matmul(a, b, offsets)
        xg = x.clone().requires_grad_()
        y = ops.grouped_matmul(xg, w, offsets)
        with pytest.raises(RuntimeError, match="forward"):
            torch.autograd.grad(y, xg, fwd.make_dual(dy, dy))


def test_group_rows_takes_no_leaf_modulo_32_bits():
    """int64 leaves outside int32 belong to no expert, as others outside the range."""
    from yggdrasil_amd import ops
    leaves = torch.tensor([2 ** 32 + 1, 1, -2 ** 32, 0, 2 ** 31, -2 ** 63, 2 ** 63 - 1, 2, 2 ** 40 + 2, -2 ** 31 - 1], device="cuda")
    offsets, order = ops.group_rows(leaves, 3)
    assert offsets.tolist() == [0, 1, 2, 3] and order.tolist() == [3, 1, 7, 0, 2, 4, 5, 6, 8, 9]
    x, w = torch.randn(10, 16, device="cuda"), torch.randn(3, 8, 16, device="cuda", requires_grad=True)
    y = ops.grouped_matmul(x, w, offsets, order)
    none = [0, 2, 4, 5, 6, 8, 9]
    assert (y[none] == 0).all() and (y[[1, 3, 7]] != 0).all()
    x2 = x.clone()
    x2[none] = 0
    want, = torch.autograd.grad(ops.grouped_matmul(x2, w, offsets, order).sum(), w)
    got, = torch.autograd.grad(y.sum(), w)
    assert torch.equal(got, want)


@pytest.mark.parametrize("M, E, dtype", [(7, 5, torch.int32), (4096, 16384, torch.int32), (16001, 64, torch.int64),
                                         (65536, 1024, torch.int32)])
def test_group_rows_in_graphs(M, E, dtype):
    """Every replay, with eager work and synchronizations between them, equals the eager call."""
    from yggdrasil_amd import ops
    leaves = torch.randint(E, (M,), device="cuda", dtype=dtype)
    ops.group_rows(leaves, E)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        offsets, order = ops.group_rows(leaves, E)
    for k in range(5):
        now = torch.randint(-2, E + 2, (M,), device="cuda", dtype=dtype)
        leaves.copy_(now)
        g.replay()
        torch.cuda.synchronize()
        want = ops.group_rows(now, E)
        torch.cuda.synchronize()
        assert torch.equal(offsets, want[0]) and torch.equal(order, want[1]), k
