"""int8_linear against the same quantisation with products in 64 bits: every type, one row to many, sizes that end inside a
tile or off an alignment, rows of zeros and of values that are not finite.

The integers are those of the definition (the quotient x / s rounded to f32, then to the nearest integer, ties to even), and
their sums are exact, so an output is off by three roundings in f32 (the sum's conversion and two products) and half a step
of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain(x, w, ws):
    x = x.double().cpu()
    bad = ~torch.isfinite(x).all(1)
    x = torch.where(bad[:, None], torch.zeros_like(x), x)
    s = (x.abs().amax(1) / 127).float().clamp_min(2.0 ** -126).double()[:, None]
    q = torch.round((x / s).float()).double()
    y = (q @ w.double().cpu().t()) * s * ws.double().cpu()
    y[bad] = math.nan
    return y


def check(x, w, ws):
    from yggdrasil_amd import ops
    y = ops.int8_linear(x, w, ws)
    ref = plain(x.reshape(-1, x.shape[-1]), w, ws)
    assert y.dtype == x.dtype and y.shape == x.shape[:-1] + (w.shape[0],)
    got = y.reshape(ref.shape).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    ok = torch.isfinite(ref)
    half, most = torch.finfo(y.dtype).eps / 2, torch.finfo(y.dtype).max
    least = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[y.dtype]
    far = ok & (ref.abs() > most * (1 - half))
    tol = (3 * 2.0 ** -24 + half) * ref.abs() * (1 + 2.0 ** -20) + least
    err = (got - ref).abs()
    assert (err <= tol)[ok & ~far].all(), float((err - tol)[ok & ~far].max())
    return y


def make(M, N, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype).cuda()
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8).cuda()
    ws = ((0.5 + torch.rand(N, generator=g)) / (73 * math.sqrt(K))).cuda()
    return x, w, ws


SIZES = [(1, 1, 1), (1, 8, 16), (1, 300, 1000), (2, 33, 77), (3, 256, 128), (4, 1000, 4096), (5, 64, 64), (16, 100, 512),
         (17, 257, 1001), (33, 129, 200), (64, 512, 256), (77, 503, 1000), (130, 260, 300), (256, 256, 512), (300, 600, 130),
         (513, 1030, 264), (1, 70, 8192), (2, 40, 33000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, N, K", SIZES)
def test_sizes(M, N, K, dtype):
    check(*make(M, N, K, dtype, M + K))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_rows_of_zeros_ties_and_values_that_are_not_finite(M, dtype):
    x, w, ws = make(M + 6, 96, 160, dtype)
    x[0] = 0
    x[1, 5] = math.nan
    x[2, 159] = math.inf
    x[3, 0] = -math.inf
    x[4] = (torch.arange(160) % 255 - 127).to(dtype) / 2     # halves of a step: ties to even
    x[4, 0] = 127.0
    x[5] = torch.finfo(dtype).tiny                           # the least normal values
    y = check(x, w, ws)
    assert (y[0] == 0).all() and torch.isnan(y[1:4]).all() and torch.isfinite(y[4]).all()
    if M == 1:
        for r in range(6):                                   # each of them as a call of its own
            check(x[r:r + 1].contiguous(), w, ws)


def test_sums_past_24_bits():
    """The longest sums of the largest products: 131072 x 127 x 128 stays in 32 bits."""
    K = 131072
    x = torch.full((2, K), 3.0, device="cuda")
    x[1] = -3.0
    w = torch.full((5, K), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    check(x, w, torch.full((5,), 1e-6, device="cuda"))


def test_extreme_scales():
    x, w, ws = make(40, 64, 256, torch.float32)
    x[0] *= 1e36 / x[0].abs().max()
    x[1] *= 1e-37
    x[2] = 1e-44                                             # below the least scale
    ws[3] = 0.0
    ws[4] = -1.0
    check(x, w, ws)


def test_shapes_views_and_streams():
    from yggdrasil_amd import ops
    x, w, ws = make(24, 70, 136, torch.bfloat16)
    want = check(x, w, ws)
    assert torch.equal(ops.int8_linear(x.reshape(2, 3, 4, 136), w, ws).reshape(24, 70), want)
    assert torch.equal(ops.int8_linear(x[0], w, ws), ops.int8_linear(x[:1], w, ws)[0])
    wide = torch.zeros(24, 272, dtype=torch.bfloat16, device="cuda")
    wide[:, 1::2] = x
    assert torch.equal(ops.int8_linear(wide[:, 1::2], w, ws), want)
    assert torch.equal(ops.int8_linear(x, w.t().contiguous().t(), ws), want)
    check(x[:1].expand(9, 136), w, ws)
    check(x[3:, 1:], w[:, 1:], ws)                           # rows off their alignment
    flat = torch.zeros(70 * 136 + 3, dtype=torch.int8, device="cuda")
    odd = flat[3:].view(70, 136)                             # a matrix off its alignment
    odd.copy_(w)
    assert torch.equal(ops.int8_linear(x, odd, ws), want)
    assert ops.int8_linear(x[:0], w, ws).shape == (0, 70)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.int8_linear(x, w, ws)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("M", [1, 24, 200])
def test_graphs(M):
    from yggdrasil_amd import ops
    x, w, ws = make(M, 200, 264, torch.bfloat16)
    ops.int8_linear(x, w, ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.int8_linear(x, w, ws)
    for k in range(4):
        x2, w2, ws2 = make(M, 200, 264, torch.bfloat16, k + 9)
        for a, b in ((x, x2), (w, w2), (ws, ws2)):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        want = ops.int8_linear(x2, w2, ws2)
        torch.cuda.synchronize()
        assert torch.equal(out, want), k


def test_quantize_weight_round_trip():
    from yggdrasil_amd import ops
    g = torch.Generator().manual_seed(1)
    w = torch.randn(50, 96, generator=g)
    q, s = ops.quantize_weight(w.cuda())
    hq, hs = ops.quantize_weight(w)
    assert torch.equal(q.cpu(), hq) and torch.equal(s.cpu(), hs)
    check(torch.randn(7, 96, generator=g).cuda(), q, s)


def test_refusals():
    from yggdrasil_amd import ops
    x, w, ws = make(4, 6, 8, torch.float32)
    for a in ((x, w.float(), ws), (x, w[:, :7], ws), (x, w, ws[:5]), (x, w, ws.double()), (x, w.cpu(), ws), (x, w[0], ws),
              (x.double(), w, ws), (x.int(), w, ws), (x, w[:0], ws[:0]), (x[:, :0], w[:, :0], ws)):
        with pytest.raises(ValueError):
            ops.int8_linear(*a)
    with pytest.raises(ValueError, match="gradient"):
        ops.int8_linear(x.requires_grad_(), w, ws)
    with torch.no_grad():
        ops.int8_linear(x, w, ws)


@pytest.mark.parametrize("M, N, K", [(4100, 4100, 1008), (4096, 4096, 2048), (5000, 3000, 1040), (4111, 4099, 333)])
def test_large_tiles(M, N, K):
    """Enough tiles for the largest ones, ends inside a tile and a step; the integers' products in 64 bits on the GPU."""
    from yggdrasil_amd import ops
    x, w, ws = make(M, N, K, torch.float32)
    s = (x.double().abs().amax(1) / 127).float().double()[:, None]
    ref = (torch.round((x.double() / s).float()).double() @ w.double().t().contiguous()) * s * ws.double()
    err = (ops.int8_linear(x, w, ws).double() - ref).abs()
    assert (err <= 4 * 2.0 ** -24 * ref.abs() * (1 + 2.0 ** -20) + 2.0 ** -126).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M, N, K", [(1, 50, 15), (1, 50, 16), (1, 50, 17), (8, 40, 1000), (8, 40, 8192), (9, 40, 1000), (7, 33, 2047),
                                     (32, 70, 1024), (33, 70, 1024), (77, 100, 2049), (1, 20, 33000), (600, 700, 64)])
def test_borders_between_the_kernels(M, N, K, dtype):
    check(*make(M, N, K, dtype, M + N + K))


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwd
    from yggdrasil_amd import ops
    x, w, ws = make(4, 6, 8, torch.float32)
    with fwd.dual_level():
        for a, s in ((fwd.make_dual(x, x), ws), (x, fwd.make_dual(ws, ws)), (fwd.make_dual(x, x).reshape(2, 2, 8), ws)):
            with pytest.raises((RuntimeError, ValueError), match="forward"), torch.no_grad():
                ops.int8_linear(a, w, s)


def test_no_gradient_of_the_scales():
    """As for x: refused where it would be asked for."""
    from yggdrasil_amd import ops
    x, w, ws = make(4, 6, 8, torch.float32)
    want = ops.int8_linear(x, w, ws)
    for s in (ws.clone().requires_grad_(), torch.nn.Parameter(ws.clone())):
        with pytest.raises(ValueError, match="gradient"):
            ops.int8_linear(x, w, s)
        with torch.no_grad():
            assert torch.equal(ops.int8_linear(x, w, s), want)


def test_as_many_rows_as_a_call_takes():
    """2^24 rows: their scales and integers come from two launches."""
    from yggdrasil_amd import ops
    M, N, K = 1 << 24, 2, 16
    x, w, ws = make(1 << 12, N, K, torch.float16)
    y = ops.int8_linear(x.repeat(M >> 12, 1), w, ws)
    assert torch.equal(y.view(-1, 1 << 12, N), check(x, w, ws).expand(M >> 12, 1 << 12, N))
