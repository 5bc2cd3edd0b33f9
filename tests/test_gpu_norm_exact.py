"""layer_norm where its values are known exactly or nearly so: rows of one value, whose z is 0, and rows far from zero whose mean f32
holds. Every form of the kernels: rows of less than a piece, of a few lanes, a wave, a workgroup, wider than registers.

Tolerance for rows of whole numbers about a whole mean, where sums and deviations are exact in f32: z is (x - m) times 1 / sqrt(variance +
eps), which the division by n, the sum with eps, the root, the reciprocal and the product round (at most 1.5 + 0.5 + 1 + 0.5 roundings
of 2^-24 and one for eps itself): 5 u of z, with the weight and the bias 2 u more of each term. Then half a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24
SIZES = [1, 2, 3, 5, 8, 9, 16, 40, 64, 100, 300, 1000, 1500, 2048, 5003, 9000, 12000, 16384, 20000, 33000, 70000]


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", SIZES)
def test_rows_of_one_value(n, dtype, wide):
    """Few bits, whose sums f32 holds: z is 0, y the bias, the weight's gradient 0."""
    from yggdrasil_amd import ops
    g = torch.Generator().manual_seed(n)
    kind = torch.float32 if wide else dtype
    w, b = (torch.randn(n, generator=g).to(kind).cuda().requires_grad_() for _ in range(2))
    value = torch.tensor([14336.0, -10240.0, 0.0, 11264.0, 13.0, 5 * 2.0 ** -12])
    x = value[:, None].repeat(1, n).to(dtype).cuda().requires_grad_()
    dy = torch.randn(6, n, generator=g).to(dtype).cuda()
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y, b.detach().to(dtype).expand(6, n))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert not dw.any()
    assert dx.isfinite().all() and (n > 1 or not dx.any())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", [2, 6, 8, 24, 64, 100, 300, 1000])
def test_rows_far_from_zero(n, dtype):
    """-2 to 2 about a mean that the type holds steps of 1 at, in f32 as far as 3000; rows of up to a wave, whose mean comes out whole (those of
    more are joined from their waves' means, which are rounded)."""
    from yggdrasil_amd import ops
    mean = {torch.float32: 3000.0, torch.bfloat16: 128.0, torch.float16: 1024.0}[dtype]
    g = torch.Generator().manual_seed(n)
    off = torch.randint(0 if dtype == torch.bfloat16 else -2, 3, (20, n // 2), generator=g)
    if dtype == torch.bfloat16:      # steps of 1 from 128 up to 256 alone
        off = torch.cat([off, 4 - off], 1)
        m = mean + 2
    else:
        off = torch.cat([off, -off], 1)
        m = mean
    if dtype == torch.float16:       # and of float16 from 1024 on
        off, m = off + 2, m + 2
    off = off[:, torch.randperm(n, generator=g)].double()
    x = mean + off
    assert torch.equal(x.to(dtype).double(), x) and (x.mean(1) == m).all()
    w, b = 1 + 0.3 * torch.randn(n, generator=g), torch.randn(n, generator=g)
    z = (x - m) / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + 1e-5)
    xg, wg = x.to(dtype).cuda().requires_grad_(), w.cuda().requires_grad_()
    y = ops.layer_norm(xg, wg, b.cuda())
    ref, room = z * w.double() + b.double(), 7 * U * (z * w.double()).abs() + 2 * U * b.double().abs()
    half = torch.finfo(dtype).eps / 2
    err = (y.detach().cpu().double() - ref).abs()
    assert (err <= room + half * (ref.abs() + room)).all(), float((err / (room + half * (ref.abs() + room))).max())
    dy = torch.randint(-3, 4, (20, n), generator=g)
    dw, = torch.autograd.grad(y, wg, dy.to(dtype).cuda())
    ref, each = (dy * z).sum(0), (dy * z).abs().sum(0)
    err = (dw.cpu().double() - ref).abs()
    assert (err <= (5 + 20) * U * each + U * ref.abs()).all(), float((err / each.clamp_min(1e-9)).max())
