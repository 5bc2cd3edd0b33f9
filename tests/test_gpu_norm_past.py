"""layer_norm of results so large that they are written past the caches (256 MB in whole lines, or rows of 4096 bytes and more), with weight and
bias and their gradients over that many rows, against 64 bits; and what an infinity or a NaN reaches.

Tolerances as a row's sums bring them, u = 2^-24, D = 48 + n / 1024 additions on a value's way into one: the mean is off by dm = D u mean|x| +
u |mean|, 1 / sqrt(variance + eps) by rel = (D + 6) u / 2 + 3 u and the mean's part, z by both; dw and db go through at most 64 + rows / 256
additions. Then half a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def near(got, ref, tol, name):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.detach().double() - ref).abs()
    room = tol + half * (ref.abs() + tol) + 2.0 ** -25
    assert (err <= room).all(), (name, float((err / room).max()))


@pytest.mark.parametrize("rows, n, dtype", [(65541, 2048, torch.bfloat16), (65003, 1037, torch.float32), (33001, 4100, torch.float16),
                                            (16501, 8200, torch.bfloat16), (8300, 8200, torch.float32), (7001, 20001, torch.bfloat16),
                                            (3501, 20000, torch.float32), (1001, 70001, torch.float32)])
def test_past_the_caches(rows, n, dtype):
    from yggdrasil_amd import ops
    size = torch.finfo(dtype).bits // 8
    assert rows * n * size >= 1 << 28 and (n * size % 128 == 0 or n * size >= 4096)
    g = torch.Generator("cuda").manual_seed(n)
    x = torch.randn(rows, n, generator=g, device="cuda").to(dtype).requires_grad_()
    w, b = (torch.randn(n, generator=g, device="cuda").requires_grad_() for _ in range(2))
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    D, w64, b64 = 48 + n / 1024, w.detach().double(), b.detach().double()
    rw, tw, rb, tb = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(4))
    R = 64 + rows / 256
    for at in range(0, rows, 2048):
        part = slice(at, at + 2048)
        v, d = x.detach()[part].double(), dy[part].double()
        m = v.mean(-1, keepdim=True)
        rs = 1 / torch.sqrt(((v - m) ** 2).mean(-1, keepdim=True) + 1e-5)
        z = (v - m) * rs
        dm = D * U * v.abs().mean(-1, keepdim=True) + U * m.abs()
        rel = 0.5 * ((D + 6) * U + dm ** 2 * rs ** 2) + 3 * U
        dz = z.abs() * (rel + 2 * U) + dm * rs
        near(y[part], z * w64 + b64, w64.abs() * dz + 2 * U * ((z * w64).abs() + b64.abs()), "y")
        q = w64 * d
        s1, s2 = q.mean(-1, keepdim=True), (q * z).mean(-1, keepdim=True)
        d1 = (D + 2) * U * q.abs().mean(-1, keepdim=True)
        d2 = (D + 3) * U * (q * z).abs().mean(-1, keepdim=True) + (q.abs() * dz).mean(-1, keepdim=True)
        want = (q - s1 - z * s2) * rs
        tol = rs * (6 * U * (q.abs() + s1.abs() + (z * s2).abs()) + d1 + z.abs() * d2 + (s2.abs() + d2) * dz) + rel * want.abs()
        near(dx[part], want, tol, "dx")
        rw += (d * z).sum(0)
        tw += (R * U * (d * z).abs() + d.abs() * dz).sum(0)
        rb += d.sum(0)
        tb += R * U * d.abs().sum(0)
    near(dw, rw, tw, "dw")
    near(db, rb, tb, "db")


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n", [5, 9, 37, 130, 515, 1003, 2500, 5003, 9001, 13001, 17001, 66001])
def test_values_that_are_not_finite(n, dtype, bad):
    """Of dy one stays in its row of dx and its column of dw and db; of the weight in its column of y, and in all rows of dx; of x in its row of y
    and dx, and in all of dw. What it does not reach is as it was."""
    from yggdrasil_amd import ops
    g = torch.Generator().manual_seed(n)
    x, dy = (torch.randn(7, n, generator=g).to(dtype).cuda() for _ in range(2))
    w, b = (torch.randn(n, generator=g).cuda() for _ in range(2))

    def call(x, w, dy):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = ops.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    y, dx, dw, db = call(x, w, dy)
    rows = torch.arange(7, device="cuda") != 3
    for col in sorted({0, n // 2, max(n - 9, 0), n - 4, n - 1}):
        cols = torch.arange(n, device="cuda") != col
        t = dy.clone()
        t[3, col] = bad
        y1, dx1, dw1, db1 = call(x, w, t)
        assert torch.equal(y1, y) and torch.equal(dx1[rows], dx[rows]) and not dx1[3].isfinite().any()
        assert torch.equal(dw1[cols], dw[cols]) and torch.equal(db1[cols], db[cols])
        assert not dw1[col].isfinite() and not db1[col].isfinite()
        t = w.clone()
        t[col] = bad
        y1, dx1, dw1, db1 = call(x, t, dy)
        assert torch.equal(y1[:, cols], y[:, cols]) and not y1[:, col].isfinite().any() and not dx1.isfinite().any()
        assert torch.equal(dw1, dw) and torch.equal(db1, db)
        t = x.clone()
        t[3, col] = bad
        y1, dx1, dw1, db1 = call(t, w, dy)
        assert torch.equal(y1[rows], y[rows]) and torch.equal(dx1[rows], dx[rows])
        assert y1[3].isnan().all() and dx1[3].isnan().all() and dw1.isnan().all() and torch.equal(db1, db)
