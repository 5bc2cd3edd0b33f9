"""gated_linear's weights' gradient over rows of more than 2^31 values: dy is zero but in the last rows, so it is that of the call on those
alone.

Tolerance: a call on fewer rows may add g and u in another order, so a dg or du next to a middle of two values of the type may be rounded
to the other one: h (half a step) of itself in either call, 2 h |d| together, times |x| and summed; g and u themselves are off by the 2^-16 that
they are kept to and less by their sums, which 1.02 covers. Each result is rounded too: 2 h of itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M, N, K", [(270_001, 4100, 64), (540_000, 2048, 200), (17_000, 600, 130_000)])
def test_weights_gradient(M, N, K, dtype):
    from yggdrasil_amd import ops
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("less than 80 GB of device memory free")
    assert M * max(2 * N, K) > 1 << 31
    g = torch.Generator("cuda").manual_seed(K)
    x = torch.randn(M, K, generator=g, device="cuda", dtype=dtype)
    w = (torch.randn(2, N, K, generator=g, device="cuda", dtype=dtype) / K ** 0.5).requires_grad_()
    dy = torch.zeros(M, N, device="cuda", dtype=dtype)
    dy[-300:] = torch.randn(300, N, generator=g, device="cuda", dtype=dtype)
    dw, = torch.autograd.grad(ops.gated_linear(x, w), w, dy)
    end, dy = x[-300:].clone(), dy[-300:].clone()
    want, = torch.autograd.grad(ops.gated_linear(end, w), w, dy)
    h = torch.finfo(dtype).eps / 2
    end, dy = end.float(), dy.float()
    a, u = (torch.mm(end, v.float().t()) for v in w.detach())
    p = torch.sigmoid(a)
    each = [torch.mm((dy * u * (p + a * p * (1 - p))).abs().t(), end.abs()), torch.mm((dy * a * p).abs().t(), end.abs())]
    for got, ref, most in zip(dw.float(), want.float(), each):
        err, room = (got - ref).abs(), 1.02 * 2 * h * (most + ref.abs()) + 2.0 ** -24
        assert (err <= room).all(), float((err / room).max())
        assert float(room.mean()) < 0.1 * float(ref.abs().mean())       # another row's products would show
    torch.cuda.empty_cache()
