"""The recurrent block's operators on tensors of more than 2^31 values: what lies at their end against the same call on the end alone, forward
and backward. A call on fewer rows may add in another order: tolerances are four steps of the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -8     # of bf16


def near(a, b):
    a, b = a.detach().float(), b.detach().float()
    assert ((a - b).abs() <= 4 * STEP * (b.abs() + 1e-2 * float(b.abs().max()))).all()


def of(shape, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("less than 80 GB of device memory free")
    yield
    torch.cuda.empty_cache()


def test_layer_norm():
    from yggdrasil_amd import ops
    rows, n = 2_200_003, 1000
    x, dy = of((rows, n), 0).requires_grad_(), of((rows, n), 1)
    y = ops.layer_norm(x)
    dx, = torch.autograd.grad(y, x, dy)
    end = x.detach()[-300:].clone().requires_grad_()
    want = ops.layer_norm(end)
    near(y[-300:], want)
    near(dx[-300:], torch.autograd.grad(want, end, dy[-300:].clone())[0])


@pytest.mark.parametrize("B, T, n", [(3, 700_001, 1030), (300, 4000, 1800)])
def test_gated_scan(B, T, n):
    """Gates of 0 begin anew near the end, so that it does not depend on what comes before."""
    from yggdrasil_amd import ops
    gate = torch.sigmoid(of((B, T, n), 2))
    gate[:, -200] = 0
    x, dh = of((B, T, n), 3).requires_grad_(), of((B, T, n), 4)
    gate.requires_grad_()
    h, last = ops.gated_scan(gate, x)
    dg, dx = torch.autograd.grad(h, (gate, x), dh)
    ends = [t.detach()[-1:, -200:].clone().requires_grad_() for t in (gate, x)]
    want, want_last = ops.gated_scan(*ends)
    near(h[-1:, -200:], want)
    near(last[-1:], want_last)
    wg, wx = torch.autograd.grad(want, ends, dh[-1:, -200:].clone())
    near(dx[-1:, -200:], wx)
    near(dg[-1:, -199:], wg[:, 1:])


@pytest.mark.parametrize("M, N, K", [(270_001, 4100, 64), (540_000, 2048, 200)])
def test_gated_linear(M, N, K):
    from yggdrasil_amd import ops
    x, w, dy = of((M, K), 5).requires_grad_(), (of((2, N, K), 6) / 16).requires_grad_(), of((M, N), 7)
    y = ops.gated_linear(x, w)
    dx, = torch.autograd.grad(y, x, dy)
    end = x.detach()[-300:].clone().requires_grad_()
    want = ops.gated_linear(end, w.detach())
    near(y[-300:], want)
    near(dx[-300:], torch.autograd.grad(want, end, dy[-300:].clone())[0])


def test_clip_grad_norm():
    from yggdrasil_amd import ops
    v = torch.ones((1 << 31) + 4099, dtype=torch.bfloat16, device="cuda")
    v[-1] = 3.0
    norm = float(v.numel() + 8) ** 0.5
    (out,), got = ops.clip_grad_norm([v], norm / 2)
    assert abs(float(got) - norm) <= norm * 2.0 ** -23
    assert (out[:-1] == 0.5).all() and float(out[-1]) == 1.5
