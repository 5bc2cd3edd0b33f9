"""The routed head of examples/routed_head.py: the three operators together on a model's states, its loss and gradient against
the same head in 64 bits, and its training."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "routed_head.py"
    spec = importlib.util.spec_from_file_location("routed_head", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_loss_and_gradient_against_64_bits():
    """The logits' two parts are rounded to bf16 (2^-8 of each), so logits are within 2^-7 of their size and the loss and the
    leaves' gradients, sums of p - [c = t] with p off by as much, within 2^-6 of the largest term."""
    m = example()
    g = torch.Generator().manual_seed(0)
    rows, n, V, E = 200, 64, 50, 9
    h = (torch.rand(rows, n, generator=g) * 2 - 1).to(torch.bfloat16).cuda()
    leaves = torch.randint(E, (rows,), generator=g).cuda()
    t = torch.randint(V, (rows,), generator=g, dtype=torch.int32).cuda()
    t[::7] = -1
    head = m.RoutedHead(V, E, n, "cuda")
    with torch.no_grad():
        head.w += (torch.randn(E, V, n, generator=g) / 8).to(torch.bfloat16).cuda()
    before = head.w.detach().double().clone()
    loss = head.step(h, leaves, t, 1.0)
    x = h.double()
    s = (x.abs().amax(1) / 127).float().double()[:, None]
    base = (torch.round((x / s).float()).double() @ head.q.double().t().contiguous()) * s * head.scale.double()
    logits = base + (before[leaves] * x[:, None, :]).sum(-1)
    logp = torch.log_softmax(logits, 1)
    given = t >= 0
    ref = -logp[given, t[given].long()].sum() / given.sum()
    off = 2.0 ** -7 * float(logits.abs().max())
    assert abs(float(loss) - float(ref)) <= 2 * off
    d = torch.exp(logp)
    d[given, t[given].long()] -= 1
    d = d * given[:, None] / given.sum()
    grad = torch.zeros_like(before).index_add_(0, leaves, d[:, :, None] * x[:, None, :])
    most = torch.zeros_like(before).index_add_(0, leaves, d.abs()[:, :, None] * x.abs()[:, None, :])
    p = torch.zeros_like(before).index_add_(0, leaves, (torch.exp(logp) * given[:, None] / given.sum())[:, :, None] * x.abs()[:, None, :])
    # the step's own rounding of w to bf16, the gradient's, and the probabilities'
    tol = 2.0 ** -8 * (before.abs() + grad.abs()) + 2.0 ** -7 * most + 4 * off * p + 1e-6
    assert ((before - grad - head.w.detach().double()).abs() <= tol).all()


def test_training_lowers_the_loss(capsys):
    losses, ids = example().main(steps=20)
    assert losses[-1] < losses[0] - 0.1 and all(b < a + 0.05 for a, b in zip(losses, losses[1:]))
    assert ids.shape[1] == 5 and "nats a token" in capsys.readouterr().out
