"""A recurrent block of the operators together, as a program trains and serves it: norm, gated projections, gated recurrence, norm, gated
feed-forward, the tokens' log-probabilities, the gradients of all parameters and their clipping.

Tolerance in f32 against 64 bits, of a value relative to the largest of its tensor: each of the dozen operations on its way is off by at
most 64 roundings of 2^-24 (sums of up to 300 terms of mixed signs), and hands errors on enlarged at most twofold on the average of
a path (the norms' 1 / sd is about 1, the others contract): 12 * 64 * 2^-24 * 5 = 2^-12."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -12


class Plain:
    """The operators' formulas in elementary torch, in the inputs' type."""

    @staticmethod
    def layer_norm(x, w, b):
        off = x - x.mean(-1, keepdim=True)
        return off / torch.sqrt((off * off).mean(-1, keepdim=True) + 1e-5) * w + b

    @staticmethod
    def gated_linear(x, w, act):
        g, u = x @ w[0].t(), x @ w[1].t()
        return (g * torch.sigmoid(g) if act == "silu" else g * torch.special.ndtr(g)) * u

    @staticmethod
    def gated_scan(gate, x, state):
        out = []
        for t in range(x.shape[1]):
            state = gate[:, t] * state + x[:, t]
            out.append(state)
        return torch.stack(out, 1), state

    @staticmethod
    def logp(logits, targets):
        return torch.log_softmax(logits, -1).gather(-1, targets[..., None].long())[..., 0]


class Own:
    @staticmethod
    def layer_norm(x, w, b):
        from yggdrasil_amd import ops
        return ops.layer_norm(x, w, b)

    @staticmethod
    def gated_linear(x, w, act):
        from yggdrasil_amd import ops
        return ops.gated_linear(x, w, act)

    @staticmethod
    def gated_scan(gate, x, state):
        from yggdrasil_amd import ops
        return ops.gated_scan(gate, x, state)

    @staticmethod
    def logp(logits, targets):
        from yggdrasil_amd import ops
        return ops.token_logprobs(logits, targets).logp


def parameters(n=48, wide=96, vocab=40, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return [1 + 0.1 * r(n), 0.1 * r(n), r(n, n) / math.sqrt(n), 2 + r(n), r(2, n, n) / math.sqrt(n), 1 + 0.1 * r(n), 0.1 * r(n),
            r(2, wide, n) / math.sqrt(n), r(n, wide) / math.sqrt(wide), r(vocab, n) / math.sqrt(n)]


def block(f, p, x, state):
    """x (B, T, n) -> logits, the last state"""
    w1, b1, w_gate, b_gate, w_in, w2, b2, w_up, w_down, head = p
    z = f.layer_norm(x, w1, b1)
    h, last = f.gated_scan(torch.sigmoid(z @ w_gate.t() + b_gate), f.gated_linear(z, w_in, "silu"), state)
    x = x + h
    x = x + f.gated_linear(f.layer_norm(x, w2, b2), w_up, "gelu") @ w_down.t()
    return x @ head.t(), last


def loss_of(f, p, x, state, targets):
    logits, last = block(f, p, x, state)
    return -f.logp(logits, targets).mean(), logits, last


def near(got, ref, name):
    assert got.shape == ref.shape, name
    assert float((got.detach().double().cpu() - ref).abs().max()) <= TOL * max(float(ref.abs().max()), 1e-6), name


@pytest.mark.parametrize("B, T", [(1, 1), (3, 7), (2, 130), (1, 2100)])
def test_training_step_against_64_bits(B, T):
    from yggdrasil_amd import ops
    g = torch.Generator().manual_seed(B + T)
    x, state, targets = torch.randn(B, T, 48, generator=g), torch.randn(B, 48, generator=g), torch.randint(40, (B, T), generator=g)
    p = parameters()
    p64 = [t.double().requires_grad_() for t in p]
    s64 = state.double().requires_grad_()
    loss, logits, last = loss_of(Plain, p64, x.double(), s64, targets)
    ref = torch.autograd.grad(loss, [*p64, s64])
    dev = [t.cuda().requires_grad_() for t in p]
    sd = state.cuda().requires_grad_()
    got, got_logits, got_last = loss_of(Own, dev, x.cuda(), sd, targets.cuda())
    grads = torch.autograd.grad(got, [*dev, sd])
    near(got_logits, logits.detach(), "logits")
    near(got_last, last.detach(), "last")
    near(got, loss.detach(), "loss")
    for i, (a, r) in enumerate(zip(grads, ref)):
        near(a, r, i)
    norm = torch.sqrt(sum((r * r).sum() for r in ref))
    clipped, got_norm = ops.clip_grad_norm(grads, 0.5 * float(norm))
    near(got_norm, norm, "norm")
    for i, (a, r) in enumerate(zip(clipped, ref)):
        near(a, 0.5 * r, i)


def test_served_step_by_step():
    """One token at a time with the state carried on gives the sequence's logits."""
    g = torch.Generator().manual_seed(1)
    x, state = torch.randn(4, 70, 48, generator=g), torch.randn(4, 48, generator=g)
    p = [t.cuda() for t in parameters(seed=1)]
    ref, ref_last = block(Plain, [t.double() for t in parameters(seed=1)], x.double(), state.double())
    s, steps = state.cuda(), []
    for t in range(70):
        logits, s = block(Own, p, x[:, t:t + 1].cuda(), s)
        steps.append(logits)
    near(torch.cat(steps, 1), ref, "logits")
    near(s, ref_last, "last")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_training_step_in_a_graph(dtype):
    """A whole step (forward, backward, clipping in place, the parameters' update) captured and replayed is the eager one each time."""
    from yggdrasil_amd import ops

    def step(p, x, state, targets):
        loss, _, last = loss_of(Own, p, x, state, targets)
        grads, norm = ops.clip_grad_norm(torch.autograd.grad(loss, p), 0.1)
        with torch.no_grad():
            for t, d in zip(p, grads):
                t -= 0.5 * d
        return loss.detach(), last.detach(), norm

    def data(seed):
        g = torch.Generator().manual_seed(seed)
        return (torch.randn(2, 140, 48, generator=g).to(dtype).cuda(), torch.randn(2, 48, generator=g).cuda(),
                torch.randint(40, (2, 140), generator=g).cuda())
    eager, eager_p = [], [t.to(dtype).cuda().requires_grad_() for t in parameters(seed=2)]
    for k in range(4):
        eager.append([t.clone() for t in step(eager_p, *data(k))])
    p = [t.to(dtype).cuda().requires_grad_() for t in parameters(seed=2)]
    held = data(0)
    warm = [t.detach().clone().requires_grad_() for t in p]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(warm, *held)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(p, *held)
    for k in range(4):
        for t, v in zip(held, data(k)):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager[k])), k
    assert all(torch.equal(a, b) for a, b in zip(p, eager_p))
