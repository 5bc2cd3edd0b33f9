"""gated_scan and its gradients against the recurrence in 64 bits: every pair of types, lengths from none to those cut into segments,
channels from one on, gates of 0 and 1, strides.

Tolerance: a term x_s times the t - s gates after it goes through at most 2 (t - s) + 8 roundings in f32 (each step of its way is
added once and its gates are multiplied once), so with S the recurrence of the magnitudes and W the one that counts steps,
W_t = |a_t| (W_{t-1} + S_{t-1}), h is off by at most u (2 W + 8 S), u = 2^-24; backwards alike. The gates' gradient takes h
in f32. Then half a step of the output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
         (torch.float16, torch.float16), (torch.float16, torch.float32)]
U = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def make(B, T, n, dtype, gate_type, seed=0):
    g = torch.Generator().manual_seed(seed)
    gate = torch.sigmoid(torch.randn(B, T, n, generator=g) + 5 * torch.rand(n, generator=g))
    gate[torch.rand(B, T, generator=g) < 0.02] = 0.0
    gate[torch.rand(B, T, generator=g) < 0.02] = 1.0
    x = torch.randn(B, T, n, generator=g)
    return (gate.to(gate_type), x.to(dtype), torch.randn(B, n, generator=g), torch.randn(B, T, n, generator=g).to(dtype),
            torch.randn(B, n, generator=g))


def near(got, ref, tol, name):
    assert got.shape == ref.shape, name
    half = torch.finfo(got.dtype).eps / 2
    err = (got.detach().double().cpu() - ref).abs()
    room = tol + half * (ref.abs() + tol) + LEAST[got.dtype]
    assert (err <= room).all(), (name, float((err / room).max()))


def reference(gate, x, state, dh, dlast):
    """Outputs and gradients in 64 bits, each with its tolerance."""
    a, x, s, dh, e = gate.double(), x.double(), state.double(), dh.double(), dlast.double()
    B, T, n = x.shape
    before, h, room = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    S, W = s.abs(), torch.zeros_like(s)
    for t in range(T):
        before[:, t] = s
        s = a[:, t] * s + x[:, t]
        W = a[:, t].abs() * (W + S)
        S = a[:, t].abs() * S + x[:, t].abs()
        h[:, t], room[:, t] = s, U * (2 * W + 8 * S)
    last_room = U * (2 * W + 8 * S)
    dx, back = torch.zeros_like(x), torch.zeros_like(x)
    S, W = e.abs(), torch.zeros_like(e)
    for t in range(T - 1, -1, -1):
        e = e + dh[:, t]
        S = S + dh[:, t].abs()
        dx[:, t], back[:, t] = e, U * (2 * W + 8 * S)
        e = e * a[:, t]
        W = a[:, t].abs() * (W + S)
        S = a[:, t].abs() * S
    return (h, room), (s, last_room), (dx, back), before, (e, U * (2 * W + 8 * S))


def check(gate, x, state, dh, dlast, on_device=None):
    from yggdrasil_amd import ops
    gg, xg = [t.cuda() for t in (gate, x)] if on_device is None else on_device
    gg, xg, sg = gg.detach().requires_grad_(), xg.detach().requires_grad_(), state.cuda().requires_grad_()
    h, last = ops.gated_scan(gg, xg, sg)
    assert h.dtype == x.dtype and last.dtype == torch.float32 and h.is_contiguous()
    (rh, th), (rl, tl), (rx, tx), before, (rs, ts) = reference(gate, x, state, dh, dlast)
    near(h, rh, th, "h")
    near(last, rl, tl, "last")
    dg, dx, ds = torch.autograd.grad((h, last), (gg, xg, sg), (dh.cuda(), dlast.cuda()))
    assert dg.dtype == gate.dtype and dx.dtype == x.dtype and ds.dtype == torch.float32
    near(dx, rx, tx, "dx")
    near(ds, rs, ts, "dstate")
    prior = torch.cat([torch.zeros_like(th[:, :1]), th[:, :-1]], 1)
    near(dg, rx * before, rx.abs() * prior + tx * (before.abs() + prior) + 2 * U * (rx * before).abs(), "dgate")


@pytest.mark.parametrize("dtype, gate_type", TYPES, ids=str)
@pytest.mark.parametrize("B, T, n", [(1, 1, 1), (3, 2, 5), (2, 7, 8), (2, 8, 16), (1, 9, 3), (4, 16, 100), (2, 63, 64), (2, 64, 130), (3, 65, 1),
                                     (1, 127, 7), (2, 128, 12), (2, 129, 40), (1, 257, 257), (2, 300, 2), (5, 100, 1000)])
def test_shapes(B, T, n, dtype, gate_type):
    check(*make(B, T, n, dtype, gate_type, seed=B + T + n))


@pytest.mark.parametrize("dtype, gate_type", TYPES, ids=str)
@pytest.mark.parametrize("B, T, n", [(1, 5000, 24), (1, 20011, 3), (3, 1030, 130), (2, 2500, 66), (40, 600, 32), (10, 300, 600), (10, 290, 1300)])
def test_long(B, T, n, dtype, gate_type):
    """Sequences that are cut into segments, the last of them short."""
    check(*make(B, T, n, dtype, gate_type, seed=T))


@pytest.mark.parametrize("dtype, gate_type", TYPES, ids=str)
def test_many_sequences(dtype, gate_type):
    check(*make(700, 40, 6, dtype, gate_type, seed=1))
    check(*make(300, 13, 70, dtype, gate_type, seed=2))
    check(*make(5000, 1, 9, dtype, gate_type, seed=3))


@pytest.mark.parametrize("dtype, gate_type", TYPES, ids=str)
def test_strides(dtype, gate_type):
    """Parts of wider rows, off an alignment; time before the batch; one gate for all sequences; channels that lie apart."""
    gate, x, state, dh, dlast = make(3, 70, 37, dtype, gate_type, seed=4)
    for at in (1, 8):
        wide_g, wide_x = (torch.full((3, 70, 60), 7.0, dtype=t.dtype, device="cuda") for t in (gate, x))
        wide_g[..., at:at + 37], wide_x[..., at:at + 37] = gate.cuda(), x.cuda()
        check(gate, x, state, dh, dlast, (wide_g[..., at:at + 37], wide_x[..., at:at + 37]))
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1).cuda() for t in (gate, x)]
    check(gate, x, state, dh, dlast, swapped)
    apart = [t.transpose(1, 2).contiguous().transpose(1, 2).cuda() for t in (gate, x)]
    check(gate, x, state, dh, dlast, apart)
    one = gate[:1].expand(3, 70, 37)
    check(one.contiguous(), x, state, dh, dlast, (gate[:1].cuda().expand(3, 70, 37), x.cuda()))


def test_broadcast_gates_and_no_state():
    """The gradient of gates that are the same at every step, and of a gate of one value a step, come back in their shapes."""
    from yggdrasil_amd import ops
    gate, x, state, dh, dlast = make(2, 50, 12, torch.float32, torch.float32, seed=5)
    for small in (gate[:, :1, :], gate[0, 0], gate[:, :, :1]):
        leaf = small.cuda().requires_grad_()
        h, last = ops.gated_scan(leaf.expand(2, 50, 12), x.cuda())
        got, = torch.autograd.grad((h, last), leaf, (dh.cuda(), dlast.cuda()))
        full = small.expand(2, 50, 12)
        (rh, th), _, (rx, tx), before, _ = reference(full, x, torch.zeros(2, 12), dh, dlast)
        near(h, rh, th, "h")
        each = rx * before
        room = tx * before.abs() + rx.abs() * torch.cat([torch.zeros_like(th[:, :1]), th[:, :-1]], 1) + 200 * U * each.abs()
        near(got, each.sum_to_size(small.shape), 2 * room.sum_to_size(small.shape), "dgate")


@pytest.mark.parametrize("dtype, gate_type", TYPES, ids=str)
def test_in_parts_and_step_by_step(dtype, gate_type):
    """A sequence in parts with the state carried on is the sequence, one step at a time too."""
    from yggdrasil_amd import ops
    gate, x, state, dh, dlast = make(2, 90, 33, dtype, gate_type, seed=6)
    (rh, th), (rl, tl), *_ = reference(gate, x, state, dh, dlast)
    for step in (1, 5, 40):
        s, parts = state.cuda(), []
        for t in range(0, 90, step):
            h, s = ops.gated_scan(gate[:, t:t + step].cuda(), x[:, t:t + step].cuda(), s)
            parts.append(h)
        near(torch.cat(parts, 1), rh, th, "h")
        near(s, rl, tl, "last")


def test_padding_resets_and_nan():
    """A gate of 1 with x 0 keeps the state, a gate of 0 begins anew, and a NaN stays in its sequence and channel, from its step
    on until a gate of 0 would make it NaN still."""
    from yggdrasil_amd import ops
    gate, x, state, *_ = (t.cuda() for t in make(3, 400, 20, torch.float32, torch.float32, seed=7))
    h, last = ops.gated_scan(gate, x, state)
    padded_g, padded_x = torch.cat([gate, torch.ones_like(gate)], 1), torch.cat([x, torch.zeros_like(x)], 1)
    h2, last2 = ops.gated_scan(padded_g, padded_x, state)
    near(last2, last.double().cpu(), 1e-5 * last.double().cpu().abs() + 1e-6, "last")
    gate[:, 100] = 0.0
    h3, _ = ops.gated_scan(gate, x, state)
    assert torch.equal(h3[:, 100], x[:, 100])
    x[1, 50, 3] = math.nan
    h4, last4 = ops.gated_scan(gate, x, state)
    bad = h4.isnan()
    assert bad[1, 50:, 3].all() and bad.sum() == 350 and last4.isnan().sum() == 1
    ones, big = torch.ones(1, 5000, 4, device="cuda"), torch.ones(1, 5000, 4, device="cuda")
    assert (ops.gated_scan(ones, big)[0][0, :, 0] == torch.arange(1, 5001, device="cuda")).all()


def test_gates_above_one():
    """Gates past 1 whose products stay finite, and negative ones."""
    g = torch.Generator().manual_seed(8)
    gate = 0.9 + 0.25 * torch.rand(2, 300, 10, generator=g)
    gate[..., ::2] *= -1
    check(gate, torch.randn(2, 300, 10, generator=g), torch.randn(2, 10, generator=g), torch.randn(2, 300, 10, generator=g),
          torch.randn(2, 10, generator=g))


def test_parts_of_the_gradient():
    """One output's gradient without the other's, and one input's by itself."""
    from yggdrasil_amd import ops
    gate, x, state, dh, dlast = (t.cuda() for t in make(2, 333, 50, torch.bfloat16, torch.float32, seed=9))
    leaves = [t.requires_grad_() for t in (gate, x, state)]
    h, last = ops.gated_scan(*leaves)
    whole = torch.autograd.grad((h, last), leaves, (dh, torch.zeros_like(dlast)), retain_graph=True)
    alone = torch.autograd.grad(h, leaves, dh, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(whole, alone))
    whole = torch.autograd.grad((h, last), leaves, (torch.zeros_like(dh), dlast), retain_graph=True)
    alone = torch.autograd.grad(last, leaves, dlast, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(whole, alone))
    whole = torch.autograd.grad((h, last), leaves, (dh, dlast), retain_graph=True)
    for i, leaf in enumerate(leaves):
        assert torch.equal(torch.autograd.grad((h, last), leaf, (dh, dlast), retain_graph=True)[0], whole[i])
        others = [t.detach().requires_grad_(k == i) for k, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(ops.gated_scan(*others), others[i], (dh, dlast))[0], whole[i])


def test_against_differences():
    """The recurrence is linear in each value of x, gate and state alone, so a difference is off by roundings only: those of h,
    2^-24 times a few hundred, over the step of 2^-4."""
    from yggdrasil_amd import ops
    gate, x, state, dh, dlast = (t.cuda() for t in make(1, 70, 3, torch.float32, torch.float32, seed=10))
    leaves = [t.requires_grad_() for t in (gate, x, state)]
    grads = torch.autograd.grad(ops.gated_scan(*leaves), leaves, (dh, dlast))
    with torch.no_grad():
        for i, (leaf, grad) in enumerate(zip(leaves, grads)):
            for k in range(0, leaf.numel(), 17):
                ends = []
                for step in (2.0 ** -5, -2.0 ** -5):
                    moved = leaf.clone()
                    moved.view(-1)[k] += step
                    h, last = ops.gated_scan(*[moved if j == i else t for j, t in enumerate(leaves)])
                    ends.append((h.double() * dh.double()).sum() + (last.double() * dlast.double()).sum())
                assert abs((ends[0] - ends[1]) * 16 - grad.view(-1)[k].double()) < 1e-2


def test_nothing_to_do():
    from yggdrasil_amd import ops
    state = torch.randn(3, 5, device="cuda", requires_grad=True)
    e = torch.zeros(3, 0, 5, device="cuda", requires_grad=True)
    h, last = ops.gated_scan(e, e, state)
    assert h.shape == (3, 0, 5) and torch.equal(last, state)
    w = torch.randn(3, 5, device="cuda")
    d, de = torch.autograd.grad(last, (state, e), w)
    assert torch.equal(d, w) and de.shape == e.shape
    assert not ops.gated_scan(e, e)[1].any()
    none = torch.zeros(0, 4, 5, device="cuda", requires_grad=True)
    h, last = ops.gated_scan(none, none)
    assert h.shape == (0, 4, 5) and last.shape == (0, 5)
    assert torch.autograd.grad(h.sum() + last.sum(), none)[0].shape == (0, 4, 5)


@pytest.mark.parametrize("B, T, n", [(64, 1, 256), (1, 3000, 48), (2, 100, 300)])
def test_streams_and_graphs(B, T, n):
    from yggdrasil_amd import ops
    gate, x, state, dh, dlast = (t.cuda() for t in make(B, T, n, torch.bfloat16, torch.bfloat16, seed=11))
    leaves = [t.requires_grad_() for t in (gate, x, state)]

    def both(leaves, dh, dlast):
        r = ops.gated_scan(*leaves)
        return (*(t.detach() for t in r), *torch.autograd.grad(r, leaves, (dh, dlast)))
    want = both(leaves, dh, dlast)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(leaves, dh, dlast)
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del want, got
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both(leaves, dh, dlast)
    for k in range(3):
        new = make(B, T, n, torch.bfloat16, torch.bfloat16, seed=30 + k)
        with torch.no_grad():
            for t, v in zip((gate, x, state, dh, dlast), new):
                t.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        fresh = [v.cuda() for v in new]
        want = both([t.requires_grad_() for t in fresh[:3]], *fresh[3:])
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(kept, want)), k


def test_refusals():
    from yggdrasil_amd import ops
    x, s = torch.zeros(2, 4, 8, device="cuda"), torch.zeros(2, 8, device="cuda")
    for bad in (lambda: ops.gated_scan(x, x[0]), lambda: ops.gated_scan(x[0], x[0]), lambda: ops.gated_scan(x[:, :3], x),
                lambda: ops.gated_scan(x.half(), x), lambda: ops.gated_scan(x.bfloat16(), x.half()), lambda: ops.gated_scan(x.cpu(), x),
                lambda: ops.gated_scan(x, x, s.half()), lambda: ops.gated_scan(x, x, s[:1]), lambda: ops.gated_scan(x, x, s.cpu()),
                lambda: ops.gated_scan(x[..., :0], x[..., :0]), lambda: ops.gated_scan(x.double(), x.double()),
                lambda: ops.gated_scan(None, x)):
        with pytest.raises(ValueError):
            bad()
    x.requires_grad_()
    g, = torch.autograd.grad(ops.gated_scan(x.detach(), x)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ops.gated_scan(x.detach(), fwd.make_dual(x.detach(), torch.ones_like(x)))
