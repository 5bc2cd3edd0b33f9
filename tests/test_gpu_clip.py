"""grad_norm and clip_grad_norm against the formula in 64 bits: every type, mixed ones, tensors of no value to many chunks, more tensors
than a launch takes, views, in place, values outside f32's squares.

Tolerances: the norm is summed in 64 bits and rounded once to f32 (2^-24 of itself; 2^-40 covers the sum); a value is multiplied in 64
bits, rounded to f32 and then to its type: half a step of it and 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def make(sizes, dtypes=DTYPES, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * (1 + i % 3) * torch.randn(n, generator=g)).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def norm_of(grads):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


def check(grads, share, in_place=False, device=None):
    from yggdrasil_amd import ops
    dev = [g.cuda() for g in grads] if device is None else device
    norm = norm_of(grads)
    most = norm * share
    assert abs(float(ops.grad_norm(dev)) - norm) <= norm * (2.0 ** -24 + 2.0 ** -40)
    kept = [d.clone() for d in dev]
    out, got = ops.clip_grad_norm(dev, most, out=dev if in_place else None)
    assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - norm) <= norm * (2.0 ** -24 + 2.0 ** -40)
    by = min(1.0, most / norm) if norm else 1.0
    assert len(out) == len(grads)
    for o, d, k, g in zip(out, dev, kept, grads):
        assert o.shape == g.shape and o.dtype == g.dtype
        assert (o is d) if in_place else torch.equal(d, k)
        if by == 1.0:
            assert torch.equal(o.cpu(), g)
            continue
        ref = g.double() * by
        err = (o.cpu().double() - ref).abs()
        assert (err <= ref.abs() * (torch.finfo(g.dtype).eps / 2 + 2.0 ** -24) + LEAST[g.dtype]).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("share", [0.1, 0.99, 1.5])
@pytest.mark.parametrize("sizes", [[1], [7], [16384], [16385], [3, 1, 200], [100000, 5, 0, 16384, 33, 4096], [0, 0, 9]])
def test_sizes(sizes, share, in_place):
    for dtypes in ([torch.float32], [torch.bfloat16], [torch.float16], DTYPES):
        check(make(sizes, dtypes, seed=len(sizes)), share, in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("count", [127, 128, 129, 300])
def test_many_tensors(count, in_place):
    check(make([1 + 37 * i % 501 for i in range(count)], seed=count), 0.3, in_place)


def test_large():
    check(make([3_000_001, 1_000_000], seed=1), 0.5, True)


def test_values_outside_f32_squares():
    """Squares past f32's largest and below its smallest number: the norm and what is left of the values are right."""
    check(make([1000, 20], [torch.float32], scale=1e30), 0.2)
    check(make([1000, 20], [torch.float32, torch.bfloat16], scale=1e-30), 0.2)
    from yggdrasil_amd import ops
    huge = [torch.full((16,), 3e38, device="cuda")]
    out, norm = ops.clip_grad_norm(huge, 1.0)
    assert norm.isinf()        # its norm, 1.2e39, is no f32, and yet the values come to a norm of 1
    assert torch.allclose(out[0], torch.full_like(out[0], 0.25))


def test_zero_norm_and_zero_bound():
    from yggdrasil_amd import ops
    z = [torch.zeros(5, device="cuda"), torch.zeros(3, dtype=torch.float16, device="cuda")]
    out, norm = ops.clip_grad_norm(z, 1.0)
    assert norm == 0 and all(torch.equal(a, b) for a, b in zip(out, z))
    out, norm = ops.clip_grad_norm([torch.ones(4, device="cuda")], 0.0)
    assert norm == 2 and not out[0].any()
    out, norm = ops.clip_grad_norm([torch.ones(4, device="cuda")], math.inf)
    assert norm == 2 and out[0].eq(1).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_norm_that_is_not_finite_changes_nothing(bad):
    from yggdrasil_amd import ops
    grads = [g.cuda() for g in make([50, 3000], seed=2)]
    grads[1][77] = bad
    for out in (None, grads):
        kept = [g.clone() for g in grads]
        r, norm = ops.clip_grad_norm(grads, 0.1, out=out)
        assert not norm.isfinite()
        assert all(torch.equal(a.nan_to_num(1.0, 2.0, 3.0), b.nan_to_num(1.0, 2.0, 3.0)) for a, b in zip(r, kept))


def test_views():
    """Matrices in other orders, parts of one buffer at any address, and tensors that are not dense."""
    g = make([600, 35, 640], [torch.bfloat16], seed=3)
    whole = torch.zeros(2000, dtype=torch.bfloat16, device="cuda")
    parts = [whole[1:601].view(20, 30).t(), whole[701:736], whole[801:1441].view(8, 8, 10).permute(2, 0, 1)]
    for p, v in zip(parts, g):
        p.copy_(v.view(p.shape))
    cpu = [p.cpu() for p in parts]
    check(cpu, 0.4, False, parts)
    before = whole.clone()
    check(cpu, 0.4, True, parts)
    same = torch.ones(2000, dtype=torch.bool)
    for lo, hi in ((1, 601), (701, 736), (801, 1441)):
        same[lo:hi] = False
    assert torch.equal(whole.cpu()[same], before.cpu()[same])
    check([p.cpu() for p in (whole[::3], whole[:5].expand(4, 5))], 0.4, False, [whole[::3], whole[:5].expand(4, 5)])


def test_into_other_tensors_and_none():
    from yggdrasil_amd import ops
    grads = [g.cuda() for g in make([40, 60], [torch.float32], seed=4)]
    grads[1] = grads[1].view(6, 10).t()
    want, norm = ops.clip_grad_norm(grads, 1.0)
    to = [torch.empty(40, device="cuda"), torch.empty(10, 6, device="cuda")]
    got, n2 = ops.clip_grad_norm(grads, 1.0, out=to)
    assert got[1] is to[1] and torch.equal(n2, norm) and all(torch.equal(a, b) for a, b in zip(got, want))
    got, n3 = ops.clip_grad_norm([None, grads[0], None, grads[1]], 1.0)
    assert got[0] is None and got[2] is None and torch.equal(got[3], want[1]) and torch.equal(n3, norm)
    assert torch.equal(ops.grad_norm([None, *grads]), norm)


def test_same_result_every_time_and_version():
    from yggdrasil_amd import ops
    grads = [g.cuda() for g in make([300000, 70000], seed=5)]
    a, b = ops.clip_grad_norm(grads, 1.0), ops.clip_grad_norm(grads, 1.0)
    assert torch.equal(a[1], b[1]) and all(torch.equal(x, y) for x, y in zip(a[0], b[0]))
    v = [g._version for g in grads]
    ops.clip_grad_norm(grads, 1.0, out=grads)
    assert all(g._version > w for g, w in zip(grads, v))
    with torch.inference_mode():
        t = torch.ones(9, device="cuda")
        ops.clip_grad_norm([t], 1.0, out=[t])
        assert t.sum() == 3


@pytest.mark.parametrize("in_place", [False, True])
def test_streams_and_graphs(in_place):
    from yggdrasil_amd import ops
    grads = [g.cuda() for g in make([5000, 33, 70000], seed=6)]
    s = torch.cuda.Stream()
    want = ops.clip_grad_norm(grads, 5.0)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.clip_grad_norm(grads, 5.0)
    s.synchronize()
    assert torch.equal(got[1], want[1]) and all(torch.equal(a, b) for a, b in zip(got[0], want[0]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, norm = ops.clip_grad_norm(grads, 5.0, out=grads if in_place else None)
    for k in range(3):
        new = [v.cuda() for v in make([5000, 33, 70000], seed=60 + k)]
        for t, v in zip(grads, new):
            t.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        want = ops.clip_grad_norm(new, 5.0)
        torch.cuda.synchronize()
        assert torch.equal(norm, want[1]) and all(torch.equal(a, b) for a, b in zip(out, want[0])), k


def test_refusals():
    from yggdrasil_amd import ops
    x = torch.ones(8, device="cuda")
    for bad in (lambda: ops.clip_grad_norm([], 1.0), lambda: ops.clip_grad_norm([None], 1.0), lambda: ops.clip_grad_norm([x], -1.0),
                lambda: ops.clip_grad_norm([x], math.nan), lambda: ops.clip_grad_norm([x], x.sum()), lambda: ops.clip_grad_norm([x.cpu()], 1.0),
                lambda: ops.clip_grad_norm([x.double()], 1.0), lambda: ops.clip_grad_norm([x], 1.0, out=[]),
                lambda: ops.clip_grad_norm([x], 1.0, out=[x[:7]]), lambda: ops.clip_grad_norm([x], 1.0, out=[x.half()]),
                lambda: ops.clip_grad_norm([x, x], 1.0, out=[x, x]), lambda: ops.clip_grad_norm([x[:6], x[4:]], 1.0, out=[x[:6], x[4:]]),
                lambda: ops.clip_grad_norm([x[:4], x[4:]], 1.0, out=[x[4:], x[:4]]), lambda: ops.clip_grad_norm([x[:4]], 1.0, out=[x[2:6]]),
                lambda: ops.clip_grad_norm([x[:4]], 1.0, out=[x[::2]]), lambda: ops.clip_grad_norm([x], 1.0, out=[None]),
                lambda: ops.clip_grad_norm([x.clone().requires_grad_()], 1.0), lambda: ops.grad_norm([x, None, 3])):
        with pytest.raises(ValueError):
            bad()
    assert x.eq(1).all()
    out, norm = ops.clip_grad_norm([x, x], 1.0)     # the same one twice counts twice, and is only read
    assert norm == 4 and torch.equal(out[0], out[1])
