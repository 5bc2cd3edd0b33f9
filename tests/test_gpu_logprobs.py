"""token_logprobs against the formulas in 64 bits: every type, vocabularies from one class to wide odd ones, masks, rows
without a distribution, ties, strides, and the gradient against the formula's and against differences.

Tolerances, from the arithmetic alone (e = 2^-23, a step of f32): d = x - max is off by e |d| / 2, an exponential by a few
e and e |d| relative (its argument's rounding), a sum of V terms by the terms' errors and a rounding for each addition on
the longest path (at most V / 64 + 64 of them here), a logarithm by e. So log-probabilities and entropies are within
e (4 |value| + 8 + V / 128) (the additions' roundings average out; they are counted by half)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E32 = 2.0 ** -23
INF = math.inf


def plain(x, t, top):
    """In 64 bits on the host: logp (None without targets), entropy, top values and ids."""
    x = x.double().cpu()
    V = x.shape[1]
    bad = ~(x < INF).all(1)
    m = x.max(1, keepdim=True).values
    none = (m == -INF)[:, 0] & ~bad
    d = torch.where(torch.isneginf(m) | bad[:, None], torch.zeros_like(x), x - m)
    e = torch.exp(d)
    Z = e.sum(1, keepdim=True)
    # the others' sum apart from the maximum's own terms, for rows sure of their token
    rest = torch.where(d < 0, e, torch.zeros_like(e)).sum(1, keepdim=True)
    logz = torch.log1p((d == 0).sum(1, keepdim=True) - 1 + rest)
    lp = d - logz
    p = e / Z
    H = -torch.where(p > 0, p * torch.where(p > 0, lp, torch.zeros_like(lp)), torch.zeros_like(p)).sum(1)
    H[none] = 0
    H[bad] = math.nan
    lp[none] = -INF
    lp[bad] = math.nan
    out = {"entropy": H}
    if t is not None:
        t = t.cpu().long()
        inside = (t >= 0) & (t < V)
        v = lp.gather(1, torch.where(inside, t, torch.zeros_like(t))[:, None])[:, 0]
        out["logp"] = torch.where(t == -1, torch.zeros_like(v), torch.where(inside, v, torch.full_like(v, math.nan)))
    if top:
        ids = torch.sort(torch.where(bad[:, None], torch.full_like(x, -INF), x), dim=1, descending=True,
                         stable=True).indices[:, :top]
        val = lp.gather(1, ids)
        gone = torch.isneginf(x.gather(1, ids)) | bad[:, None]
        ids = torch.where(gone, torch.full_like(ids, -1), ids)
        val = torch.where(gone, torch.full_like(val, -INF), val)
        more = max(0, top - V)
        ids = torch.nn.functional.pad(ids, (0, more), value=-1)
        val = torch.nn.functional.pad(val, (0, more), value=-INF)
        val[bad] = math.nan
        out["top_ids"], out["top_logp"] = ids, val
    return out


def near(got, ref, V, extra=0.0):
    got, ref = got.double().cpu(), ref.double()
    ref = torch.where(ref.abs() > torch.finfo(torch.float32).max, ref.float().double(), ref)   # past f32: infinite there
    assert got.shape == ref.shape
    odd = ~torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    same = odd & ~torch.isnan(ref)
    assert torch.equal(got[same], ref[same])
    err, tol = (got - ref)[~odd].abs(), E32 * (4 * ref[~odd].abs() + 8 + V / 128) + extra
    assert (err <= tol).all(), (err - tol).max()


def check(x, t, top):
    from yggdrasil_amd import ops
    r = ops.token_logprobs(x, t, top=top)
    ref = plain(x, t, top)
    V = x.shape[1]
    near(r.entropy, ref["entropy"], V)
    if t is None:
        assert r.logp is None
    else:
        near(r.logp, ref["logp"], V)
    if top:
        assert r.top_ids.dtype == torch.int32
        np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ref["top_ids"].numpy())
        near(r.top_logp, ref["top_logp"], V)
    else:
        assert r.top_ids is None and r.top_logp is None
    return r


def rows_of(n, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, V, generator=g) * spread).to(dtype)
    t = torch.randint(V, (n,), generator=g)
    return x.cuda(), t.cuda()


SIZES = [(1, 1), (3, 2), (70, 5), (5, 16), (33, 27), (9, 63), (130, 64), (7, 255), (65, 256), (6, 257), (5, 1000), (17, 1024),
         (3, 1025), (4, 2048), (3, 4097), (2, 8192), (3, 50257), (1, 131075)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n, V", SIZES)
def test_sizes(n, V, dtype):
    x, t = rows_of(n, V, dtype, n + V)
    check(x, t.int(), 0)
    check(x, t, 5)
    check(x, None, 20)


@pytest.mark.parametrize("V", [256, 1024, 3000, 40000])
@pytest.mark.parametrize("top", [1, 31, 32, 33, 64])
def test_many_alternatives(V, top):
    x, t = rows_of(5, V, torch.float32, top)
    check(x, t, top)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [1, 3, 64, 256, 700, 1500, 9001, 70000])
def test_masks_and_rows_without_a_distribution(V, dtype):
    x, t = rows_of(12, V, dtype, V)
    low = torch.finfo(dtype).min
    x[0] = -INF                                     # nothing left
    x[1, 1:] = -INF                                 # one token left, the first
    x[2, :-1] = -INF                                # one token left, the last
    x[3] = low                                      # masked with the type's lowest value
    x[4, ::2] = low
    x[5, V // 2] = math.nan
    x[6, -1] = INF
    x[7] = 0.0                                      # all equal
    x[8, ::3] = -INF
    x[9] = torch.finfo(dtype).max
    x[9, V // 2] = low                              # differences past the type's range
    x[10, 0] = -0.0
    t[8] = V - 1
    t[11] = -1
    r = check(x, t, 7)
    check(x, t, 0)
    assert r.logp[0] == -INF and r.entropy[0] == 0 and (r.top_ids[0] == -1).all()
    assert r.logp[11] == 0
    assert r.top_ids[7].tolist() == [c if c < V else -1 for c in range(7)]
    if V > 1:
        assert r.logp[1] == (0 if t[1] == 0 else -INF) and r.entropy[1] == 0


@pytest.mark.parametrize("V", [2, 256, 5000])
def test_bad_targets_are_nan(V):
    x, t = rows_of(6, V, torch.float32, V)
    t[:5] = torch.tensor([-2, V, V + 5, -100, -1])
    r = check(x, t, 0)
    assert torch.isnan(r.logp[:4]).all() and r.logp[4] == 0
    check(x, t.int(), 3)
    t[0] = 1 << 40                                  # no int32 value
    assert torch.isnan(check(x, t, 0).logp[0])


@pytest.mark.parametrize("V", [256, 1000, 9000, 70001])
def test_rows_sure_of_their_token_keep_their_digits(V):
    """Log-probability of the token and entropy where nearly all of it is on one token: values far below 1 keep their
    relative precision (their terms have one sign: the exponentials' e |d| and a few e)."""
    from yggdrasil_amd import ops
    x, t = rows_of(8, V, torch.float32, 3, 1.0)
    t[:] = V // 3
    gap = torch.tensor([15.0, 20, 25, 30, 35, 40, 50, 60], device="cuda")
    x[:, V // 3] = x.max(1).values + gap
    r, ref = ops.token_logprobs(x, t), plain(x, t, 0)
    for k in ("logp", "entropy"):
        rel = (getattr(r, k).double().cpu() - ref[k]).abs() / ref[k].abs()
        assert (rel <= E32 * (2 * gap.cpu() + 12 + V / 128)).all(), (k, rel)


@pytest.mark.parametrize("order", ["rising", "falling", "steps", "equal", "late"])
@pytest.mark.parametrize("V", [200, 1000, 8192, 60000])
def test_alternatives_in_orders_that_hurt(V, order):
    c = torch.arange(V, dtype=torch.float32)
    row = {"rising": c / V, "falling": -c / V, "steps": torch.floor(c / 37), "equal": torch.full((V,), 1.5),
           "late": torch.where(c > V - 30, 5.0, 0.0)}[order]
    x = torch.stack([row, row.flip(0), row * 1e-3]).cuda()
    for top in (1, 20, 64):
        check(x, None, top)
    check(x.bfloat16(), None, 20)


def test_strides_shapes_and_views():
    from yggdrasil_amd import ops
    whole, _ = rows_of(6, 1040, torch.bfloat16, 1)
    for a, b in ((0, 1000), (3, 1003), (1, 1040), (8, 264)):
        x = whole[:, a:b]
        t = torch.arange(6, device="cuda")
        check(x, t, 4)
    x3 = whole[:, :500].reshape(2, 3, 500)
    t3 = torch.arange(6, device="cuda").reshape(2, 3)
    r, f = ops.token_logprobs(x3, t3, top=2), ops.token_logprobs(whole[:, :500], torch.arange(6, device="cuda"), top=2)
    assert r.logp.shape == (2, 3) and r.entropy.shape == (2, 3) and r.top_ids.shape == (2, 3, 2)
    assert torch.equal(r.logp.reshape(-1), f.logp) and torch.equal(r.top_ids.reshape(6, 2), f.top_ids)
    one = ops.token_logprobs(whole[0], torch.tensor(3, device="cuda"), top=1)       # a single row without a batch axis
    assert one.logp.shape == () and one.top_ids.shape == (1,)
    check(whole.t()[:200], torch.zeros(200, dtype=torch.int64, device="cuda"), 2)   # columns as rows
    check(whole[:1].expand(4, 1040), torch.arange(4, device="cuda"), 2)             # one row for all
    e = ops.token_logprobs(torch.empty(0, 9, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert e.logp.shape == (0,) and e.top_ids.shape == (0, 3)


def test_many_rows():
    """More rows than a grid's workgroups take at once, of a small vocabulary."""
    x, t = rows_of(300001, 3, torch.float32, 0)
    check(x, t, 2)
    x, t = rows_of(70000, 33, torch.bfloat16, 0)
    check(x, t.int(), 3)


def _weights(n, top, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, generator=g), torch.randn(n, generator=g), torch.randn(n, max(top, 1), generator=g)


def _grad64(x, t, top, gl, gh, gt):
    """The formula's gradient in 64 bits, and what each entry's arithmetic in f32 may be off by (a few e of each factor)."""
    ref = plain(x, t, top)
    x64 = x.detach().double().cpu()
    V = x64.shape[1]
    none = torch.isneginf(x64).all(1)
    m = x64.max(1, keepdim=True).values
    d0 = torch.where(none[:, None], torch.zeros_like(x64), x64 - m)
    lp = d0 - torch.log(torch.exp(d0).sum(1, keepdim=True))
    p = torch.exp(lp)
    H = ref["entropy"][:, None]
    tc = t.cpu().long()
    g = torch.where(tc == -1, torch.zeros(len(tc), dtype=torch.double), gl.double())
    hit = torch.zeros_like(p)
    hit[torch.arange(len(tc))[tc >= 0], tc[tc >= 0]] = g[tc >= 0]
    whole = g.clone()
    size = g.abs()
    if top:
        ids, k = ref["top_ids"], gt.double()[:, :top]
        k = torch.where(ids >= 0, k, torch.zeros_like(k))
        hit.scatter_add_(1, ids.clamp(min=0), k)
        whole += k.sum(1)
        size = size + k.abs().sum(1)
    safe = torch.where(p > 0, lp, torch.zeros_like(lp))
    d = hit - p * whole[:, None] - torch.where(p > 0, gh.double()[:, None] * p * (safe + H), torch.zeros_like(p))
    tol = E32 * (2 * hit.abs() + p * (size[:, None] + gh.double().abs()[:, None] * (safe.abs() + H)) * (12 + V / 128 + 3 * safe.abs()))
    d[none] = 0
    return d, tol


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n, V, top", [(1, 1, 0), (9, 5, 2), (33, 256, 5), (4, 257, 0), (5, 1000, 20), (3, 4099, 3), (3, 50257, 0),
                                       (2, 70000, 33)])
def test_gradient(n, V, top, dtype):
    from yggdrasil_amd import ops
    x, t = rows_of(n, V, dtype, V)
    if n > 2 and V > 2:
        x[0, 1:V - 1] = -INF
        t[0] = 0
        x[1] = -INF
        t[2] = -1
    x.requires_grad_()
    gl, gh, gt = _weights(n, top, V)
    r = ops.token_logprobs(x, t, top=top)
    outs, gs = [r.logp, r.entropy], [gl.cuda(), gh.cuda()]
    if top:
        outs.append(r.top_logp)
        gs.append(gt[:, :top].cuda())
    dx, = torch.autograd.grad(outs, x, gs)
    ref, tol = _grad64(x, t, top, gl, gh, gt)
    assert dx.dtype == dtype and dx.shape == x.shape
    step = torch.finfo(dtype).eps / 2
    small = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[dtype]
    err = (dx.double().cpu() - ref).abs()
    assert (err <= tol + step * (ref.abs() + tol) + small).all(), (err - tol - step * ref.abs()).max()


def test_gradient_of_some_outputs_and_views():
    """One output alone, expanded gradients (a sum's), logits that are a view with a row stride, leading axes."""
    from yggdrasil_amd import ops
    whole, _ = rows_of(6, 300, torch.float32, 5)
    base = whole.clone().requires_grad_()
    x = base[:, 7:264]
    t = torch.arange(6, device="cuda")
    ops.token_logprobs(x, t).logp.sum().backward()
    ref, tol = _grad64(x, t, 0, torch.ones(6), torch.zeros(6), None)
    got = base.grad.double().cpu()
    assert (got[:, :7] == 0).all() and (got[:, 264:] == 0).all()
    assert ((got[:, 7:264] - ref).abs() <= tol + 2.0 ** -24 * ref.abs() + 2.0 ** -126).all()
    x3 = whole[:, :200].reshape(2, 3, 200).clone().requires_grad_()
    ops.token_logprobs(x3).entropy.mean().backward()
    ref, tol = _grad64(x3.reshape(6, 200), -torch.ones(6, dtype=torch.int64), 0, torch.zeros(6), torch.full((6,), 1 / 6), None)
    assert ((x3.grad.reshape(6, 200).double().cpu() - ref).abs() <= tol + 2.0 ** -24 * ref.abs() + 2.0 ** -126).all()


def test_gradient_against_differences():
    """Central differences of the 64-bit formula along random directions: off by h^2 / 6 of the third derivative (the
    gradients' weights and probabilities are below about 3 here, so below 1e-6 for h = 1e-4) and by rounding."""
    from yggdrasil_amd import ops
    n, V, top = 4, 50, 3
    x, t = rows_of(n, V, torch.float32, 11, 1.0)
    x.requires_grad_()
    gl, gh, gt = _weights(n, top, 2)
    r = ops.token_logprobs(x, t, top=top)
    dx, = torch.autograd.grad((r.logp, r.entropy, r.top_logp), x, (gl.cuda(), gh.cuda(), gt.cuda()))

    def f(z):
        p = plain(z, t, top)
        return float((p["logp"] * gl).sum() + (p["entropy"] * gh).sum() + (p["top_logp"] * gt).sum())
    h = 1e-4
    for s in range(5):
        v = torch.randn(n, V, generator=torch.Generator().manual_seed(s)).double()
        z = x.detach().double().cpu()
        want = (f(z + h * v) - f(z - h * v)) / (2 * h)
        got = float((dx.double().cpu() * v).sum())
        assert abs(got - want) <= 1e-5 * (1 + abs(want)), (got, want)


def test_bad_rows_do_not_train_silently():
    from yggdrasil_amd import ops
    x, t = rows_of(4, 40, torch.float32, 0)
    x[1, 3] = math.nan
    t[2] = 40
    x.requires_grad_()
    ops.token_logprobs(x, t).logp.sum().backward()
    assert torch.isnan(x.grad[1]).all() and torch.isnan(x.grad[2]).all()
    assert torch.isfinite(x.grad[0]).all() and torch.isfinite(x.grad[3]).all()


def test_refusals():
    from yggdrasil_amd import ops
    x = torch.zeros(3, 8, device="cuda")
    for kw in (dict(targets=torch.zeros(3)), dict(targets=torch.zeros(2, dtype=torch.int64, device="cuda")),
               dict(targets=torch.zeros(3, device="cuda")), dict(top=65), dict(top=-1), dict(top=1.0)):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, **kw)
    for bad in (x.double(), x.int(), torch.zeros(3, 0, device="cuda"), torch.tensor(1.0, device="cuda")):
        with pytest.raises(ValueError):
            ops.token_logprobs(bad)


@pytest.mark.parametrize("n, V, top", [(64, 256, 5), (2, 100000, 20)])
def test_streams_and_graphs(n, V, top):
    """On a stream of its own, and captured: every replay equals the eager call on the same inputs."""
    from yggdrasil_amd import ops
    x, t = rows_of(n, V, torch.bfloat16, 1)
    want = ops.token_logprobs(x, t, top=top)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.token_logprobs(x, t, top=top)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.token_logprobs(x, t, top=top)
    for k in range(4):
        x2, t2 = rows_of(n, V, torch.bfloat16, 50 + k)
        x.copy_(x2)
        t.copy_(t2)
        g.replay()
        torch.cuda.synchronize()
        want = ops.token_logprobs(x2, t2, top=top)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [15, 16, 17, 64, 65, 128, 129, 511, 512, 513, 1023, 1537, 2047, 2049, 32767, 32769])
@pytest.mark.parametrize("top", [8, 9, 40])
def test_borders_between_the_kernels(V, top, dtype):
    x, t = rows_of(5, V, dtype, V + top)
    x[1, ::2] = -INF
    x[2] = 1.0
    x[3, V // 2] = math.nan
    check(x, t.int(), top)


def test_second_derivatives_are_refused():
    from yggdrasil_amd import ops
    x, t = rows_of(3, 20, torch.float32, 0)
    x.requires_grad_()
    g, = torch.autograd.grad(ops.token_logprobs(x, t).logp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_outputs_alone_and_kept_graphs():
    """Each output's gradient by itself, a graph used twice, and logits that are used twice."""
    from yggdrasil_amd import ops
    x, t = rows_of(5, 300, torch.float32, 4)
    x.requires_grad_()
    r = ops.token_logprobs(x, t, top=3)
    assert not r.top_ids.requires_grad and r.logp.requires_grad and r.entropy.requires_grad and r.top_logp.requires_grad
    gl, gh, gt = _weights(5, 3, 9)
    parts = [(r.logp, gl), (r.entropy, gh), (r.top_logp, gt[:, :3])]
    one = [torch.autograd.grad(o, x, w.cuda(), retain_graph=True)[0] for o, w in parts]
    whole, = torch.autograd.grad([o for o, _ in parts], x, [w.cuda() for _, w in parts], retain_graph=True)
    again, = torch.autograd.grad([o for o, _ in parts], x, [w.cuda() for _, w in parts])
    assert torch.equal(whole, again)
    # each part's own roundings: a few steps of the largest of them
    size = sum(o.abs() for o in one)
    assert ((sum(one) - whole).abs() <= 2.0 ** -20 * size + 1e-30).all()
    with torch.no_grad():
        assert not ops.token_logprobs(x, t).logp.requires_grad


def masked_rows(V, dtype, low):
    """Rows whose masked entries hold a finite value far below the others: whole threads, waves and parts of a row see nothing
    else before (or after) they meet an allowed one."""
    x, t = rows_of(8, V, dtype, V, 2.0)
    x[0, :V // 2] = low                             # the first half
    x[1, V // 2:] = low                             # the last half
    x[2, :min(4096, V - 5)] = low                   # a whole part
    x[3, torch.rand(V, generator=torch.Generator().manual_seed(V)).cuda() < 0.9] = low
    x[4, 3:] = low                                  # three left, fewer than the alternatives
    x[5, :V - 1] = low                              # one left, the last
    x[6, :-3] = low
    x[6, :7] = -INF                                 # both masks in one row
    x[7, V // 3:V // 3 + 700] = low
    t[:] = torch.tensor([V - 1, 0, V - 2, V // 5, 1, V - 1, V - 3, 2])
    return x, t


@pytest.mark.parametrize("dtype, low", [(torch.float32, -1.0), (torch.float32, -1e38), (torch.float32, -1e9), (torch.bfloat16, -1.0),
                                        (torch.bfloat16, -1e38), (torch.float16, -1.0)], ids=str)
@pytest.mark.parametrize("V", [300, 2048, 2049, 9001, 40000, 131072])
def test_masks_of_a_finite_value(V, dtype, low):
    """low -1: the type's lowest value."""
    x, t = masked_rows(V, dtype, torch.finfo(dtype).min if low == -1 else low)
    r = check(x, t, 7)
    check(x, t.int(), 0)
    assert torch.isfinite(r.entropy).all() and torch.isfinite(r.logp).all()
    assert r.entropy[5] == 0 and r.logp[5] == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [300, 2049, 9001, 40000, 131072])
@pytest.mark.parametrize("of_logp, of_entropy", [(True, False), (False, True), (True, True)])
def test_gradient_under_masks_of_a_finite_value(V, dtype, of_logp, of_entropy):
    from yggdrasil_amd import ops
    x, t = masked_rows(V, dtype, torch.finfo(dtype).min)
    x.requires_grad_()
    gl, gh, _ = _weights(8, 0, V)
    gl, gh = gl * of_logp, gh * of_entropy
    r = ops.token_logprobs(x, t)
    outs = [(r.logp, gl)] * of_logp + [(r.entropy, gh)] * of_entropy
    dx, = torch.autograd.grad([o for o, _ in outs], x, [w.cuda() for _, w in outs])
    ref, tol = _grad64(x, t, 0, gl, gh, None)
    step = torch.finfo(dtype).eps / 2
    small = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[dtype]
    err = (dx.double().cpu() - ref).abs()
    assert (err <= tol + step * (ref.abs() + tol) + small).all(), (err - tol - step * ref.abs()).max()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [9, 256, 3000])
def test_bad_targets_make_their_whole_gradient_row_nan(V, dtype):
    """Masked entries and those whose probability underflows among them; a row without a distribution has no gradient all the
    same, and the other rows keep theirs."""
    from yggdrasil_amd import ops
    x, t = rows_of(6, V, dtype, V, 1.0)
    x[:, 1::3] = -INF
    x[:, 2] = -30000.0
    x[4] = -INF
    t[:] = torch.tensor([0, V, -2, 1 << 40, V + 7, -1])
    x.requires_grad_()
    ops.token_logprobs(x, t).logp.sum().backward()
    g = x.grad
    assert torch.isnan(g[1:4]).all()
    assert (g[4] == 0).all() and (g[5] == 0).all() and torch.isfinite(g[0]).all()


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwd
    from yggdrasil_amd import ops
    x, t = rows_of(3, 20, torch.float32, 0)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for bad in (dual, dual.reshape(3, 1, 20)[:, 0], dual[:, :17]):
            with pytest.raises(RuntimeError, match="forward"):
                ops.token_logprobs(bad, t)
            with pytest.raises(RuntimeError, match="forward"), torch.no_grad():
                ops.token_logprobs(bad, top=2)
        # a tangent of the gradient that comes in
        y = x.clone().requires_grad_()
        r = ops.token_logprobs(y, t)
        g = torch.ones(3, device="cuda")
        with pytest.raises(RuntimeError, match="forward"):
            torch.autograd.grad(r.logp, y, fwd.make_dual(g, g))
        want = ops.token_logprobs(x, t)             # nothing in hand has a tangent
        assert torch.equal(r.logp.detach(), want.logp)
    assert torch.equal(ops.token_logprobs(x, t).logp, want.logp)
    for f in (lambda: torch.func.jvp(lambda v: ops.token_logprobs(v, t).logp, (x,), (x,)),
              lambda: torch.func.vmap(lambda v: ops.token_logprobs(v).entropy)(x)):
        with pytest.raises(RuntimeError):           # transforms of torch.func hold no tensor that a kernel could read
            f()


def test_more_rows_than_a_launch_takes():
    """2^26 rows of 64 lanes are 2^32 threads: the last ones come from a second launch."""
    from yggdrasil_amd import ops
    n, V, top = (1 << 26) + 1000, 17, 9
    x = torch.randn(1 << 12, V, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).bfloat16()
    x = x.repeat((n >> 12) + 1, 1)[:n]
    t = torch.arange(n, dtype=torch.int32, device="cuda") % V
    x[-1], x[-2, 3], t[-3] = -INF, math.nan, -1
    r = ops.token_logprobs(x, t, top=top)
    for at in (slice(0, 3000), slice((1 << 26) - 3000, (1 << 26) + 3000), slice(n - 3000, n)):
        check(x[at], t[at], top)
        want = ops.token_logprobs(x[at], t[at], top=top)
        assert all(torch.equal(a[at].nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(r, want))
    # every row: the pattern comes again after 2^12 rows, the targets after V
    whole = ops.token_logprobs(x[:1 << 12], top=top)
    most = n >> 12 << 12
    assert bool((r.entropy[:most].view(-1, 1 << 12) == whole.entropy).all())
    assert bool((r.top_ids[:most].view(-1, 1 << 12, top) == whole.top_ids).all())


def test_a_single_rows_stride_is_not_used():
    """One row's distance to the next may be anything, through the C-ABI."""
    import ctypes
    from yggdrasil_amd import _lib, ops
    x, _ = rows_of(1, 300, torch.float32, 8)
    want = ops.token_logprobs(x)
    for stride in (0, -5, 2 ** 62, -2 ** 63):
        got = torch.full((1,), 7.0, device="cuda")
        _lib.check(_lib.lib().ygg_logprobs(x.data_ptr(), 0, 1, 300, ctypes.c_int64(stride), None, 0, 0, None, got.data_ptr(), None,
                                           None, None, None, 0, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(got, want.entropy)
