"""What the operators of a recurrent block are timed on: layer norm, the gated recurrence, the gated projections of a feed-forward
block and the clipping of gradients by their global norm, as a program that trains or serves such a block beside the model calls
them.

A case's "op" is the operator, its other entries the call's shape:

  norm   ``layer_norm``: ``rows`` rows of ``inner`` values in ``dtype``, weight and bias in ``wide`` type (f32) or the rows' own;
         ``train``: also the gradients of the rows, the weight and the bias
  scan   ``gated_scan``: ``batch`` sequences of ``steps`` steps of ``inner`` channels in ``dtype``, h_t = gate_t h_{t-1} + x_t from a
         carried state, gates in f32 (``wide``) or the type of x; ``train``: also the gradients of x, the gates and the state
  gated  ``gated_linear``: ``rows`` rows of ``inner`` values in ``dtype``, act(x Wg^T) (x Wu^T) with ``outer`` outputs;
         ``train``: also the gradients of the rows and of both matrices
  clip   ``clip_grad_norm``: the gradients of ``tensors`` tensors, ``total`` values in all, f32 or (``mixed``) some of each type,
         brought to a norm of at most ``share`` of their own
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
    return [
        # one stream's state before its head: the smallest call
        dict(name="norm_step_b1", op="norm", rows=1, inner=256, dtype="f32", wide=True, train=False),
        # a training batch of 16 sequences of 4096 tokens
        dict(name="norm_train", op="norm", rows=65536, inner=2048, dtype="bf16", wide=True, train=True),
        # a training batch of odd sizes, everything in half precision
        dict(name="norm_odd_train", op="norm", rows=4095, inner=5003, dtype="f16", wide=False, train=True),
        # one token of each of 64 served streams
        dict(name="scan_step_b64", op="scan", batch=64, steps=1, inner=256, dtype="f32", wide=True, train=False),
        # one long document read by a narrow block, its state carried from the part before
        dict(name="scan_long", op="scan", batch=1, steps=131072, inner=256, dtype="bf16", wide=True, train=False),
        # a training batch of odd sizes in f32
        dict(name="scan_odd_train", op="scan", batch=5, steps=1001, inner=1003, dtype="f32", wide=True, train=True),
        # a training batch of 16 sequences of 4096 tokens
        dict(name="scan_train", op="scan", batch=16, steps=4096, inner=2048, dtype="bf16", wide=False, train=True),
        # one token of one stream: both matrices are read for it
        dict(name="gated_step_b1", op="gated", rows=1, inner=4096, outer=8192, dtype="bf16", act="silu", train=False),
        # a few sequences, sizes that are no multiple of a tile or of 16 bytes
        dict(name="gated_odd_train", op="gated", rows=1001, inner=1000, outer=2003, dtype="f16", act="gelu", train=True),
        # a training batch through the block, the largest products
        dict(name="gated_train", op="gated", rows=16384, inner=2048, outer=4096, dtype="bf16", act="silu", train=True),
        # the gradients of a small head
        dict(name="clip_head", op="clip", tensors=6, total=70000, mixed=False, share=0.25),
        # those of a model of many matrices and vectors
        dict(name="clip_model", op="clip", tensors=60, total=120_000_000, mixed=True, share=0.25),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of one of the operators, its sizes spread over the logarithm of their ranges."""
    op = rng.choice(["norm", "scan", "scan", "gated", "gated", "clip"])
    dtype, train = rng.choice(list(DTYPES)), rng.random() < 0.6
    if op == "norm":
        inner = _log_int(rng, 8, 50000)
        most = 134_000_000 // inner // (2 if dtype == "f32" else 1)
        return dict(op=op, rows=_log_int(rng, 1, max(1, min(500_000, most))), inner=inner, dtype=dtype, wide=rng.random() < 0.5,
                    train=train)
    if op == "scan":
        most = 60_000_000 if dtype == "f32" else 100_000_000
        inner = _log_int(rng, 1, 4096)
        steps = _log_int(rng, 1, min(16384 if train else 131072, max(1, most // inner)))
        return dict(op=op, batch=_log_int(rng, 1, max(1, min(256, most // inner // steps))), steps=steps, inner=inner, dtype=dtype,
                    wide=rng.random() < 0.5, train=train)
    if op == "gated":
        inner, outer = _log_int(rng, 64, 4096), _log_int(rng, 64, 8192)
        most = int(5.4e11 / (4 * inner * outer) / (4 if dtype == "f32" else 1))
        return dict(op=op, rows=_log_int(rng, 1, max(1, min(16384, most))), inner=inner, outer=outer, dtype=dtype,
                    act=rng.choice(["silu", "gelu", "sigmoid"]), train=train)
    tensors = _log_int(rng, 1, 60)
    return dict(op=op, tensors=tensors, total=_log_int(rng, tensors, 120_000_000), mixed=rng.random() < 0.5,
                share=rng.choice([0.1, 0.25, 0.9, 2.0]))


def _parts(case):
    """Sizes and types of a case's gradients: matrices of a few sizes and short vectors, as a model's parameters are."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["total"])
    k = case["tensors"]
    weights = [rng.choice([0.01, 1.0, 1.0, 4.0]) * rng.uniform(0.5, 1.5) for _ in range(k)]
    rest = case["total"] - k
    sizes = [1 + int(rest * w / sum(weights)) for w in weights]
    sizes[-1] += case["total"] - sum(sizes)
    kinds = ["f32", "bf16", "f16"] if case["mixed"] else ["f32"]
    return [(n, kinds[i % len(kinds)]) for i, n in enumerate(sizes)]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op = case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    s = dict(case=case)
    if op == "clip":
        # gradients of a mean loss: each tensor with a scale of its own
        s["grads"] = [(normal(n) * float(10.0 ** (i % 5 - 3))).to(DTYPES[t]) for i, (n, t) in enumerate(_parts(case))]
        norm = math.sqrt(sum(float((v.double() ** 2).sum()) for v in s["grads"]))
        s["most"] = norm * case["share"]
        return s
    dtype = DTYPES[case["dtype"]]
    leaf = (lambda t: t.requires_grad_()) if case["train"] else (lambda t: t)
    if op == "norm":
        M, n = case["rows"], case["inner"]
        w_type = torch.float32 if case["wide"] else dtype
        # a block's inputs: channels of different size, a few large, rows off zero
        channel = (0.3 + uniform(n)) * (1.0 + 9.0 * (uniform(n) < 0.01))
        x = normal(M, n) * channel
        x += 0.5 * normal(M, 1)
        s["x"] = leaf(x.to(dtype))
        s["weight"], s["bias"] = leaf((1 + 0.2 * normal(n)).to(w_type)), leaf((0.1 * normal(n)).to(w_type))
        if case["train"]:
            s["d_y"] = normal(M, n).to(dtype)
        return s
    if op == "scan":
        B, T, n = case["batch"], case["steps"], case["inner"]
        g_type = torch.float32 if case["wide"] else dtype
        # channels that forget within a few steps and channels that hold for hundreds; a document begins every 2000 steps or so
        gate = torch.sigmoid(normal(B, T, n) + 6.0 * uniform(n) - 1.0)
        x = normal(B, T, n) * torch.sqrt(1 - gate * gate)
        gate *= uniform(B, T, 1) >= 0.0005
        s["gate"], s["x"], s["state"] = leaf(gate.to(g_type)), leaf(x.to(dtype)), leaf(normal(B, n))
        if case["train"]:
            s["d_h"], s["d_last"] = normal(B, T, n).to(dtype), normal(B, n)
        return s
    M, K, N = case["rows"], case["inner"], case["outer"]
    s["x"] = leaf(normal(M, K).to(dtype))
    s["w"] = leaf((normal(2, N, K) / math.sqrt(K)).to(dtype))
    if case["train"]:
        s["d_y"] = normal(M, N).to(dtype)
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _plain_norm(s):
    """With m and v a row's mean and variance, z = (x - m) / sqrt(v + eps): y = z w + b. With q = w dy: dx = (q - mean(q) -
    z mean(q z)) / sqrt(v + eps), dw = sum over the rows of dy z, db of dy."""
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    off = x - x.mean(-1, keepdim=True)
    inv = 1.0 / torch.sqrt((off * off).mean(-1, keepdim=True) + EPS)
    z = off * inv
    out = {"y": (z * w + b).to(s["x"].dtype)}
    if s["case"]["train"]:
        dy = s["d_y"].float()
        q = dy * w
        dx = (q - q.mean(-1, keepdim=True) - z * (q * z).mean(-1, keepdim=True)) * inv
        out["d_x"] = dx.to(s["x"].dtype)
        out["d_weight"] = (dy * z).sum(0).to(s["weight"].dtype)
        out["d_bias"] = dy.sum(0).to(s["bias"].dtype)
    return out


def _doubled(a, v):
    """v_t + a_t v_{t-1} + a_t a_{t-1} v_{t-2} + ... along axis 1, in place: each step from the one `by` before it, by doubling."""
    by, T = 1, v.shape[1]
    while by < T:
        v[:, by:] += a[:, by:] * v[:, :-by]
        a[:, by:] = a[:, by:] * a[:, :-by]
        by *= 2
    return v


def _plain_scan(s):
    """h_t = gate_t h_{t-1} + x_t. With e_t = dh_t + gate_{t+1} e_{t+1} (the last one's with the final state's gradient):
    dx_t = e_t, dgate_t = e_t h_{t-1}, dstate = gate_0 e_0."""
    gate, x, state = s["gate"].detach().float(), s["x"].detach().float(), s["state"].detach()
    h = x if x.data_ptr() != s["x"].data_ptr() else x.clone()
    h[:, 0] += gate[:, 0] * state
    h = _doubled(gate.clone(), h)
    out = {"h": h.to(s["x"].dtype), "last": h[:, -1].clone()}
    if s["case"]["train"]:
        e = s["d_h"].float().flip(1)
        e[:, 0] += s["d_last"]
        after = torch.cat([torch.zeros_like(gate[:, :1]), gate[:, 1:].flip(1)], 1)
        e = _doubled(after, e).flip(1)
        out["d_x"] = e.to(s["x"].dtype)
        out["d_gate"] = (e * torch.cat([state[:, None], h[:, :-1]], 1)).to(s["gate"].dtype)
        out["d_state"] = gate[:, 0] * e[:, 0]
    return out


def _act(name, g):
    """An activation and its derivative."""
    if name == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    p = 1.0 / (1.0 + torch.exp(-g))
    return (g * p, p * (1.0 + g * (1.0 - p))) if name == "silu" else (p, p * (1.0 - p))


def _plain_gated(s):
    """With g = x Wg^T and u = x Wu^T: y = act(g) u; dg = dy u act'(g), du = dy act(g); dx = dg Wg + du Wu, dWg = dg^T x,
    dWu = du^T x."""
    c, x, w = s["case"], s["x"].detach().float(), s["w"].detach().float()
    g, u = torch.mm(x, w[0].t()), torch.mm(x, w[1].t())
    a, slope = _act(c["act"], g)
    out = {"y": (a * u).to(s["x"].dtype)}
    if c["train"]:
        dy = s["d_y"].float()
        dg, du = dy * u * slope, dy * a
        out["d_x"] = (torch.mm(dg, w[0]) + torch.mm(du, w[1])).to(s["x"].dtype)
        out["d_w"] = torch.stack([torch.mm(dg.t(), x), torch.mm(du.t(), x)]).to(s["w"].dtype)
    return out


def _plain_clip(s):
    """norm = sqrt of the sum of all squares (in 64 bits); where it is more than the most allowed, every value times most / norm."""
    norm = torch.sqrt(torch.stack([(v.double() ** 2).sum() for v in s["grads"]]).sum())
    most = torch.full_like(norm, s["most"])
    by = torch.where(norm > most, most / norm, torch.ones_like(norm)).float()
    return {"grads": [(v.float() * by).to(v.dtype) for v in s["grads"]], "norm": norm.float()}


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own_norm(s):
    from yggdrasil_amd import ops
    y = ops.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["d_y"])
    return {"y": y, "d_x": dx, "d_weight": dw, "d_bias": db}


def _own_scan(s):
    from yggdrasil_amd import ops
    h, last = ops.gated_scan(s["gate"], s["x"], s["state"])
    if not s["case"]["train"]:
        return {"h": h, "last": last}
    dx, dg, ds = torch.autograd.grad((h, last), (s["x"], s["gate"], s["state"]), (s["d_h"], s["d_last"]))
    return {"h": h, "last": last, "d_x": dx, "d_gate": dg, "d_state": ds}


def _own_gated(s):
    from yggdrasil_amd import ops
    y = ops.gated_linear(s["x"], s["w"], s["case"]["act"])
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["d_y"])
    return {"y": y, "d_x": dx, "d_w": dw}


def _own_clip(s):
    from yggdrasil_amd import ops
    grads, norm = ops.clip_grad_norm(s["grads"], s["most"])
    return {"grads": grads, "norm": norm}


def run(s):
    op = s["case"]["op"]
    if own:
        return {"norm": _own_norm, "scan": _own_scan, "gated": _own_gated, "clip": _own_clip}[op](s)
    return {"norm": _plain_norm, "scan": _plain_scan, "gated": _plain_gated, "clip": _plain_clip}[op](s)


# ---------------------------------------------------------------------------------------------- work and exact values
def work(case):
    op = case["op"]
    if op == "clip":
        size = sum(n * BYTES[t] for n, t in _parts(case))
        return {"bytes": 2 * size + 4, "flops": 3 * case["total"]}
    b, train = BYTES[case["dtype"]], case["train"]
    w = 4 if case.get("wide") else b
    if op == "norm":
        n, cells = case["inner"], case["rows"] * case["inner"]
        return {"bytes": cells * b * (4 if train else 2) + n * w * (4 if train else 2), "flops": cells * (20 if train else 8)}
    if op == "scan":
        cells, ends = case["batch"] * case["steps"] * case["inner"], 4 * case["batch"] * case["inner"]
        return {"bytes": cells * ((2 * w + 4 * b) if train else (w + 2 * b)) + ends * (4 if train else 2),
                "flops": cells * (5 if train else 2)}
    M, K, N = case["rows"], case["inner"], case["outer"]
    once = M * K + 2 * N * K + M * N
    return {"bytes": once * b * (2 if train else 1), "flops": (12 if train else 4) * M * N * K}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        total = sum((v.double() * v.double()).sum() for v in s["grads"])
        norm = total.sqrt()
        by = min(1.0, s["most"] / float(norm)) if float(norm) > 0 else 1.0
        return {"grads": [v.double() * by for v in s["grads"]], "norm": norm}
    train = case["train"]
    if op == "norm":
        x, w, b = (s[k].detach().double() for k in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS)
        z = (x - mean) / sd
        out = {"y": w * z + b}
        if train:
            dy = s["d_y"].double()
            t = w * dy
            n = case["inner"]
            out["d_x"] = (n * t - t.sum(-1, keepdim=True) - z * (t * z).sum(-1, keepdim=True)) / (n * sd)
            out["d_weight"], out["d_bias"] = (z * dy).sum(0), dy.sum(0)
        return out
    if op == "scan":
        gate, x, h = s["gate"].detach().double(), s["x"].detach().double(), s["state"].detach().double()
        T = case["steps"]
        before = torch.empty_like(x)
        out = {"h": torch.empty_like(x)}
        for t in range(T):
            before[:, t] = h
            h = torch.addcmul(x[:, t], gate[:, t], h)
            out["h"][:, t] = h
        out["last"] = h
        if train:
            dh, e = s["d_h"].double(), s["d_last"].double()
            del x
            dx = torch.empty_like(dh)
            for t in range(T - 1, -1, -1):
                e = e + dh[:, t]
                dx[:, t] = e
                e = e * gate[:, t]
            out.update(d_x=dx, d_gate=dx * before, d_state=e)
        return out
    x, w = s["x"].detach().double(), s["w"].detach().double()
    g, u = x @ w[0].t(), x @ w[1].t()
    if case["act"] == "gelu":
        phi = torch.special.ndtr(g)
        a, slope = g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    else:
        p = torch.sigmoid(g)
        a, slope = (g * p, p + g * p * (1 - p)) if case["act"] == "silu" else (p, p * (1 - p))
    out = {"y": a * u}
    if train:
        dy = s["d_y"].double()
        dg, du = dy * u * slope, dy * a
        out["d_x"] = dg @ w[0] + du @ w[1]
        out["d_w"] = torch.stack([dg.t() @ x, du.t() @ x])
    return out
