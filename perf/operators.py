"""What the output head's operators are timed on: the products of routed experts, the int8 projection and the
log-probabilities, as a program that trains, scores or serves a head calls them.

A case's "op" is the operator, its other entries the call's shape:

  logprobs   ``token_logprobs``: ``rows`` rows of logits over ``vocab`` classes in ``dtype`` (each row followed by ``pad``
             unused entries): the given tokens' log-probabilities, every row's entropy and its ``top`` most likely
             tokens; ``train``: also the logits' gradient; ``masked``: a part of each row's entries is -inf
  grouped    ``grouped_matmul``: ``rows`` rows of ``inner`` values, each multiplied by the (``outer``, ``inner``) matrix of
             its expert among ``experts``, of which the share ``hot`` goes to the 16 favoured ones (a quarter of the
             experts where there are fewer than 64); ``order``: the rows lie in their own order and are gathered;
             ``train``: also the gradients of the rows and of the experts' matrices
  int8       ``int8_linear``: ``rows`` rows of ``inner`` values in ``dtype``, quantised per row, times an int8 (``outer``,
             ``inner``) matrix with a scale for each of its rows
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
SMALLEST_SCALE = 2.0 ** -126


def listed():
    return [
        # one stream's step over bytes, with the alternatives an interactive user is shown: the smallest call
        dict(name="logprobs_step_b1", op="logprobs", rows=1, vocab=256, dtype="f32", top=5, train=False, masked=False,
             pad=0),
        # scored windows over bytes, 64 streams of 4096 tokens
        dict(name="logprobs_score_bytes", op="logprobs", rows=262144, vocab=256, dtype="f32", top=5, train=False,
             masked=False, pad=0),
        # a served batch's step over a wide vocabulary whose masked tokens may not be sampled
        dict(name="logprobs_wide_b8", op="logprobs", rows=8, vocab=131072, dtype="bf16", top=20, train=False, masked=True,
             pad=0),
        # the loss of a training batch over a vocabulary of odd size
        dict(name="logprobs_loss_odd", op="logprobs", rows=4095, vocab=50257, dtype="bf16", top=0, train=True,
             masked=False, pad=0),
        # the readout of a routed layer of the deepest router: few rows an expert, most of them to a few
        dict(name="grouped_leaf_readout", op="grouped", rows=4096, experts=16384, inner=128, outer=8, dtype="f32", hot=0.9,
             order=True, train=False),
        # a training batch through the layer inputs of a routed layer of the large trained shape
        dict(name="grouped_leaf_train", op="grouped", rows=65536, experts=1024, inner=256, outer=64, dtype="f32", hot=0.5,
             order=True, train=True),
        # one token of each of a few streams through wide experts
        dict(name="grouped_step_b16", op="grouped", rows=16, experts=64, inner=2048, outer=1536, dtype="bf16", hot=0.25,
             order=False, train=False),
        # a training batch through wide experts, sizes that are no multiple of a tile, ragged loads
        dict(name="grouped_wide_train", op="grouped", rows=16001, experts=64, inner=2040, outer=1528, dtype="bf16", hot=0.5,
             order=False, train=True),
        # the prompts of a batch through few large experts, the largest product
        dict(name="grouped_large", op="grouped", rows=16384, experts=8, inner=4096, outer=4096, dtype="f16", hot=0.25,
             order=True, train=False),
        # one token of one stream through an int8 projection
        dict(name="int8_step_b1", op="int8", rows=1, inner=4096, outer=8192, dtype="bf16"),
        # a few requests' tokens through an int8 projection of odd sizes
        dict(name="int8_ragged_b77", op="int8", rows=77, inner=1000, outer=5003, dtype="f32"),
        # the prompts of a batch through an int8 projection
        dict(name="int8_prompt", op="int8", rows=8192, inner=4096, outer=8192, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of one of the operators, its sizes spread over the logarithm of their ranges."""
    op = rng.choice(["logprobs", "logprobs", "grouped", "grouped", "grouped", "int8", "int8"])
    if op == "logprobs":
        vocab = _log_int(rng, 2, 160000)
        train = rng.random() < 0.4
        return dict(op=op, rows=_log_int(rng, 1, max(1, min(262144, 150_000_000 // vocab))), vocab=vocab,
                    dtype=rng.choice(list(DTYPES)), top=rng.choice([0, 1, 5, 20, rng.randint(0, 32)]), train=train,
                    masked=rng.random() < 0.3, pad=rng.choice([0, 0, 0, rng.randint(1, 40)]))
    if op == "grouped" and rng.random() < 0.5:
        # the framework's routed layers: many experts of small matrices
        experts, outer, inner = 2 ** rng.randint(4, 14), _log_int(rng, 8, 64), 16 * _log_int(rng, 1, 16)
        return dict(op=op, rows=_log_int(rng, 1, 30000), experts=experts, inner=inner, outer=outer,
                    dtype=rng.choice(list(DTYPES)), hot=round(rng.uniform(0.1, 0.5), 2), order=rng.random() < 0.7,
                    train=rng.random() < 0.4 and experts * inner * outer <= 1 << 27)
    if op == "grouped":
        # few experts of large matrices
        experts, outer, inner = rng.randint(2, 64), _log_int(rng, 200, 4096), _log_int(rng, 200, 4096)
        train = rng.random() < 0.4
        most = int(5.4e11 / (2 * inner * outer * (3 if train else 1)))
        return dict(op=op, rows=_log_int(rng, 1, max(1, min(16384, most))), experts=experts, inner=inner, outer=outer,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), hot=round(rng.uniform(0.1, 0.5), 2),
                    order=rng.random() < 0.5, train=train)
    inner, outer = _log_int(rng, 64, 8192), _log_int(rng, 64, 16384)
    return dict(op=op, rows=_log_int(rng, 1, max(1, min(8192, int(2.7e11 / (inner * outer))))), inner=inner, outer=outer,
                dtype=rng.choice(list(DTYPES)))


def _hot(case):
    return min(16, case["experts"] // 4) or 1


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype, rows = DTYPES[case["dtype"]], case["rows"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "logprobs":
        V = case["vocab"]
        # a model's logits: a spread of a few nats, some rows sure of their token and some not
        whole = torch.empty(rows, V + case["pad"], dtype=dtype, device="cuda")
        for at in range(0, rows, 8192):
            part = whole[at:at + 8192]
            spread = 0.5 + 3.0 * torch.rand(len(part), 1, generator=g, device="cuda")
            part.copy_(normal(*part.shape) * spread)
        logits = whole[:, :V]
        targets = torch.randint(V, (rows,), generator=g, device="cuda", dtype=torch.int32)
        if case["masked"]:
            allowed = 0.1 + 0.8 * torch.rand(rows, 1, generator=g, device="cuda")
            for at in range(0, rows, 8192):
                part = logits[at:at + 8192]
                drop = torch.rand(part.shape, generator=g, device="cuda") > allowed[at:at + 8192]
                drop.scatter_(1, targets[at:at + 8192, None].long(), False)
                part.masked_fill_(drop, -math.inf)
        if case["train"]:
            # padding has no token: a tenth of the places
            targets[torch.rand(rows, generator=g, device="cuda") < 0.1] = -1
        s = dict(case=case, logits=logits, targets=targets)
        if case["train"]:
            s["logits"] = logits.requires_grad_()
            s["d_logp"] = -torch.rand(rows, generator=g, device="cuda") / rows      # a loss's weights
            s["d_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda")       # and an entropy bonus
        return s
    if case["op"] == "grouped":
        E, K, N = case["experts"], case["inner"], case["outer"]
        names = torch.randperm(E, generator=g, device="cuda")
        to_hot = torch.rand(rows, generator=g, device="cuda") < case["hot"]
        pick = torch.where(to_hot, torch.randint(_hot(case), (rows,), generator=g, device="cuda"),
                           torch.randint(E, (rows,), generator=g, device="cuda"))
        leaves = names[pick]
        counts = torch.bincount(leaves, minlength=E)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = counts.cumsum(0)
        order = None
        if case["order"]:
            order = torch.argsort(leaves, stable=True).to(torch.int32)
        else:
            leaves = leaves.sort().values
        s = dict(case=case, x=normal(rows, K).to(dtype), w=(normal(E, N, K) / math.sqrt(K)).to(dtype), leaves=leaves,
                 offsets=offsets, order=order, longest=int(counts.max()))
        if case["train"]:
            s["x"].requires_grad_()
            s["w"].requires_grad_()
            s["d_y"] = normal(rows, N).to(dtype)
        return s
    K, N = case["inner"], case["outer"]
    # activations with a few large channels, as quantised projections meet them
    x = normal(rows, K) * (1.0 + 7.0 * (torch.rand(K, generator=g, device="cuda") < 0.02))
    w = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    w_scale = (0.5 + torch.rand(N, generator=g, device="cuda")) / (73.0 * math.sqrt(K))
    return dict(case=case, x=x.to(dtype), w=w, w_scale=w_scale)


# ---------------------------------------------------------------------------------------------- the plain forms
def _plain_logprobs(s):
    """With x a row's logits and m their maximum: logp_c = (x_c - m) - log(sum exp(x - m)), entropy = -sum p logp, in 32
    bits; a row with no entry left gives logp -inf and entropy 0, a token of -1 gives 0. The gradient is
    (g_logp at the token) - p sum(g_logp) - g_entropy p (logp + entropy)."""
    c, logits, targets = s["case"], s["logits"].detach(), s["targets"].long()
    x = logits.float()
    top = x.max(-1, keepdim=True).values
    none = top == -math.inf
    e = torch.exp(x - torch.where(none, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    logp = torch.where(none, top, x - top - torch.log(total))
    p = torch.where(none, torch.zeros_like(e), e / total)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    entropy = -plogp.sum(-1)
    given = targets >= 0
    at = torch.where(given, targets, torch.zeros_like(targets))
    picked = logp.gather(1, at[:, None])[:, 0]
    out = {"logp": torch.where(given, picked, torch.zeros_like(picked)), "entropy": entropy}
    if c["top"]:
        k = min(c["top"], c["vocab"])
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
        best = logp.gather(1, ids)
        ids = torch.where(best == -math.inf, torch.full_like(ids, -1), ids)
        if k < c["top"]:
            ids = torch.cat([ids, ids.new_full((len(ids), c["top"] - k), -1)], 1)
            best = torch.cat([best, best.new_full((len(ids), c["top"] - k), -math.inf)], 1)
        out["top_ids"], out["top_logp"] = ids.to(torch.int32), best
    if c["train"]:
        g = torch.where(given, s["d_logp"], torch.zeros_like(s["d_logp"]))
        d = -p * g[:, None] - s["d_entropy"][:, None] * (plogp + p * entropy[:, None])
        d.scatter_add_(1, at[:, None], torch.where(none[:, 0], torch.zeros_like(g), g)[:, None])
        out["d_logits"] = d.to(logits.dtype)
    return out


def _plain_grouped(s):
    """y_i = W[expert of i] x_i; d_x_i = W[expert of i]^T d_y_i; d_W[e] = sum over its rows of d_y_i x_i^T. Few small
    products go by row over the gathered matrices, others by expert over rows padded to the longest expert's."""
    c, leaves = s["case"], s["leaves"]
    x, w = s["x"].detach(), s["w"].detach()
    dtype, M, E, N, K = x.dtype, len(x), c["experts"], c["outer"], c["inner"]
    if M * N * K <= 1 << 27:
        mine, xf = w[leaves].float(), x.float()
        out = {"y": (mine * xf[:, None, :]).sum(-1).to(dtype)}
        if c["train"]:
            dy = s["d_y"].float()
            out["d_x"] = (mine * dy[:, :, None]).sum(1).to(dtype)
            d_w = torch.zeros(E, N, K, device=x.device)
            out["d_w"] = d_w.index_add_(0, leaves, dy[:, :, None] * xf[:, None, :]).to(dtype)
        return out
    if s["order"] is not None:
        order = s["order"].long()
    else:
        order = torch.arange(M, device=x.device)
    e = leaves[order]
    place = torch.arange(M, device=x.device) - s["offsets"].long()[e]
    slot = torch.empty_like(place)
    slot[order] = place
    wf = w.float()
    xp = torch.zeros(E, s["longest"], K, device=x.device)
    xp[leaves, slot] = x.float()
    out = {"y": torch.bmm(xp, wf.transpose(1, 2).contiguous())[leaves, slot].to(dtype)}
    if c["train"]:
        dyp = torch.zeros(E, s["longest"], N, device=x.device)
        dyp[leaves, slot] = s["d_y"].float()
        out["d_x"] = torch.bmm(dyp, wf)[leaves, slot].to(dtype)
        out["d_w"] = torch.bmm(dyp.transpose(1, 2).contiguous(), xp).to(dtype)
    return out


def _plain_int8(s):
    """Row i's scale is s_i = max(max |x_i| / 127, 2^-126) in 32 bits and its integers q = round(x / s_i), ties to even;
    y = (q . w) s_i w_scale."""
    x = s["x"].float()
    most = x.abs().amax(-1, keepdim=True)
    scale = (most / torch.full_like(most, 127.0)).clamp_min(SMALLEST_SCALE)
    q = torch.round(x / scale)
    return {"y": (torch.mm(q, s["w"].float().t()) * scale * s["w_scale"]).to(s["x"].dtype)}


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own_logprobs(s):
    from yggdrasil_amd import ops
    c = s["case"]
    r = ops.token_logprobs(s["logits"], s["targets"], top=c["top"])
    out = {"logp": r.logp, "entropy": r.entropy}
    if c["top"]:
        out["top_ids"], out["top_logp"] = r.top_ids, r.top_logp
    if c["train"]:
        out["d_logits"], = torch.autograd.grad((r.logp, r.entropy), s["logits"], (s["d_logp"], s["d_entropy"]))
    return out


def _own_grouped(s):
    from yggdrasil_amd import ops
    y = ops.grouped_matmul(s["x"], s["w"], s["offsets"], s["order"])
    if not s["case"]["train"]:
        return {"y": y}
    d_x, d_w = torch.autograd.grad(y, (s["x"], s["w"]), s["d_y"])
    return {"y": y, "d_x": d_x, "d_w": d_w}


def _own_int8(s):
    from yggdrasil_amd import ops
    return {"y": ops.int8_linear(s["x"], s["w"], s["w_scale"])}


def run(s):
    op = s["case"]["op"]
    if own:
        return {"logprobs": _own_logprobs, "grouped": _own_grouped, "int8": _own_int8}[op](s)
    return {"logprobs": _plain_logprobs, "grouped": _plain_grouped, "int8": _plain_int8}[op](s)


# ---------------------------------------------------------------------------------------------- work and exact values
def work(case):
    b, M = BYTES[case["dtype"]], case["rows"]
    if case["op"] == "logprobs":
        n = M * case["vocab"]
        return {"bytes": n * b * (2 if case["train"] else 1) + M * (4 + 8 + 8 * case["top"] + (8 if case["train"] else 0)),
                "flops": n * (10 if case["train"] else 5)}
    K, N = case["inner"], case["outer"]
    if case["op"] == "grouped":
        E, hot = case["experts"], _hot(case)
        # experts that some row takes, in expectation: the matrices that have to be read
        some = (hot * -math.expm1(-M * (case["hot"] / hot + (1 - case["hot"]) / E))
                + (E - hot) * -math.expm1(-M * (1 - case["hot"]) / E))
        rows = M * (K + N) * b + 4 * (E + 1) + (4 * M if case["order"] else 0)
        matrices = some * N * K * b
        if not case["train"]:
            return {"bytes": rows + matrices, "flops": 2 * M * N * K}
        return {"bytes": 2 * M * (K + N) * b + rows - M * (K + N) * b + matrices + E * N * K * b, "flops": 6 * M * N * K}
    return {"bytes": M * K * b + N * K + 4 * N + M * N * b, "flops": 2 * M * N * K}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int8":
        x = s["x"].double()
        scale = (x.abs().max(1).values / 127).float().double().clamp(min=SMALLEST_SCALE)
        q = torch.round((x / scale[:, None]).float()).double()
        w = s["w"].double() * s["w_scale"].double()[:, None]
        return {"y": (q * scale[:, None]) @ w.t()}
    if case["op"] == "grouped":
        x, w = s["x"].detach(), s["w"].detach()
        out = {"y": torch.zeros(case["rows"], case["outer"], dtype=torch.float64, device="cuda")}
        if case["train"]:
            out["d_x"] = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
            out["d_w"] = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        ends = s["offsets"].tolist()
        rows = torch.argsort(s["leaves"], stable=True)
        for e in range(case["experts"]):
            if ends[e] == ends[e + 1]:
                continue
            mine = rows[ends[e]:ends[e + 1]]
            we, xe = w[e].double(), x[mine].double()
            out["y"][mine] = xe @ we.t()
            if case["train"]:
                dy = s["d_y"][mine].double()
                out["d_x"][mine] = dy @ we
                out["d_w"][e] = dy.t() @ xe
        return out
    logits, V, k = s["logits"].detach(), case["vocab"], case["top"]
    parts = []
    step = max(1, (1 << 26) // V)
    for at in range(0, case["rows"], step):
        x, t = logits[at:at + step].double(), s["targets"][at:at + step].long()
        logp = torch.log_softmax(x, -1)
        some = torch.isfinite(logp)
        p = torch.exp(logp)
        h = -torch.where(some, p * torch.where(some, logp, 0.0), 0.0).sum(-1)
        empty = torch.isneginf(x).all(-1)
        h = torch.where(empty, 0.0, h)
        row = torch.arange(len(x), device="cuda")
        chosen = torch.where(t < 0, 0.0, torch.where(empty, -math.inf, logp[row, t.clamp(min=0)]))
        part = {"logp": chosen, "entropy": h}
        if k:
            best, ids = torch.sort(x, dim=-1, descending=True, stable=True)
            best, ids = best[:, :k], ids[:, :k]
            gone = torch.isneginf(best)
            value = torch.where(gone, -math.inf, logp.gather(1, ids))
            more = max(0, k - V)
            part["top_ids"] = torch.nn.functional.pad(torch.where(gone, -1, ids), (0, more), value=-1).to(torch.int32)
            part["top_logp"] = torch.nn.functional.pad(value, (0, more), value=-math.inf)
        if case["train"]:
            g = torch.where(t < 0, 0.0, s["d_logp"][at:at + step].double())
            ge = s["d_entropy"][at:at + step].double()
            hit = torch.zeros_like(p)
            hit[row, t.clamp(min=0)] = 1.0
            d = g[:, None] * (hit - p) - ge[:, None] * torch.where(some, p * (torch.where(some, logp, 0.0) + h[:, None]), 0.0)
            part["d_logits"] = torch.where(empty[:, None], 0.0, d)
        parts.append(part)
    return {name: torch.cat([q[name] for q in parts]) for name in parts[0]}
