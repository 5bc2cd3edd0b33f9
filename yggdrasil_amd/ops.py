"""Operators of an output head and of a recurrent block on the GPU, for programs that train, score or serve them next to the
model's own step:

    r = token_logprobs(logits, tokens, top=5)       # .logp, .entropy, .top_logp, .top_ids; differentiable
    offsets, order = group_rows(leaves, experts)    # rows by the expert they take
    y = grouped_matmul(x, w, offsets, order)        # y_i = W[expert of i] x_i; differentiable
    y = int8_linear(x, w_int8, w_scale)             # rows quantised to int8, an int8 matrix with scales

    y = layer_norm(x, weight, bias)                 # differentiable
    h, last = gated_scan(gate, x, state)            # h_t = gate_t h_{t-1} + x_t; differentiable
    y = gated_linear(x, w, "silu")                  # silu(x w[0]^T) (x w[1]^T); differentiable
    grads, norm = clip_grad_norm(grads, 1.0)        # by the norm of all of them

The kernels are those of csrc/ygg_logprobs.hip, ygg_experts.hip and ygg_int8.hip, and of ygg_norm.hip, ygg_gated_scan.hip,
ygg_gated.hip and ygg_clip.hip, through the C-ABI of include/ygg_hip.h, on the current torch stream of the tensors' device (csrc/ygg_torch.cpp: allocation, the call, autograd).
Nothing waits for the GPU, so a call can be captured into a graph; values that only the GPU holds (tokens, offsets, an order)
are not checked here, and bad ones give wrong or NaN values, never an access out of bounds. Types: float32, bfloat16 and
float16. Derivatives are first ones in reverse mode: second ones and forward-mode tangents are refused.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOST_TOP = 64
MOST_VOCAB = 1 << 24
MOST_ROWS = 1 << 24
MOST_EXPERTS = 1 << 20
MOST_INNER = 1 << 17
MOST_STEPS = 1 << 30
MOST_VALUES = 1 << 40
ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}


def _floats(t, name: str) -> torch.Tensor:
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _TYPES):
        raise ValueError(f"{name} must be a float32, bfloat16 or float16 tensor on a ROCm device")
    return t


def _on(t, device, name: str, dtypes, shape=None) -> None:
    if not (isinstance(t, torch.Tensor) and t.device == device and t.dtype in dtypes):
        raise ValueError(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)} on {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} of shape {tuple(t.shape)}, expected {tuple(shape)}")


def _tensors(x, *others) -> bool:
    """A device tensor, and tensors: what the native calls take as they are."""
    if not (type(x) is torch.Tensor and x.is_cuda):
        return False
    for t in others:
        if type(t) is not torch.Tensor:
            return False
    return True


_ENTRIES = ("ygg_logprobs_scratch", "ygg_logprobs", "ygg_logprobs_grad", "ygg_grouped_matmul", "ygg_grouped_grad_x",
            "ygg_grouped_grad_w", "ygg_int8_scratch", "ygg_int8_linear", "ygg_layer_norm", "ygg_layer_norm_scratch",
            "ygg_layer_norm_grad", "ygg_gated_scan", "ygg_gated_scan_scratch", "ygg_gated_scan_kept", "ygg_gated_scan_grad", "ygg_gated_linear",
            "ygg_gated_linear_kept", "ygg_gated_linear_scratch", "ygg_gated_linear_grad", "ygg_clip_scratch", "ygg_clip_grad_norm", "ygg_last_error")
_module = None


def _native():
    """csrc/ygg_torch.cpp, bound to the library's entries."""
    global _module
    if _module is None:
        try:
            from . import _ygg_torch
        except ImportError as e:
            raise ImportError(f"the torch part of yggdrasil_amd is not built ({e}): run `python -m yggdrasil_amd.build`") from e
        lib = _lib.lib()
        _ygg_torch.bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _ENTRIES})
        _module = _ygg_torch
    return _module


# ---------------------------------------------------------------------------------------------- log-probabilities
class LogProbs(NamedTuple):
    logp: Optional[torch.Tensor]        # of the given tokens, None without any
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor]    # of the most likely tokens, None for top 0
    top_ids: Optional[torch.Tensor]     # int32


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """logits as (rows, V), values next to each other, rows at any distance of at least V; a copy where they are not."""
    if logits.is_contiguous() and logits.dim() == 2:
        return logits
    V = logits.shape[-1]
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if x.shape[0] <= 1:
        return x if x.stride(1) == 1 or V == 1 else x.contiguous()
    return x if (x.stride(1) == 1 or V == 1) and x.stride(0) >= V else x.contiguous()


def token_logprobs(logits, targets=None, top: int = 0) -> LogProbs:
    """logits (..., V) -> the log-probabilities (...) f32 in nats of targets (...) int32 or int64 (None: none are given), the
    entropy (...) f32 of every row's distribution, and its `top` most likely tokens (..., top) in falling order, equal ones
    by rising id: their log-probabilities f32 and ids int32. One pass over the logits; differentiable in logp, entropy and
    top_logp (one more pass).

    Entries of -inf are masked: they are never among the most likely tokens (what is missing of `top` has the id -1 and
    log-probability -inf), and a row of them alone has log-probability -inf, entropy 0 and no gradient. A target of -1 is no
    token: its log-probability is 0, without a gradient. Other targets outside [0, V), and rows that hold a NaN or +inf,
    give NaN."""
    if (_tensors(logits) if targets is None else _tensors(logits, targets)) and type(top) is int:
        r = _native().plain_token_logprobs(logits, targets, top)
        if r is not None:
            return LogProbs(*r)
    _floats(logits, "logits")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MOST_VOCAB:
        raise ValueError(f"logits of shape {tuple(logits.shape)}: the last axis holds 1 to {MOST_VOCAB} classes")
    if not (isinstance(top, int) and 0 <= top <= MOST_TOP):
        raise ValueError(f"top {top!r}: 0 to {MOST_TOP}")
    lead = logits.shape[:-1]
    if targets is not None:
        _on(targets, logits.device, "targets", (torch.int32, torch.int64), lead)
        if len(lead) != 1 or not targets.is_contiguous():
            targets = targets.reshape(-1).contiguous()
    r = _native().token_logprobs(_rows(logits), targets, top)
    if len(lead) == 1:
        return LogProbs(*r)
    return LogProbs(*(None if v is None else v.reshape(lead + v.shape[1:]) for v in r))


# ---------------------------------------------------------------------------------------------- products of experts
def group_rows(leaves, n_experts: int):
    """The rows by the expert they take, for grouped_matmul: leaves (...) int32 or int64 -> offsets (n_experts + 1) int32 and
    order (rows) int32: expert e takes the rows order[offsets[e]:offsets[e + 1]], in rising order, so that sums over them
    come out the same every time. Rows whose leaf is outside [0, n_experts) come last and belong to none."""
    if not (isinstance(leaves, torch.Tensor) and leaves.is_cuda and leaves.dtype in (torch.int32, torch.int64)):
        raise ValueError("leaves must be an int32 or int64 tensor on a ROCm device")
    if not 1 <= n_experts <= MOST_EXPERTS:
        raise ValueError(f"n_experts {n_experts}: 1 to {MOST_EXPERTS}")
    x = leaves.reshape(-1)
    x = torch.where((x >= 0) & (x < n_experts), x, n_experts).to(torch.int32)      # in this order: int64 ones may not fit
    by, order = torch.sort(x, stable=True)
    ends = torch.arange(n_experts + 1, dtype=torch.int32, device=x.device)
    return torch.searchsorted(by, ends, out_int32=True), order.to(torch.int32)


def grouped_matmul(x, w, offsets, order=None) -> torch.Tensor:
    """Rows x (M, K) times the matrix of the expert each takes, w (E, N, K) -> y (M, N) in their type, y_i = w[expert] x_i.
    offsets (E + 1) int32, rising from 0: expert e takes the places offsets[e] to offsets[e + 1] - 1, of any number. Place p
    is row order[p] (order (M) int32, a permutation; None: row p). Rows past offsets[E] get 0. Differentiable in x and w."""
    if _tensors(x, w, offsets) if order is None else _tensors(x, w, offsets, order):
        y = _native().plain_grouped_matmul(x, w, offsets, order)
        if y is not None:
            return y
    _floats(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x of shape {tuple(x.shape)}, expected (M, K)")
    _on(w, x.device, "w", (x.dtype,))
    M, K = x.shape
    if w.dim() != 3 or w.shape[2] != K:
        raise ValueError(f"w of shape {tuple(w.shape)}, expected (E, N, {K})")
    E, N, _ = w.shape
    if M > MOST_ROWS or not 1 <= E <= MOST_EXPERTS or not 1 <= N <= MOST_INNER or not 1 <= K <= MOST_INNER:
        raise ValueError(f"M = {M}, E = {E}, N = {N}, K = {K}: at most {MOST_ROWS} rows, 1 to {MOST_EXPERTS} experts, N and K "
                         f"1 to {MOST_INNER}")
    _on(offsets, x.device, "offsets", (torch.int32,), (E + 1,))
    if order is not None:
        _on(order, x.device, "order", (torch.int32,), (M,))
        if not order.is_contiguous():
            order = order.contiguous()
    if not (x.is_contiguous() and w.is_contiguous() and offsets.is_contiguous()):
        x, w, offsets = x.contiguous(), w.contiguous(), offsets.contiguous()
    return _native().grouped_matmul(x, w, offsets, order)


# ---------------------------------------------------------------------------------------------- the int8 projection
def quantize_weight(w):
    """A float matrix (N, K) -> int8 (N, K) and the scale (N) f32 of each of its rows, max |row| / 127, for int8_linear."""
    if not (isinstance(w, torch.Tensor) and w.dim() == 2 and w.is_floating_point()):
        raise ValueError("w must be a float matrix (N, K)")
    if not bool(torch.isfinite(w).all()):
        raise ValueError("w holds a NaN or an infinity")
    w = w.detach().double()
    scale = (w.abs().amax(1) / 127).float().clamp_min(2.0 ** -126)
    return torch.round(w / scale.double()[:, None]).clamp(-127, 127).to(torch.int8), scale


def int8_linear(x, w, w_scale) -> torch.Tensor:
    """x (..., K) times an int8 matrix w (N, K) whose row n has the scale w_scale[n] (f32) -> (..., N) in x's type. Each row
    of x is quantised to int8 with a scale of its own, max |row| / 127, and the products are summed in whole numbers. A row
    that holds a NaN or an infinity gives NaN. For serving: there is no gradient."""
    if _tensors(x, w, w_scale):
        y = _native().plain_int8_linear(x, w, w_scale)
        if y is not None:
            return y
    _floats(x, "x")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("int8_linear has no gradient: call it under torch.no_grad() or with x.detach()")
    if x.dim() < 1:
        raise ValueError("x needs an axis of K values")
    K = x.shape[-1]
    _on(w, x.device, "w", (torch.int8,))
    if w.dim() != 2 or w.shape[1] != K:
        raise ValueError(f"w of shape {tuple(w.shape)}, expected (N, {K})")
    N = w.shape[0]
    _on(w_scale, x.device, "w_scale", (torch.float32,), (N,))
    if w_scale.requires_grad and torch.is_grad_enabled():
        raise ValueError("int8_linear has no gradient: call it under torch.no_grad() or with w_scale.detach()")
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    M = x2.shape[0]
    if M > MOST_ROWS or not 1 <= N <= MOST_VOCAB or not 1 <= K <= MOST_INNER:
        raise ValueError(f"{M} rows, N = {N}, K = {K}: at most {MOST_ROWS} rows, N 1 to {MOST_VOCAB}, K 1 to {MOST_INNER}")
    if not (x2.is_contiguous() and w.is_contiguous() and w_scale.is_contiguous()):
        x2, w, w_scale = x2.contiguous(), w.contiguous(), w_scale.contiguous()
    y = _native().int8_linear(x2, w, w_scale)
    return y if x.dim() == 2 else y.reshape(x.shape[:-1] + (N,))


# ---------------------------------------------------------------------------------------------- a recurrent block
def layer_norm(x, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """x (..., n) -> (x - mean) / sqrt(variance + eps) * weight + bias over the last axis, in x's type. weight and bias (n) are
    f32 or in x's type, both the same; None: ones, zeros. Mean and variance (the mean of the squares about the mean) are in
    f32. Differentiable in all three; the gradients of weight and bias are summed in f32, in the same order every time. A row
    that holds a NaN or an infinity is NaN."""
    if type(eps) is float and _tensors(x, *[t for t in (weight, bias) if t is not None]):
        y = _native().plain_layer_norm(x, weight, bias, eps)
        if y is not None:
            return y
    _floats(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MOST_INNER:
        raise ValueError(f"x of shape {tuple(x.shape)}: the last axis holds 1 to {MOST_INNER} values")
    n = x.shape[-1]
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _on(t, x.device, name, (torch.float32, x.dtype), (n,))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight in {weight.dtype}, bias in {bias.dtype}: both in one type")
    if not (isinstance(eps, (int, float)) and 0 <= eps <= 1e30):
        raise ValueError(f"eps {eps!r}: a finite number of at least 0")
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    return _native().layer_norm(_rows(x), weight, bias, float(eps)).reshape(x.shape)


def _steps(t: torch.Tensor) -> torch.Tensor:
    """t (B, T, n), a step's channels next to each other; a copy where they are not."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def gated_scan(gate, x, state=None):
    """The gated recurrence h_t = gate_t h_{t-1} + x_t of every channel: gate and x (B, T, n), the gate in f32 or in x's type, and
    the state before the first step (B, n) f32 (None: zeros) -> h (B, T, n) in x's type and the last state (B, n) f32. For
    serving, one step at a time with the state carried on; for training, differentiable in all three, over long sequences.

    States are held in f32. Runs of steps are joined by the products of their gates: gates are meant to be at most 1 in
    magnitude, and others have to keep the product of every run of steps finite; a state that becomes infinite may come out as NaN
    later on. A gate of 0 begins anew (a document's first
    step); a step with gate 1 and x 0 keeps the state (padding behind a sequence's end leaves the last state right). For the gate's
    gradient every 64th state is kept, in f32, and the others are computed again from x."""
    if _tensors(x, gate) if state is None else _tensors(x, gate, state):
        r = _native().plain_gated_scan(gate, x, state)
        if r is not None:
            return r
    _floats(x, "x")
    if x.dim() != 3:
        raise ValueError(f"x of shape {tuple(x.shape)}, expected (B, T, n)")
    _on(gate, x.device, "gate", (torch.float32, x.dtype), x.shape)
    B, T, n = x.shape
    if B > MOST_ROWS or T > MOST_STEPS or not 1 <= n <= MOST_INNER:
        raise ValueError(f"B = {B}, T = {T}, n = {n}: at most {MOST_ROWS} sequences of {MOST_STEPS} steps, n 1 to {MOST_INNER}")
    if state is not None:
        _on(state, x.device, "state", (torch.float32,), (B, n))
        state = state.contiguous()
    return _native().gated_scan(_steps(gate), _steps(x), state)


def gated_linear(x, w, activation: str = "silu") -> torch.Tensor:
    """The gated projections of a feed-forward block in one kernel: x (..., K), w (2, N, K) in x's type ->
    act(x w[0]^T) (x w[1]^T) (..., N) in x's type, act "silu" (g sigmoid(g)), "gelu" (g Phi(g)) or "sigmoid". Sums and
    the product are in f32, rounded once. Differentiable in x and w: for that, both projections are kept (in f32, or its upper 24
    bits for 16-bit types), and the gradients' products take their factors in x's type: dy u act'(g) and dy act(g) are rounded to it
    before the sums. In float16 that is with a power of two for each row (for the gradient of x) and column (for that of w) where its
    range would not do, so that they reach as far as float32's, and what is under 2^-22 of the largest beside it may be lost."""
    act = ACTIVATIONS.get(activation) if isinstance(activation, str) else None
    if act is None:
        raise ValueError(f"activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    if _tensors(x, w):
        y = _native().plain_gated_linear(x, w, act)
        if y is not None:
            return y
    _floats(x, "x")
    if x.dim() < 1:
        raise ValueError("x needs an axis of K values")
    K = x.shape[-1]
    _on(w, x.device, "w", (x.dtype,))
    if w.dim() != 3 or w.shape[0] != 2 or w.shape[2] != K:
        raise ValueError(f"w of shape {tuple(w.shape)}, expected (2, N, {K})")
    N = w.shape[1]
    if not 1 <= N <= MOST_INNER // 2 or not 1 <= K <= MOST_INNER:
        raise ValueError(f"N = {N}, K = {K}: N 1 to {MOST_INNER // 2}, K 1 to {MOST_INNER}")
    x2 = x.reshape(-1, K).contiguous()
    if len(x2) > MOST_ROWS:
        raise ValueError(f"{len(x2)} rows: at most {MOST_ROWS}")
    return _native().gated_linear(x2, w.contiguous(), act).reshape(x.shape[:-1] + (N,))


def _clip(grads, most: float, clip: bool, out=None):
    grads = list(grads)
    out = out if out is None else list(out)
    if grads and _tensors(*grads) and (out is None or (out and _tensors(*out))):
        r = _native().plain_clip_grad_norm(grads, most, clip, out)
        if r is not None:
            return (r[0] if out is None else out), r[1]
    some = [i for i, g in enumerate(grads) if g is not None]
    if not some:
        raise ValueError("no gradients")
    tensors = [grads[i] for i in some]
    for g in tensors:
        _floats(g, "a gradient")
        if g.device != tensors[0].device or g.layout != torch.strided or g.numel() > MOST_VALUES:
            raise ValueError(f"gradients must be dense tensors on one device, of at most {MOST_VALUES} values each")
        if clip and g.requires_grad and torch.is_grad_enabled():
            raise ValueError("clip_grad_norm has no gradient: call it under torch.no_grad() or with detached tensors")
    if out is not None:
        if len(out) != len(grads) or any((o is None) != (g is None) for o, g in zip(out, grads)):
            raise ValueError("out must hold a tensor for every gradient, and None where there is none")
        to = [out[i] for i in some]
        for o, g in zip(to, tensors):
            _on(o, g.device, "out", (g.dtype,), g.shape)
            if o.requires_grad and torch.is_grad_enabled():
                raise ValueError("out must hold tensors that require no gradient")
        return out, _native().clip_grad_norm(tensors, most, clip, to)[1]
    r, norm = _native().clip_grad_norm(tensors, most, clip, None)
    if clip and len(some) < len(grads):
        whole = [None] * len(grads)
        for i, t in zip(some, r):
            whole[i] = t
        r = whole
    return r, norm


def grad_norm(grads) -> torch.Tensor:
    """The norm of all values of the tensors together (None: left out), the root of the sum of their squares: () f32 (infinite past its
    largest), squares summed in 64 bits, in the same order every time."""
    with torch.no_grad():
        return _clip(grads, 0.0, False)[1]


def clip_grad_norm(grads, max_norm: float, out=None):
    """Gradients (None: there is none) brought to a norm of at most max_norm together: each times min(1, max_norm / norm), rounded
    once -> the list of them, and the norm that they had, () f32. New tensors, or out: tensors of their shapes and types, also
    the gradients themselves (out=grads: in place); no others may share memory with what is written. A norm that is NaN or
    infinite in 64 bits, in which the squares are summed, leaves the values as they are, and the caller sees it in the norm; one that is
    only past float32's largest comes back as infinite too, but the values are clipped by it. Nothing waits for the GPU."""
    if not (isinstance(max_norm, (int, float)) and max_norm >= 0):
        raise ValueError(f"max_norm {max_norm!r}: a number of at least 0")
    return _clip(grads, float(max_norm), True, out)


__all__ = ["LogProbs", "token_logprobs", "group_rows", "grouped_matmul", "quantize_weight", "int8_linear", "layer_norm",
           "gated_scan", "gated_linear", "grad_norm", "clip_grad_norm"]
