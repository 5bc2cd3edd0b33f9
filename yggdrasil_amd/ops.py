"""Operators of an output head on the GPU, for programs that train, score or serve one next to the model's own step:

    r = token_logprobs(logits, tokens, top=5)       # .logp, .entropy, .top_logp, .top_ids; differentiable
    offsets, order = group_rows(leaves, experts)    # rows by the expert they take
    y = grouped_matmul(x, w, offsets, order)        # y_i = W[expert of i] x_i; differentiable
    y = int8_linear(x, w_int8, w_scale)             # rows quantised to int8, an int8 matrix with scales

The kernels are those of csrc/ygg_logprobs.hip, csrc/ygg_experts.hip and csrc/ygg_int8.hip, through the C-ABI of
include/ygg_hip.h, on the current torch stream of the tensors' device (csrc/ygg_torch.cpp: allocation, the call, autograd).
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
            "ygg_grouped_grad_w", "ygg_int8_scratch", "ygg_int8_linear", "ygg_last_error")
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


__all__ = ["LogProbs", "token_logprobs", "group_rows", "grouped_matmul", "quantize_weight", "int8_linear"]
