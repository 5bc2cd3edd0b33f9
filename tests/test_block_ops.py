"""A recurrent block's operators on any host: what their Python calls and their C-ABI refuse, before a device is touched."""
import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from yggdrasil_amd import _lib, ops

# an address that no call may reach: the sizes are refused first
P = ctypes.c_void_p(4096)


def test_python_refuses_host_tensors():
    x = torch.zeros(2, 3, 8)
    for call in (lambda: ops.layer_norm(x), lambda: ops.gated_scan(x, x), lambda: ops.gated_linear(x, torch.zeros(2, 4, 8)),
                 lambda: ops.grad_norm([x]), lambda: ops.clip_grad_norm([x], 1.0), lambda: ops.layer_norm([1.0]),
                 lambda: ops.gated_scan(None, None)):
        with pytest.raises(ValueError, match="ROCm"):
            call()
    with pytest.raises(ValueError, match="max_norm"):
        ops.clip_grad_norm([x], math.nan)
    with pytest.raises(ValueError, match="activation"):
        ops.gated_linear(x, x, "tanh")
    with pytest.raises(ValueError, match="no gradients"):
        ops.grad_norm([])


def refused(name, defaults, kw, word):
    v = dict(defaults)
    v.update(kw)
    assert getattr(_lib.lib(), name)(*v.values()) == 5
    assert word in _lib.lib().ygg_last_error()


NORM = dict(x=P, type=1, rows=2, n=8, stride=8, w=P, b=P, w_type=0, eps=1e-5, y=P, stats=None, stream=None)


@pytest.mark.parametrize("kw, word", [
    (dict(type=3), b"type"), (dict(w_type=2), b"weight_type"), (dict(rows=-1), b"rows"), (dict(n=0), b"n "), (dict(n=(1 << 17) + 1), b"n "),
    (dict(stride=7), b"apart"), (dict(eps=-1.0), b"eps"), (dict(eps=math.nan), b"eps"), (dict(eps=math.inf), b"eps"), (dict(x=None), b"NULL"),
    (dict(y=None), b"NULL")])
def test_layer_norm_refuses(kw, word):
    refused("ygg_layer_norm", NORM, kw, word)


NORM_GRAD = dict(x=P, type=1, rows=2, n=8, stride=8, w=P, w_type=0, stats=P, dy=P, dx=P, dw=P, db=P, scratch=P, bytes=1 << 40, stream=None)


@pytest.mark.parametrize("kw, word", [
    (dict(type=-1), b"type"), (dict(w_type=2), b"weight_type"), (dict(rows=-1), b"rows"), (dict(n=0), b"n "), (dict(stride=7), b"apart"),
    (dict(stats=None), b"NULL"), (dict(dy=None), b"NULL"), (dict(x=None), b"NULL"), (dict(scratch=None), b"scratch"), (dict(bytes=8), b"scratch"),
    (dict(n=20000, stride=20000, dw=None, db=None, scratch=None), b"scratch")])
def test_layer_norm_grad_refuses(kw, word):
    refused("ygg_layer_norm_grad", NORM_GRAD, kw, word)


SCAN = dict(gate=P, gate_type=0, gate_b=8, gate_t=8, x=P, type=1, x_b=8, x_t=8, B=1, T=4, n=8, state=None, h=P, last=P, kept=None, scratch=P,
            bytes=1 << 40, stream=None)


@pytest.mark.parametrize("kw, word", [
    (dict(type=3), b"type"), (dict(gate_type=2), b"gate_type"), (dict(B=-1), b"B "), (dict(B=(1 << 24) + 1), b"B "), (dict(T=-1), b"T "),
    (dict(T=(1 << 30) + 1), b"T "), (dict(n=0), b"n "), (dict(gate_t=-8), b"strides"), (dict(x_b=-1), b"strides"), (dict(gate=None), b"NULL"),
    (dict(x=None), b"NULL"), (dict(h=None), b"NULL"), (dict(last=None), b"NULL"), (dict(T=1 << 20, scratch=None), b"scratch"),
    (dict(T=1 << 20, bytes=8), b"scratch"), (dict(B=1 << 24, T=64, n=1 << 17), b"launch takes"),
    (dict(B=1 << 24, T=1 << 30, n=1 << 17), b"2^50")])
def test_gated_scan_refuses(kw, word):
    refused("ygg_gated_scan", SCAN, kw, word)


SCAN_GRAD = dict(gate=P, gate_type=0, gate_b=8, gate_t=8, x=P, type=1, x_b=8, x_t=8, B=1, T=4, n=8, state=None, kept=P, dh=P, dlast=None, dx=P,
                 dg=P, ds=None, scratch=P, bytes=1 << 40, stream=None)


@pytest.mark.parametrize("kw, word", [
    (dict(type=3), b"type"), (dict(gate_type=2), b"gate_type"), (dict(B=-1), b"B "), (dict(T=-1), b"T "), (dict(n=0), b"n "),
    (dict(gate_b=-8), b"strides"), (dict(x_t=-8), b"strides"), (dict(gate=None), b"NULL"), (dict(x=None), b"NULL"),
    (dict(T=65, kept=None), b"NULL"), (dict(T=1 << 20, scratch=None), b"scratch")])
def test_gated_scan_grad_refuses(kw, word):
    refused("ygg_gated_scan_grad", SCAN_GRAD, kw, word)


GATED = dict(x=P, w=P, type=1, act=0, M=4, N=8, K=8, y=P, gu=None, stream=None)
GATED_GRAD = dict(x=P, w=P, gu=P, dy=P, type=1, act=0, M=4, N=8, K=8, dx=P, dw=P, scratch=P, bytes=1 << 40, stream=None)
SIZES = [(dict(type=3), b"type"), (dict(act=3), b"act"), (dict(act=-1), b"act"), (dict(M=-1), b"M "), (dict(M=(1 << 24) + 1), b"M "),
         (dict(N=0), b"N "), (dict(N=(1 << 16) + 1), b"N "), (dict(K=0), b"K "), (dict(K=(1 << 17) + 1), b"K "), (dict(x=None), b"NULL"),
         (dict(w=None), b"NULL")]


@pytest.mark.parametrize("kw, word", SIZES + [(dict(y=None), b"NULL")])
def test_gated_linear_refuses(kw, word):
    refused("ygg_gated_linear", GATED, kw, word)


@pytest.mark.parametrize("kw, word", SIZES + [(dict(gu=None), b"NULL"), (dict(dy=None), b"NULL"), (dict(scratch=None), b"scratch"),
                                              (dict(bytes=100), b"scratch")])
def test_gated_linear_grad_refuses(kw, word):
    refused("ygg_gated_linear_grad", GATED_GRAD, kw, word)


def clip(sizes=(4, 4), types=(0, 1), most=1.0, tensors=(4096, 8192), out=(4096, 8192), norm=P, scratch=P, bytes=1 << 40, count=None):
    n = len(sizes)
    pointers = lambda v: None if v is None else (ctypes.c_void_p * n)(*v)
    return _lib.lib().ygg_clip_grad_norm(pointers(tensors), None if sizes is None else (ctypes.c_int64 * n)(*sizes),
                                         None if types is None else (ctypes.c_int * n)(*types), n if count is None else count, most,
                                         pointers(out), norm, scratch, bytes, None)


@pytest.mark.parametrize("kw, word", [
    (dict(count=-1), b"count"), (dict(sizes=(4, -1)), b"tensor 1"), (dict(sizes=(4, 1 << 50)), b"tensor 1"), (dict(types=(0, 3)), b"type"),
    (dict(most=-1.0), b"most"), (dict(most=math.nan), b"most"), (dict(tensors=None), b"NULL"), (dict(types=None), b"NULL"),
    (dict(norm=None), b"NULL"), (dict(tensors=(4096, None)), b"tensor 1"), (dict(out=(None, 4096)), b"tensor 0"), (dict(scratch=None), b"scratch"),
    (dict(bytes=8), b"scratch")])
def test_clip_refuses(kw, word):
    assert clip(**kw) == 5
    assert word in _lib.lib().ygg_last_error()


def test_nothing_to_do_is_done():
    L = _lib.lib()
    assert L.ygg_layer_norm(*{**NORM, "rows": 0, "x": None, "y": None}.values()) == 0
    assert L.ygg_gated_scan(*{**SCAN, "B": 0}.values()) == 0
    assert L.ygg_gated_scan_grad(*{**SCAN_GRAD, "T": 0}.values()) == 0
    assert L.ygg_gated_linear(*{**GATED, "M": 0}.values()) == 0
    assert L.ygg_gated_linear_grad(*{**GATED_GRAD, "dx": None, "dw": None}.values()) == 0
    assert L.ygg_layer_norm_scratch(0, 0, 8) == 0 and L.ygg_layer_norm_scratch(5, 1, 8) == 0
    assert L.ygg_gated_scan_scratch(0, 0, 0, 8, 8) == 0 and L.ygg_gated_scan_scratch(0, 0, 512, 100, 1024) == 0
    assert [L.ygg_gated_scan_kept(2, t, 5) for t in (0, 1, 64, 65, 128, 129, 4096)] == [0, 0, 0, 40, 40, 80, 63 * 40]
    assert L.ygg_gated_linear_scratch(7, 1, 1, 1) == 0 and L.ygg_gated_linear_scratch(1, 0, 8, 8) == 0
    assert L.ygg_gated_linear_kept(1, 0, 8) == 0 and L.ygg_gated_linear_kept(1, 5, 8) == 240 and L.ygg_gated_linear_kept(0, 5, 8) == 320
    assert L.ygg_clip_scratch(None, 3) == 0


def test_the_limits_are_the_headers():
    text = (Path(__file__).resolve().parents[1] / "include" / "ygg_hip.h").read_text()
    names = re.findall(r"#define YGG_(MOST_[A-Z]+) \(+(?:\(int64_t\))?\(?([0-9]+) << ([0-9]+)\)", text)
    assert len(names) == 2
    for name, value, by in names:
        assert getattr(ops, name) == int(value) << int(by), name
