"""The output head's operators on any host: what their Python calls and their C-ABI refuse, before a device is touched."""
import ctypes

import pytest
import torch

from yggdrasil_amd import _lib, ops


def test_python_refuses_host_tensors():
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="ROCm"):
        ops.token_logprobs(x)
    with pytest.raises(ValueError, match="ROCm"):
        ops.grouped_matmul(x, torch.zeros(2, 4, 8), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="ROCm"):
        ops.group_rows(torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="ROCm"):
        ops.int8_linear(x, torch.zeros(4, 8, dtype=torch.int8), torch.ones(4))
    with pytest.raises(ValueError, match="ROCm"):
        ops.token_logprobs(x.double())
    with pytest.raises(ValueError, match="ROCm"):
        ops.token_logprobs([1.0, 2.0])


def test_quantize_weight_on_the_host():
    w = torch.tensor([[1.0, -127.0, 63.4, 0.0], [0.0, 0.0, 0.0, 0.0], [1e-3, 2e-3, -4e-3, 3e-3]])
    q, s = ops.quantize_weight(w)
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    assert q[0].tolist() == [1, -127, 63, 0] and q[1].tolist() == [0, 0, 0, 0]
    assert s[0] == 1.0 and s[1] == 2.0 ** -126
    # half a step of each row's scale, and the scale's own rounding
    assert ((q.double() * s.double()[:, None] - w.double()).abs() <= s.double()[:, None] * (0.5 + 127 * 2.0 ** -23)).all()
    for bad in (torch.zeros(3), torch.zeros(2, 2, dtype=torch.int8), torch.tensor([[float("nan")]])):
        with pytest.raises(ValueError):
            ops.quantize_weight(bad)


# an address that no call may reach: the sizes are refused first
P = ctypes.c_void_p(4096)


def _logprobs(type=0, rows=1, V=8, stride=8, bytes=0, top=0, x=P, t=None, logp=None, ent=P, tl=None, ti=None, scratch=None,
              n=0):
    return _lib.lib().ygg_logprobs(x, type, rows, V, stride, t, bytes, top, logp, ent, tl, ti, None, scratch, n, None)


@pytest.mark.parametrize("kw, word", [
    (dict(type=3), b"type"), (dict(type=-1), b"type"), (dict(rows=-1), b"rows"), (dict(V=0), b"V"),
    (dict(V=(1 << 24) + 1), b"V"), (dict(rows=2, stride=7), b"apart"), (dict(top=-1), b"top"), (dict(top=65), b"top"),
    (dict(bytes=2), b"target_bytes"), (dict(x=None), b"NULL"), (dict(ent=None), b"NULL"), (dict(bytes=4), b"NULL"),
    (dict(bytes=4, t=P), b"NULL"), (dict(top=1), b"NULL"), (dict(top=1, tl=P), b"NULL")])
def test_logprobs_refuses(kw, word):
    assert _logprobs(**kw) == 5
    assert word in _lib.lib().ygg_last_error()


def test_logprobs_without_rows_is_done():
    assert _logprobs(rows=0, x=None, ent=None) == 0
    L = _lib.lib()
    assert L.ygg_logprobs_grad(None, 0, 0, 8, 8, None, 0, 0, None, None, None, None, None, None, None, None) == 0
    assert L.ygg_logprobs_scratch(0, 0, 8, 0) == 0 and L.ygg_logprobs_scratch(9, 1, 8, 0) == 0


@pytest.mark.parametrize("kw, word", [
    (dict(type=3), b"type"), (dict(rows=-1), b"rows"), (dict(V=0), b"V"), (dict(rows=2, stride=7), b"apart"),
    (dict(top=65), b"top"), (dict(g=P), b"target_bytes"), (dict(g=P, bytes=4), b"NULL"), (dict(out=None), b"NULL"),
    (dict(stats=None), b"NULL"), (dict(top=1, gt=P), b"NULL")])
def test_logprobs_grad_refuses(kw, word):
    a = dict(type=0, rows=1, V=8, stride=8, bytes=0, top=0, stats=P, g=None, gt=None, out=P)
    a.update(kw)
    L = _lib.lib()
    assert L.ygg_logprobs_grad(P, a["type"], a["rows"], a["V"], a["stride"], None, a["bytes"], a["top"], P, None, a["stats"],
                               a["g"], None, a["gt"], a["out"], None) == 5
    assert word in L.ygg_last_error()


@pytest.mark.parametrize("entry", ["ygg_grouped_matmul", "ygg_grouped_grad_x", "ygg_grouped_grad_w"])
@pytest.mark.parametrize("kw, word", [
    (dict(type=3), b"type"), (dict(M=-1), b"M "), (dict(M=(1 << 24) + 1), b"M "), (dict(E=0), b"E "),
    (dict(E=(1 << 20) + 1), b"E "), (dict(N=0), b"N "), (dict(K=0), b"K "), (dict(K=(1 << 17) + 1), b"K "),
    (dict(off=None), b"NULL"), (dict(a=None), b"NULL"), (dict(b=None), b"NULL"), (dict(out=None), b"NULL")])
def test_grouped_refuses(entry, kw, word):
    v = dict(a=P, b=P, type=0, off=P, M=4, E=2, N=8, K=8, out=P)
    v.update(kw)
    L = _lib.lib()
    assert getattr(L, entry)(v["a"], v["b"], v["type"], v["off"], None, v["M"], v["E"], v["N"], v["K"], v["out"], None) == 5
    assert word in L.ygg_last_error()


def test_grouped_without_rows_is_done():
    L = _lib.lib()
    assert L.ygg_grouped_matmul(None, None, 0, P, None, 0, 2, 8, 8, None, None) == 0
    assert L.ygg_grouped_grad_x(None, None, 0, P, None, 0, 2, 8, 8, None, None) == 0


@pytest.mark.parametrize("kw, word", [
    (dict(type=7), b"type"), (dict(M=-1), b"M "), (dict(N=0), b"N "), (dict(K=0), b"K "), (dict(K=(1 << 17) + 1), b"K "),
    (dict(x=None), b"NULL"), (dict(w=None), b"NULL"), (dict(ws=None), b"NULL"), (dict(y=None), b"NULL"),
    (dict(M=9, N=3, K=77, n=0), b"scratch"), (dict(M=9, N=3, K=77, scratch=None), b"scratch")])
def test_int8_refuses(kw, word):
    v = dict(x=P, type=0, w=P, ws=P, M=1, N=8, K=8, y=P, scratch=P, n=1 << 30)
    v.update(kw)
    L = _lib.lib()
    assert L.ygg_int8_linear(v["x"], v["type"], v["w"], v["ws"], v["M"], v["N"], v["K"], v["y"], v["scratch"], v["n"],
                             None) == 5
    assert word in L.ygg_last_error()
    assert L.ygg_int8_scratch(0, 8, 8) == 0 and L.ygg_int8_scratch(1, 8, 1 << 18) == 0
    assert L.ygg_int8_linear(None, 0, None, None, 0, 8, 8, None, None, 0, None) == 0


def test_native_errors_are_raised():
    """The torch part raises the library's message (sizes the library refuses, on host tensors that it never reads)."""
    with pytest.raises(RuntimeError, match="NULL|type|outside"):
        ops._native()
        _lib.check(_lib.lib().ygg_int8_linear(None, 7, None, None, 1, 1, 1, None, None, 0, None))


@pytest.mark.gpu
def test_the_torch_part_raises_the_librarys_errors():
    """Sizes that ops.py would refuse, given to the torch part itself: the library refuses them and its message is raised. No
    kernel runs."""
    m = ops._native()
    x, w = torch.zeros(2, ops.MOST_INNER + 1, device="cuda"), torch.zeros(3, ops.MOST_INNER + 1, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError, match=r"K 131073 outside \[1, 131072\] \(error 5\)"):
        m.int8_linear(x, w, torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError, match=r"top 65 outside \[0, 64\] \(error 5\)"):
        m.token_logprobs(torch.zeros(2, 100, device="cuda"), None, 65)
    off = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match=r"K 131073 outside \[1, 131072\] \(error 5\)"):
        m.grouped_matmul(x, torch.zeros(1, 1, ops.MOST_INNER + 1, device="cuda"), off, None)


def test_the_limits_are_the_headers():
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "ygg_hip.h").read_text()
    names = re.findall(r"YGG_(MOST_[A-Z]+) = ([0-9 <]+)", text)
    assert len(names) == 5
    for name, value in names:
        a = [int(v) for v in value.split("<<")]
        assert getattr(ops, name) == (a[0] if len(a) == 1 else a[0] << a[1]), name


@pytest.mark.parametrize("entry, N, K", [("ygg_grouped_matmul", 2048, 8), ("ygg_grouped_matmul", 1 << 17, 1 << 17),
                                         ("ygg_grouped_grad_x", 8, 8192), ("ygg_grouped_grad_w", 8, 2048),
                                         ("ygg_grouped_grad_w", 1 << 17, 1 << 17)])
@pytest.mark.parametrize("type", [0, 1, 2])
def test_more_tiles_than_a_launch_takes(entry, N, K, type):
    """A launch holds less than 2^32 threads: sizes within the limits that make more are refused as arguments, not by the
    device."""
    L = _lib.lib()
    assert getattr(L, entry)(P, P, type, P, None, 1 << 21, 1 << 20, N, K, P, None) == 5
    assert b"launch takes" in L.ygg_last_error()
