"""clip_grad_norm's memory and roundings: gradients that do not lie densely beside tensors that are written, and values rounded once."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_expanded_gradients_beside_what_is_written():
    """A gradient of one value that is read a thousand times reaches over four bytes, not four thousand."""
    from yggdrasil_amd import ops
    whole = torch.full((1001,), 7.0, device="cuda")
    whole[0] = 2.0
    grad, out = whole[:1].expand(1000), whole[1:]
    r, norm = ops.clip_grad_norm([grad], 1.0, out=[out])
    assert r[0] is out and abs(float(norm) - 2 * math.sqrt(1000)) < 1e-4
    assert torch.allclose(out, torch.full_like(out, 1 / math.sqrt(1000)), rtol=2.0 ** -23, atol=0) and whole[0] == 2.0


def test_gradients_apart_in_what_is_written():
    """Every second value of a buffer whose second half is written: they are read before."""
    from yggdrasil_amd import ops
    whole = torch.arange(1.0, 2001.0, device="cuda")
    grad = whole[::2]
    want = grad.double() * (1.0 / grad.double().norm())
    r, norm = ops.clip_grad_norm([grad], 1.0, out=[whole[1000:]])
    assert abs(float(norm) - math.sqrt(sum(v * v for v in range(1, 2001, 2)))) < 1e-2
    assert torch.allclose(r[0].double(), want, rtol=2.0 ** -23, atol=0)
    assert torch.equal(whole[:1000], torch.arange(1.0, 1001.0, device="cuda"))


def test_what_is_read_in_place_is_still_refused():
    from yggdrasil_amd import ops
    whole = torch.ones(100, device="cuda")
    for grads, out in (([whole[:40]], [whole[20:60]]), ([whole[:40], whole[40:80]], [whole[40:80], whole[:40]]),
                       ([whole[:40], whole[50:90]], [torch.zeros(40, device="cuda"), whole[30:70]]),
                       ([whole[::2], whole[1:51]], [whole[40:90], torch.zeros(50, device="cuda")])):
        with pytest.raises(ValueError):
            ops.clip_grad_norm(grads, 1.0, out=out)
    assert whole.eq(1).all()
