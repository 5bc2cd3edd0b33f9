"""clip_grad_norm rounds each value once: a product next to the middle of two of the type's values goes to the nearer one, also where f32
between would be that middle."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rounded_once(v, dtype):
    """v (f64) to the nearest of dtype, ties to even, in whole numbers of its step."""
    e = torch.frexp(v)[1] - 1
    least = {torch.bfloat16: -126, torch.float16: -14}[dtype]
    bits = {torch.bfloat16: 7, torch.float16: 10}[dtype]
    step = torch.ldexp(torch.ones_like(v), e.clamp_min(least) - bits)
    return ((v / step).round() * step).to(dtype)      # round: ties to even; the result is a value of dtype


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_next_to_the_middle(dtype):
    """A tensor of ones of norm 1 times 1/2 + half a step, and 2^-40 more or less."""
    from yggdrasil_amd import ops
    half = 0.5 + torch.finfo(dtype).eps / 4
    for sign in (1.0, -1.0):
        for to in (half + 2.0 ** -40, half - 2.0 ** -40, half):
            v = torch.zeros(100, dtype=dtype, device="cuda")
            v[37] = sign
            (out,), norm = ops.clip_grad_norm([v], to)
            assert norm == 1
            want = rounded_once(torch.tensor([sign * to], dtype=torch.float64), dtype)
            assert out[37].cpu() == want[0], (sign, to - half)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_all_values(dtype):
    """Every finite value of the type, times a factor close to a number of few bits, so that many products lie next to a middle."""
    from yggdrasil_amd import ops
    v = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[v.isfinite()]
    norm = v.double().norm()
    for factor in (0.75 + 2.0 ** -33, 0.625 - 2.0 ** -33, 0.5 + 2.0 ** -12 + 2.0 ** -38, 0.3):
        most = float(norm * factor)
        (out,), got = ops.clip_grad_norm([v.cuda()], most)
        # the norm that the call divides by is a sum in another order: the factor is known to 2^-50, so products that lie closer to a
        # middle than that are left out
        exact = v.double() * (most / float(norm))
        lo, hi = rounded_once(exact * (1 - 2.0 ** -48), dtype), rounded_once(exact * (1 + 2.0 ** -48), dtype)
        sure = lo == hi
        assert sure.float().mean() > 0.5
        assert torch.equal(out.cpu()[sure], lo[sure])
