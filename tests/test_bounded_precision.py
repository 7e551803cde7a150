"""The bound of bounded_precision.py tells rounded weights from split ones: both
worked out on the CPU in 64 bits, with the 16-bit roundings planted."""
import pytest
import torch

from bounded_precision import bound


def attend(dtype, n, D, split):
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(m, D, generator=g).to(dtype).double() for m in (8, n, n))
    s = q @ k.T / D ** 0.5
    p = torch.exp(s - s.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    hi = p.to(dtype).double()
    w = hi + (p - hi).to(dtype).double() if split else hi
    got = ((w @ v) / total).to(dtype).double()
    over = (got - p @ v / total).abs() > bound(p @ v / total, p @ v.abs() / total, v.abs().sum(0), n, dtype)
    return int(over.sum())


@pytest.mark.parametrize("n,D", [(40, 64), (100, 128), (64, 256)])
def test_bound_needs_the_remainder(n, D):
    for dtype in (torch.float16, torch.bfloat16):
        assert attend(dtype, n, D, split=True) == 0
    assert attend(torch.bfloat16, n, D, split=False) > 20
