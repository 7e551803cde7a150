"""Angles of far positions in the paged append: the turns since position 0 are
dropped before anything is rounded, so that keys are rotated as exactly there as
near 0.  Reference: angles to 60 decimal digits, reduced, then 64 bits."""
from decimal import Decimal, getcontext

import pytest
import torch

import b2engine as b2
import kv4_ref as R
from test_gpu_append import empty_cache


def turn():
    """2 pi to 60 digits: 16 atan 1/5 - 4 atan 1/239 is pi."""
    getcontext().prec = 80

    def atan_inverse(n):
        term = total = Decimal(1) / n
        k = 1
        while abs(term) > Decimal(10) ** -75:
            term /= -n * n
            k += 2
            total += term / k
        return total
    return 2 * (16 * atan_inverse(5) - 4 * atan_inverse(239))


def angles(positions, inv_freq):
    """position * inv_freq less whole turns, in 64 bits: off by less than 2^-51."""
    full = turn()
    out = [[float(((Decimal(p) * Decimal(f) + full / 2) % full) - full / 2) for f in inv_freq] for p in positions]
    return torch.tensor(out, dtype=torch.float64)


def test_angles_of_the_reference():
    a = angles([0, 1, 7, 1000], [1.0, 0.25])
    assert a[0].tolist() == [0, 0] and a[1].tolist() == [1, 0.25] and a[2, 1] == 1.75
    want = torch.tensor([7.0, 1000.0], dtype=torch.float64)
    assert torch.allclose(torch.sin(a[2:, 0]), torch.sin(want), rtol=0, atol=1e-14)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 64), (256, 256), (128, 72)])
@pytest.mark.parametrize("at", [0, 8190, 131071, 2 ** 24 + 1, 2 ** 31 - 300])
def test_keys_that_nearly_vanish(cuda, D, rot, at):
    """x1 cos a - x2 sin a of (x1, x2) = r (sin a, cos a), rounded to halves: 2^-12 r and less is left, in groups whose
    codes then step by 2^-15 r.  An angle off by 2^-22 moves a code by 2^-7 of a step, so that a few in a thousand come
    out otherwise.  Keys rotated to 2^-47 of r hold what the reference holds; its own, off by 2^-50 r or so, are nearer
    to a border between two codes than that once in 2^30 codes."""
    n, nkv, half = 128, 2, rot // 2
    freq = [1.0 - i / (4 * half) for i in range(half)]  # all of them turn fast
    a = angles(range(at, at + n), freq)[:, None, :].cuda()
    g = torch.Generator(device="cuda").manual_seed(5)
    r = 1 + torch.rand(n, nkv, half, generator=g, device="cuda", dtype=torch.float64)
    x = torch.zeros(n, nkv, D, dtype=torch.float64, device="cuda")
    x[..., :half], x[..., half:rot] = r * torch.sin(a), r * torch.cos(a)
    x = x.half()
    v = torch.randn(n, nkv, D, generator=g, device="cuda").half()
    kv = empty_cache(4, 1, n // 16, 16, nkv, D, "fp16", [n])
    b2.paged_kv_append(kv, x[None], v[None], rope=b2.Rope(rot, inv_freq=freq),
                       positions=torch.tensor([at], dtype=torch.int32, device="cuda"))
    x1, x2 = x[..., :half].double(), x[..., half:rot].double()
    want = torch.cat((x1 * torch.cos(a) - x2 * torch.sin(a), x2 * torch.cos(a) + x1 * torch.sin(a), x[..., rot:].double()), -1)
    k, vv = (y[kv.block_tables[0].long()].reshape(n, nkv, D) for y in R.pool_rows(kv.pool, D))
    assert want[..., :min(half, 32)].abs().max() < 2.0 ** -9
    assert torch.equal(k, R.held(want)), int((k != R.held(want)).sum())
    assert torch.equal(vv, R.held(v.double()))
