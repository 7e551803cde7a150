"""Attention over a 4-bit paged cache does not round its weights to 16 bits, for
outputs of either type.

A weight rounded to a half (half a step: 2^-11 of it) meets the codes, its 32-bit
value the rest of the row and the sum of the weights: of a row whose m + u s
vanishes 2^-11 of a few s would be left.  Kept as a half and its remainder it is
off by 2^-22."""
import math

import pytest
import torch

import b2engine as b2
import kv4_ref as R
from test_gpu_kv4 import DT, ws_for
from test_gpu_kv4_split import shares

pytestmark = pytest.mark.gpu


def worst_rounded(heads, dtype, by):
    """Numbers a of the type for which p = exp(-a by), as a half, is off by most of half a step of it."""
    a = (torch.arange(1, 400, dtype=torch.float64) / 256).to(dtype).unique()
    p = torch.exp(-a.double() * by)
    off = ((p.half().double() - p) / p).abs() * (p > 0.1)
    best = off.argsort(descending=True)[:heads]
    assert off[best].min() > 2.0 ** -12
    return a[best]


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", [4, 8, 16])
def test_rows_that_vanish(cuda, dt, D, heads):
    """64 positions, the first of weight 1 and the others of p each; values 0 and 15, so s = 1, and on the channels of
    zeros the rest of the row takes back the 4 or more of its weight that a code's product has too little.  Weights as
    halves leave 2^-12 of that, times the share of the first warp's others, a half or more: 5e-4 and up.  Allowed: 40
    additions (4 tiles of products with the constant and with the codes, of halves and of remainders, the lanes', the
    warps', the groups') off by at most 2^-22 of the largest partial sum, 31 (15, and up to 8 less and back), and 2^-22
    of 8 for the remainder."""
    n, bs = 64, 16
    k, v = (torch.zeros(n // bs, bs, 1, D, device="cuda") for _ in "kv")
    k[0, 0, 0, 0] = 15.0
    v[..., 1::2] = 15.0
    pool = R.fill_pool(k, v)
    kr, vr = R.pool_rows(pool, D)
    assert torch.equal(vr, v.double())
    kv = b2.PagedKV4(pool, torch.arange(n // bs, dtype=torch.int32, device="cuda")[None],
                     torch.tensor([n], dtype=torch.int32, device="cuda"), D, DT[dt])
    q = torch.zeros(1, heads, D, dtype=DT[dt], device="cuda")
    q[0, :, 0] = worst_rounded(heads, DT[dt], 15 / math.sqrt(D)).cuda()
    out = torch.full_like(q, 7.0)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, heads))
    want, _ = R.decode(q, kr, vr, kv.block_tables, [n])
    tol = torch.finfo(DT[dt]).eps / 2 * want.abs() + 40 * 2.0 ** -22 * 31 + 2.0 ** -22 * 8
    err = (out.double() - want).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float(err[..., ::2].max()))


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("heads", [4, 8, 16])
def test_values_of_very_different_sizes(cuda, dt, heads):
    """Scales of V that grow and shrink by 2^20 from tile to tile, with rows that vanish in every second channel: what is
    left there is held to 40 additions and 40 more that join units, off by 2^-22 of the largest partial sum (31 / 15 of
    the largest value), and the remainder's 2^-22 of 8 / 15 of it."""
    g = torch.Generator(device="cuda").manual_seed(3)
    nb, bs, D = 40, 16, 128
    k = torch.randn(nb, bs, 1, D, generator=g, device="cuda")
    order = torch.randperm(nb, generator=g, device="cuda")
    v = torch.zeros(nb, bs, 1, D, device="cuda")
    v[..., 1::2] = 15.0 * (2.0 ** (order // 2 - 12).float())[:, None, None, None]
    pool = R.fill_pool(k, v)
    kr, vr = R.pool_rows(pool, D)
    assert torch.equal(vr, v.double())
    kv = b2.PagedKV4(pool, torch.arange(nb, dtype=torch.int32, device="cuda")[None],
                     torch.tensor([nb * bs], dtype=torch.int32, device="cuda"), D, DT[dt])
    q = (torch.randn(1, heads, D, generator=g, device="cuda") / 4).to(DT[dt])
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, heads))
    want, mag = R.decode(q, kr, vr, kv.block_tables, [nb * bs])
    top = float(v.max())
    zeros, rest = (out.double() - want).abs()[..., ::2], (out.double() - want).abs()[..., 1::2]
    assert zeros.max() <= 80 * 2.0 ** -22 * top * 31 / 15 + 2.0 ** -22 * top * 8 / 15
    # the others add up rows of one sign: the rounding of the output, and 2^-17 M of every weight (M: what the logits'
    # partial sums may reach, sum |q| 3 max|k| / sqrt(D)), as in the other tests of this kernel
    M = q.double().abs().sum(-1, keepdim=True) * 3 * kr.abs().max() / math.sqrt(D)
    tol = torch.finfo(DT[dt]).eps / 2 * want.abs() + 2.0 ** -17 * M * mag + 80 * 2.0 ** -22 * top * 31 / 15
    assert (rest <= tol[..., 1::2]).all()


@pytest.mark.parametrize("heads", [4, 8])
def test_long_contexts_are_rounded_once(cuda, heads):
    """131001 tokens, whose output is 1 / 200 of the values: what the sums lose on the way stays below a quarter of what
    the output's own rounding to a half does, root mean square, so together they are off by at most sqrt(1 + 1 / 16) of
    it."""
    g = torch.Generator(device="cuda").manual_seed(11)
    L, bs, D, nkv = 131001, 64, 128, 2
    nb = -(-L // bs)
    k, v = (torch.randn(nb, bs, nkv, D, generator=g, device="cuda") for _ in "kv")
    kv = b2.PagedKV4(R.fill_pool(k, v), torch.arange(nb, dtype=torch.int32, device="cuda")[None],
                     torch.tensor([L], dtype=torch.int32, device="cuda"), D, torch.float16)
    q = torch.randn(1, nkv * heads, D, generator=g, device="cuda").half()
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, nkv * heads))
    want, _ = shares(q, kv, [L])
    once = (want.half().double() - want).square().mean().sqrt()
    assert (out.double() - want).square().mean().sqrt() <= math.sqrt(1 + 1 / 16) * once
