"""Attention over a 4-bit paged cache whose work is cut between CTAs: several units
in a piece, segments cut in the middle of a CTA's share, several segments in one
share, more units than are looked up at a time, and the same over long lists.

Values tell where a row is: channel c of a row is 1 in the tiles of 16 positions
whose number is c modulo the channels, else 0, so an output is the share of the
weight that its tiles have, and a tile that is left out or taken twice moves it by a
large part of itself.  Bound: half a step of the type, 2^-17 M of every weight as in
test_gpu_kv4.py (M = sum |q| 3 max|k| / sqrt(D)) and 2^-18 for the exponential and
the split of the weights, of the output.  Beside those, as codes' sums start at up to
-8 of all weights, with a scale of 1 / 15: a unit's 16 products off by 2^-22 of 31 / 15
of its weight; and of all weights so far, times 16 / 15, 2^-24 in each of 9
additions a unit (one of the outputs, 8 of what is added back) for the n units that
a CTA adds up."""
import math

import pytest
import torch

import b2engine as b2
import kv4_ref as R
from test_gpu_kv4 import DT, ws_for

pytestmark = pytest.mark.gpu


def marked(seed, lens, nq, nkv, D, bs, dt):
    """Keys at random, values that tell the tile; rows past a sequence's end hold NaN scales."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, mb = len(lens), max(1, -(-max(lens) // bs))
    tables = torch.randperm(B * mb, generator=g, device="cuda").to(torch.int32).view(B, mb)
    k = torch.randn(B * mb, bs, nkv, D, generator=g, device="cuda") / 2
    v = torch.zeros(B, mb * bs, nkv, D, device="cuda")
    pos = torch.arange(mb * bs, device="cuda")
    v[:, pos, :, pos // 16 % D] = 1.0
    # every group of 64 channels spans 0 to 15 / 15, so that the code of a 1 is 15 or the group all 0
    pool = R.fill_pool(k, v.view(B * mb, bs, nkv, D)[torch.argsort(tables.flatten().long())])
    ng = -(-R.padded(D) // 64)
    for b, n in enumerate(lens):
        for blk in range(n // bs, mb):
            tiles = pool[int(tables[b, blk])]
            for p in range(max(0, n - blk * bs), bs):
                for value in (0, 1):
                    at = R.scale_place(D, p % 16, 0, value)
                    tiles[:, p // 16, at:at + 4 * ng] = 255
    q = (torch.randn(B, nq, D, generator=g, device="cuda") * 0.7).to(DT[dt])
    kv = b2.PagedKV4(pool, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), D, DT[dt])
    return q, kv


def shares(q, kv, lens, blocks=None, window=0, sinks=0):
    """The outputs in 64 bits, a sequence at a time; largest |k|."""
    B, nq, D = q.shape
    nkv, bs, G = kv.nkv, kv.block_size, nq // kv.nkv
    out = torch.zeros(B, nq, D, dtype=torch.float64, device="cuda")
    top = 0.0
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k, v = (x.reshape(-1, nkv, D)[:n] for x in R.pool_rows(kv.pool[kv.block_tables[b].long()[:-(-n // bs)]], D))
        top = max(top, float(k.abs().max()))
        z = torch.einsum("hgd,nhd->hgn", q[b].double().view(nkv, G, D), k) / math.sqrt(D)
        pos = torch.arange(n, device="cuda")
        seen = torch.ones(nkv, n, dtype=torch.bool, device="cuda")
        if window:
            seen &= (pos < sinks) | (pos >= n - window)
        if blocks is not None:
            listed = torch.zeros(nkv, kv.block_tables.shape[1], dtype=torch.bool, device="cuda")
            seen = listed.scatter(1, blocks[b].long(), True)[:, pos // bs]
        p = torch.softmax(z.masked_fill(~seen[:, None], -math.inf), -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(nq, D)
    return out, top


def check(out, want, top, q, run, tile=None):
    """run: most units that a CTA adds up; tile: what a tile's share of an output is at least."""
    u = torch.finfo(out.dtype).eps / 2
    M = q.double().abs().sum(-1, keepdim=True) * 3 * top / math.sqrt(q.shape[-1])
    seen = (want.amax(-1, keepdim=True) > 0).double()
    tol = (u + 2.0 ** -18 + 2.0 ** -17 * M) * want + (16 * 2.0 ** -22 * 31 + 9 * run * 2.0 ** -24 * 16) / 15 * seen
    tol += 2.0 ** -25
    err = (out.double() - want).abs()
    assert (err <= tol).all(), (int((err > tol).sum()), (err > tol).nonzero()[0].tolist(), float((err / tol).max()))
    if tile:  # a tile that is missing would be seen
        whole = want > want.amax(-1, keepdim=True) / 2
        assert float((tol / want)[whole].max()) < tile / 2


def units(n, D, G):
    """Units of a segment of n positions, as the kernel cuts them, and the CTAs that share all of them."""
    wide = 256 if D <= 128 and G <= 8 else 128
    return max(1, -(-n // wide)), 2 * torch.cuda.get_device_properties(0).multi_processor_count


LONG = [
    # lens, nq, nkv, D, bs, dtype
    ([40001], 32, 8, 128, 16, "bf16"),
    ([40001], 64, 8, 128, 64, "fp16"),
    ([20011], 128, 8, 128, 16, "bf16"),
    ([131001], 32, 8, 64, 64, "fp16"),
    ([15000], 64, 16, 256, 32, "bf16"),
    ([9000, 100, 16000, 16, 0, 333], 32, 8, 128, 16, "fp16"),
    ([1000 + 97 * i for i in range(20)], 64, 16, 128, 16, "bf16"),
    ([700 + 61 * i for i in range(20)], 128, 16, 64, 16, "fp16"),
    ([1000 + 97 * i for i in range(20)], 16, 16, 256, 16, "fp16"),
    ([300 + 83 * (i * 7 % 40) for i in range(40)], 32, 8, 128, 16, "fp16"),
    ([4000 + 83 * (i * 7 % 40) for i in range(40)], 16, 4, 128, 16, "bf16"),
    ([5 + 40 * i for i in range(150)], 16, 2, 64, 32, "fp16"),
    ([5 + 40 * i for i in range(150)], 8, 4, 96, 32, "bf16"),
]


def in_a_row(lens, nq, nkv, D, split):
    """Most units that a CTA adds up: of equal pieces up to an eighth or two above the even share; or a whole segment."""
    each, grid = zip(*(units(n, D, nq // nkv) for n in lens))
    if not split:
        return max(each)
    even = -(-sum(each) * nkv * -(-(nq // nkv) // 16) // grid[0])
    assert even > 1  # more than a unit for most CTAs
    return min(max(each), even + max(2, even // 8))


@pytest.mark.parametrize("lens,nq,nkv,D,bs,dt", LONG)
def test_cut_anywhere(cuda, lens, nq, nkv, D, bs, dt):
    q, kv = marked(1, lens, nq, nkv, D, bs, dt)
    want, top = shares(q, kv, lens)
    for split in (True, False):
        ws, out = ws_for(kv, nq) if split else None, torch.full_like(q, 7.0)
        for _ in range(2):
            b2.paged_decode_gqa(q, kv, out, ws=ws)
        check(out, want, top, q, in_a_row(lens, nq, nkv, D, split), 1 / (max(lens) // 16 // D + 2) if split else None)


@pytest.mark.parametrize("lens,nq,nkv,D,bs,dt", LONG[:2] + LONG[5:8])
def test_windows_cut_anywhere(cuda, lens, nq, nkv, D, bs, dt):
    q, kv = marked(2, lens, nq, nkv, D, bs, dt)
    window, sinks = max(lens) - 300, 133
    want, top = shares(q, kv, lens, window=window, sinks=sinks)
    out = torch.full_like(q, 7.0)
    b2.paged_decode_gqa(q, kv, out, window=window, sinks=sinks, ws=ws_for(kv, nq))
    check(out, want, top, q, in_a_row(lens, nq, nkv, D, True) + 1, 1 / (max(lens) // 16 // D + 2))


@pytest.mark.parametrize("lens,nq,nkv,D,bs,dt,n", [
    ([30000, 9000], 32, 8, 128, 16, "bf16", 1500),
    ([30000, 30000], 64, 8, 128, 32, "fp16", 900),
    ([6000 + 200 * (i * 11 % 40) for i in range(40)], 32, 8, 128, 16, "fp16", 200),
])
def test_long_lists(cuda, lens, nq, nkv, D, bs, dt, n):
    """More entries than sequences have blocks, too: as many are looked at as there are blocks."""
    q, kv = marked(3, lens, nq, nkv, D, bs, dt)
    g = torch.Generator().manual_seed(4)
    blocks = torch.zeros(len(lens), nkv, n, dtype=torch.int32)  # (padding behind all of a sequence's blocks is not looked at)
    for b, L in enumerate(lens):
        for h in range(nkv):
            pick = torch.randperm(-(-L // bs), generator=g)[:n]
            blocks[b, h, :len(pick)] = pick.int()
    blocks = blocks.cuda()
    want, top = shares(q, kv, lens, blocks=blocks)
    seen = [min(n, -(-L // bs)) * bs for L in lens]
    for split in (True, False):
        out = torch.full_like(q, 7.0)
        b2.paged_decode_gqa(q, kv, out, blocks=blocks, ws=ws_for(kv, nq) if split else None)
        check(out, want, top, q, in_a_row(seen, nq, nkv, D, split), 0.1 if split else None)
