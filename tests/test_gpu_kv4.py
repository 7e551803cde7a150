"""Attention over a 4-bit paged cache, and over listed blocks of either kind of
cache, on the GPU against 64-bit references (kv4_ref.py).

Bounds.  With u half a step of the output's type: the output's own rounding, u
|o| (2^-25 below half's normal range).  A logit is a sum of D products of exact
operands in 32 bits: at most 32 additions along the way (16 products of 16
terms, the groups, the minima), each off by at most 2^-23 of the largest partial
sum, which is below M = sum_d |q_d| 3 max|k| / sqrt(D), since m and 15 s of a
group are each at most 3 max|k| together: 2^-18 M.  That changes every weight by
that relative amount and their sum likewise, 2^-17 M A with A = sum_j p_j |v_j|;
the exponential and the split of the weights add less than 2^-20 A; for outputs
in bf16 the weights are rounded to halves instead, 2^-11 of each weight times its
scale at most, which moves an output by 2^-11 sum_j p_j |v_j - mid_j| <= 2^-11 A'
with A' below 3 max|v| / 2 (a group's codes less 8 times its scale are at most half
its range, |m| + 15 s <= 3 max|v|).  Outputs add
up 16 positions at a time, n / 16 + 64 additions (the joins among them) off by at
most 2^-23 of 3 max|v|."""
import math

import pytest
import torch

import b2engine as b2
import kv4_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def close(got, want, mag, q, k, v, n):
    """k, v: the row pools in 64 bits (NaN where nothing was written)."""
    fin = lambda x: x[torch.isfinite(x)].abs().max().item() if torch.isfinite(x).any() else 0.0  # noqa: E731
    u = torch.finfo(got.dtype).eps / 2
    M = q.double().abs().sum(-1, keepdim=True) * 3 * fin(k) / math.sqrt(q.shape[-1])
    half = 2.0 ** -11 * 1.5 * fin(v) if got.dtype == torch.bfloat16 else 0.0
    tol = u * want.abs() + half + (2.0 ** -17 * M + 2.0 ** -20) * mag + (n / 16 + 64) * 2.0 ** -23 * 3 * fin(v) + 2.0 ** -25
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (int((err > tol).sum()), float((err - tol).max()), (err > tol).nonzero()[0].tolist())


def make(seed, lens, nq, nkv, D, bs, dt, mb=None, extra=3, scale=1.0):
    """A cache whose rows past a sequence's end were never written (bytes 0xff: NaN scales), its rows in 64 bits."""
    g = gen(seed)
    B = len(lens)
    mb = mb or max(1, -(-max(lens) // bs))
    nb = B * mb + extra
    k = torch.randn(nb, bs, nkv, D, generator=g, device="cuda")
    v = torch.randn(nb, bs, nkv, D, generator=g, device="cuda") * scale
    pool = R.fill_pool(k, v)
    tables = torch.randperm(nb, generator=g, device="cuda")[: B * mb].to(torch.int32).view(B, mb)
    written = torch.zeros(nb, bs, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        pos = torch.arange(min(n, mb * bs), device="cuda")
        written[tables[b].long()[pos // bs], pos % bs] = True
    for blk, slot in (~written).nonzero().tolist():
        p = slot % 16
        tile = pool[blk, :, slot // 16]
        for value in (0, 1):
            for gr in range(-(-R.padded(D) // 64)):
                at = R.scale_place(D, p, gr, value)
                tile[:, at:at + 4] = 255
    q = torch.randn(B, nq, D, generator=g, device="cuda").to(DT[dt])
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return q, b2.PagedKV4(pool, tables, sl, D, DT[dt]), *R.pool_rows(pool, D)


def ws_for(kv, nq):
    return b2.Workspace(b2.paged_decode_workspace_bytes(kv.batch, nq, kv.nkv, kv.head_dim,
                                                        kv.block_tables.shape[1] * kv.block_size))


CASES = [
    # lens, nq, nkv, D, bs, dtype, window, sinks
    ([1], 1, 1, 64, 16, "fp16", 0, 0),
    ([0, 1, 15, 16, 17], 4, 2, 64, 16, "bf16", 0, 0),
    ([301], 14, 2, 64, 16, "fp16", 0, 0),
    ([700, 33, 129], 32, 8, 128, 16, "fp16", 0, 0),
    ([700, 33, 129], 32, 8, 128, 32, "bf16", 0, 0),
    ([1000, 77], 64, 8, 128, 64, "fp16", 0, 0),
    ([500, 500], 16, 1, 128, 16, "bf16", 0, 0),
    ([300], 17, 1, 128, 16, "fp16", 0, 0),
    ([300], 40, 1, 64, 16, "fp16", 0, 0),
    ([257, 90], 9, 3, 80, 16, "fp16", 0, 0),
    ([257, 90], 8, 1, 96, 48, "bf16", 0, 0),
    ([130, 31], 10, 2, 72, 16, "bf16", 0, 0),
    ([64, 65], 3, 3, 8, 16, "fp16", 0, 0),
    ([400, 9], 8, 4, 256, 16, "fp16", 0, 0),
    ([400, 9], 24, 2, 256, 32, "bf16", 0, 0),
    ([200, 200], 6, 2, 136, 16, "fp16", 0, 0),
    ([200, 100], 4, 1, 192, 16, "bf16", 0, 0),
    ([700, 33, 129], 32, 8, 128, 16, "fp16", 64, 4),
    ([700, 33, 129], 14, 2, 64, 16, "bf16", 33, 133),
    ([700, 1], 8, 8, 64, 16, "fp16", 1, 0),
    ([700, 5], 8, 8, 64, 16, "fp16", 100, 600),
    ([5] * 40 + [300], 8, 2, 64, 16, "fp16", 0, 0),
    ([20] * 150, 4, 4, 64, 16, "bf16", 0, 0),
]


@pytest.mark.parametrize("lens,nq,nkv,D,bs,dt,window,sinks", CASES)
@pytest.mark.parametrize("split", [True, False])
def test_decode(cuda, lens, nq, nkv, D, bs, dt, window, sinks, split):
    q, kv, k, v = make(1, lens, nq, nkv, D, bs, dt)
    out = torch.full_like(q, 7.0)
    ws = ws_for(kv, nq) if split else None
    assert b2.paged_decode_gqa(q, kv, out, window=window, sinks=sinks, ws=ws) is out
    want, mag = R.decode(q, k, v, kv.block_tables, lens, window, sinks)
    close(out, want, mag, q, k, v, max(lens))
    again = torch.empty_like(out)
    b2.paged_decode_gqa(q, kv, again, window=window, sinks=sinks, ws=ws)
    assert torch.equal(out, again)  # the same bits every run, and counters left as they were found


def test_many_pieces(cuda):
    """A few long sequences, cut into one piece per CTA, and an uneven batch, cut anywhere."""
    for seed, lens in ((2, [9000]), (3, [4000, 100, 7001, 16, 0, 333])):
        q, kv, k, v = make(seed, lens, 8, 2, 128, 16, "bf16")
        out = torch.empty_like(q)
        b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, 8))
        want, mag = R.decode(q, k, v, kv.block_tables, lens)
        close(out, want, mag, q, k, v, max(lens))


def test_lengths_past_the_table_and_below_zero(cuda):
    q, kv, k, v = make(4, [64, 64], 4, 2, 64, 16, "fp16")
    kv.seq_lens.copy_(torch.tensor([1000, -3]))
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, 4))
    want, mag = R.decode(q, k, v, kv.block_tables, [64, 0])
    close(out, want, mag, q, k, v, 64)
    assert out[1].abs().max() == 0


def test_table_entries_that_are_none(cuda):
    q, kv, k, v = make(5, [90, 90], 8, 2, 64, 16, "fp16")
    kv.block_tables[0, 1] = -1
    kv.block_tables[0, 4] = kv.num_blocks
    kv.block_tables[1] = 2 ** 31 - 1
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, 8))
    want, mag = R.decode(q, k, v, kv.block_tables, [90, 90])
    close(out, want, mag, q, k, v, 90)
    assert out[1].abs().max() == 0


def test_views(cuda):
    """q out of a fused projection, blocks further apart than they are long."""
    q, kv, k, v = make(6, [90, 40], 8, 2, 64, 16, "bf16")
    wide = torch.randn(2, 20, 64, device="cuda").bfloat16()
    wide[:, 4:12] = q
    far = torch.zeros(kv.num_blocks, 3, *kv.pool.shape[1:], dtype=torch.uint8, device="cuda")
    far[:, 1] = kv.pool
    kv2 = b2.PagedKV4(far[:, 1], kv.block_tables, kv.seq_lens, 64, torch.bfloat16)
    a, b = torch.empty_like(q), torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, a, ws=ws_for(kv, 8))
    b2.paged_decode_gqa(wide[:, 4:12], kv2, b, ws=ws_for(kv, 8))
    assert torch.equal(a, b)
    want, mag = R.decode(q, k, v, kv.block_tables, [90, 40])
    close(a, want, mag, q, k, v, 90)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 300.0, 60000.0])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_sizes_of_queries(cuda, size, dt):
    """Queries of any size (so many orders that scaling them is seen): small ones average, large ones pick one row."""
    q, kv, k, v = make(7, [200], 8, 2, 64, 16, dt)
    q = (q.double().clamp(-1, 1) * size).to(DT[dt])
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, 8))
    want, mag = R.decode(q, k, v, kv.block_tables, [200])
    assert torch.isfinite(out).all()
    if size < 1:
        close(out, want, mag, q, k, v, 200)
    else:
        # a logit is off by up to 2^-18 M, past 1 here: what the softmax picks from must lie within that of the largest
        z = torch.einsum("bhd,nhd->bhn", q.double(), k[kv.block_tables[0].long()].flatten(0, 1)[:200]
                         .repeat_interleave(4, 1)) / 8
        M = q.double().abs().sum(-1) * 3 * k[torch.isfinite(k)].abs().max() / 8 * 2.0 ** -17
        near = z >= z.amax(-1, keepdim=True) - M[..., None] - 20
        vv = v[kv.block_tables[0].long()].flatten(0, 1)[:200].repeat_interleave(4, 1)
        lo = torch.where(near.transpose(1, 2)[..., None], vv[None], math.inf).amin(1)
        hi = torch.where(near.transpose(1, 2)[..., None], vv[None], -math.inf).amax(1)
        slack = 2.0 ** -7 * vv.abs().max()
        assert (out.double() >= lo - slack).all() and (out.double() <= hi + slack).all()


def test_values_of_very_different_sizes(cuda):
    """Scales of V that grow and shrink by orders of magnitude from tile to tile."""
    g = gen(8)
    nb, bs, nkv, D = 40, 16, 2, 128
    k = torch.randn(nb, bs, nkv, D, generator=g, device="cuda")
    v = torch.randn(nb, bs, nkv, D, generator=g, device="cuda")
    order = torch.randperm(nb, generator=g, device="cuda")
    v *= (2.0 ** (order.float() / 2 - 12))[:, None, None, None]
    pool = R.fill_pool(k, v)
    k, v = R.pool_rows(pool, D)
    kv = b2.PagedKV4(pool, torch.arange(nb, dtype=torch.int32, device="cuda")[None],
                     torch.tensor([nb * bs], dtype=torch.int32, device="cuda"), D, torch.float16)
    q = torch.randn(1, 8, D, generator=g, device="cuda").half()
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, 8))
    want, mag = R.decode(q, k, v, kv.block_tables, [nb * bs])
    # relative to A alone: what a row adds is held to its own size
    err = (out.double() - want).abs()
    assert (err <= 2.0 ** -11 * want.abs() + 2.0 ** -10 * mag * 0.1 + 2.0 ** -25).all()


def test_one_row_outweighs_many(cuda):
    """Weights far below the largest one add up: 8000 rows e^-17 each beside a row of weight 1, with values 2^10 times
    its own."""
    D, bs, nb = 64, 16, 500
    k = torch.zeros(nb, bs, 1, D, device="cuda")
    k[0, 0, 0, :] = 1.0
    v = torch.full((nb, bs, 1, D), 1024.0, device="cuda") + torch.arange(D, device="cuda") / 64
    v[0, 0] = torch.arange(D, device="cuda") / 64
    pool = R.fill_pool(k, v)
    k, v = R.pool_rows(pool, D)
    kv = b2.PagedKV4(pool, torch.arange(nb, dtype=torch.int32, device="cuda")[None],
                     torch.tensor([nb * bs], dtype=torch.int32, device="cuda"), D, torch.float16)
    q = torch.full((1, 4, D), 17.0 / 8, device="cuda").half()
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, 4))
    want, mag = R.decode(q, k, v, kv.block_tables, [nb * bs])
    assert want.max() < 1.5 and want.min() > 0.3
    assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -12 * mag).all()


def test_nan_shows_where_it_is(cuda):
    """A group of V without a number: its channels of that head's outputs; a row of K: all of that head's."""
    q, kv, k, v = make(9, [90], 8, 2, 128, 16, "bf16")
    clean = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, clean, ws=ws_for(kv, 8))
    blk = int(kv.block_tables[0, 2])
    at = R.scale_place(128, 5, 1, 1)
    kv.pool[blk, 1, 0, at:at + 4] = 255
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, 8))
    assert torch.equal(out[0, :4], clean[0, :4]) and torch.isnan(out[0, 4:, 64:]).all()
    assert torch.isfinite(out[0, 4:, :64]).all()
    at = R.scale_place(128, 5, 0, 0)
    kv.pool[blk, 0, 0, at:at + 4] = 255
    b2.paged_decode_gqa(q, kv, out, ws=ws_for(kv, 8))
    assert torch.isnan(out[0, :4]).all()


def make16(seed, lens, nq, nkv, D, bs, dt, layout="slot"):
    g = gen(seed)
    B, mb = len(lens), max(1, -(-max(lens) // bs))
    shape = (B * mb, bs, nkv, D) if layout == "slot" else (B * mb, nkv, bs, D)
    k, v = (torch.randn(shape, generator=g, device="cuda").to(DT[dt]) for _ in "kv")
    if layout == "head":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    tables = torch.randperm(B * mb, generator=g, device="cuda").to(torch.int32).view(B, mb)
    for b, n in enumerate(lens):
        for pos in range(n, mb * bs):
            k[int(tables[b, pos // bs]), pos % bs] = math.nan
            v[int(tables[b, pos // bs]), pos % bs] = math.nan
    q = torch.randn(B, nq, D, generator=g, device="cuda").to(DT[dt])
    kv = b2.PagedKV(k, v, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return q, kv, k.double(), v.double()


LISTS = [([700, 33, 129], 32, 8, 128, 16, "fp16"), ([300], 14, 2, 64, 16, "bf16"), ([257, 90], 9, 3, 80, 16, "fp16"),
         ([500, 20], 16, 1, 128, 32, "bf16"), ([400, 0], 8, 4, 256, 64, "fp16"), ([40] * 35, 4, 2, 64, 16, "fp16")]


def lists(seed, lens, nkv, mb, n):
    """Blocks in any order, some none, some past the end, some twice."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-2, mb + 2, (len(lens), nkv, n), generator=g, dtype=torch.int32)
    x[0, 0, -1] = 2 ** 31 - 1
    if n > 2:
        x[0, :, 1] = x[0, :, 0]
        x[-1, -1] = -1
    return x


@pytest.mark.parametrize("lens,nq,nkv,D,bs,dt", LISTS)
@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("bits", [4, 16])
def test_listed_blocks(cuda, lens, nq, nkv, D, bs, dt, n, bits):
    q, kv, k, v = (make if bits == 4 else make16)(10, lens, nq, nkv, D, bs, dt)
    blocks = lists(n, lens, nkv, kv.block_tables.shape[1], n)
    for split in (True, False):
        out = torch.empty_like(q)
        b2.paged_decode_gqa(q, kv, out, blocks=blocks.cuda(), ws=ws_for(kv, nq) if split else None)
        want, mag = R.decode(q, k, v, kv.block_tables, lens, blocks=blocks)
        close(out, want, mag, q, k, v, n * bs)


@pytest.mark.parametrize("bs", [1, 3, 8, 24])
def test_listed_blocks_of_any_size(cuda, bs):
    """A 16-bit cache's blocks need not hold whole groups of 16 positions."""
    lens = [100, 17]
    q, kv, k, v = make16(11, lens, 8, 2, 64, bs, "fp16", layout="head")
    blocks = lists(4, lens, 2, kv.block_tables.shape[1], 9)
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, blocks=blocks.cuda(), ws=ws_for(kv, 8))
    want, mag = R.decode(q, k, v, kv.block_tables, lens, blocks=blocks)
    close(out, want, mag, q, k, v, 9 * bs)


@pytest.mark.parametrize("bits", [4, 16])
def test_lists_longer_than_the_sequences(cuda, bits):
    """As many entries as a sequence has blocks are looked at: what stands behind them is padding, whatever it says."""
    lens = [1, 16, 17, 0, 400]
    q, kv, k, v = (make if bits == 4 else make16)(13, lens, 8, 2, 64, 16, "bf16")
    blocks = torch.arange(60, dtype=torch.int32).expand(5, 2, 60).contiguous() % 25
    outs = []
    for x in (blocks, torch.where(torch.arange(60) < torch.tensor([1, 1, 2, 0, 25])[:, None, None], blocks, -1)):
        outs.append(torch.empty_like(q))
        b2.paged_decode_gqa(q, kv, outs[-1], blocks=x.cuda(), ws=ws_for(kv, 8))
    want, mag = R.decode(q, k, v, kv.block_tables, lens)
    close(outs[0], want, mag, q, k, v, 400)
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("bits", [4, 16])
def test_all_blocks_listed_is_the_whole_cache(cuda, bits):
    q, kv, k, v = (make if bits == 4 else make16)(12, [333, 60], 8, 2, 128, 16, "bf16")
    mb = kv.block_tables.shape[1]
    a, b = torch.empty_like(q), torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, a, ws=ws_for(kv, 8))
    b2.paged_decode_gqa(q, kv, b, ws=ws_for(kv, 8),
                        blocks=torch.arange(mb, dtype=torch.int32, device="cuda").expand(2, 2, mb).contiguous())
    assert torch.equal(a, b)


def test_refusals_of_the_binding(cuda):
    q, kv, _, _ = make(13, [40], 8, 2, 64, 16, "fp16")
    out = torch.empty_like(q)
    blocks = torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda")
    for more in (dict(window=4), dict(sinks=1), dict(scores=torch.zeros(1, device="cuda"))):
        with pytest.raises(ValueError):
            b2.paged_decode_gqa(q, kv, out, blocks=blocks, **more)
    for bad in (blocks.long(), blocks[:, :1], blocks.cpu(), blocks.transpose(0, 1)[:1].expand(1, 2, 3)[..., ::2]):
        with pytest.raises(ValueError):
            b2.paged_decode_gqa(q, kv, out, blocks=bad)
    with pytest.raises(ValueError):
        b2.paged_decode_gqa(q, kv, out, scores=torch.zeros(kv.num_blocks, 2, 16, device="cuda"))
    with pytest.raises(ValueError):
        b2.paged_decode_gqa(q.bfloat16(), kv, out.bfloat16())
    with pytest.raises(b2.B2Error) as e:
        b2.paged_decode_gqa(q, kv, out, ws=b2.Workspace(16))
    assert e.value.status == -3


def test_captured_with_new_lengths(cuda):
    """Lengths, tables and lists are read on the device: a graph follows them."""
    q, kv, k, v = make(14, [200, 100], 8, 2, 64, 16, "fp16", mb=13)
    ws, out = ws_for(kv, 8), torch.empty_like(q)
    blocks = torch.zeros(2, 2, 4, dtype=torch.int32, device="cuda")
    few = torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, out, ws=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b2.paged_decode_gqa(q, kv, out, ws=ws)
        b2.paged_decode_gqa(q, kv, few, blocks=blocks, ws=ws)
    for lens, first in (([200, 100], 0), ([17, 1], 0), ([0, 99], 3)):
        kv.seq_lens.copy_(torch.tensor(lens))
        blocks.copy_(torch.arange(first, first + 4).expand(2, 2, 4))
        g.replay()
        want, mag = R.decode(q, k, v, kv.block_tables, lens)
        close(out, want, mag, q, k, v, 200)
        want, mag = R.decode(q, k, v, kv.block_tables, lens, blocks=blocks.cpu())
        close(few, want, mag, q, k, v, 64)


def test_two_streams_with_a_workspace_each(cuda):
    jobs = [make(15 + i, [3000, 50], 8, 2, 128, 16, "bf16") for i in range(2)]
    streams = [torch.cuda.Stream() for _ in jobs]
    spaces, outs = [ws_for(j[1], 8) for j in jobs], [torch.empty_like(j[0]) for j in jobs]
    torch.cuda.synchronize()
    for _ in range(20):
        for j, s, w, o in zip(jobs, streams, spaces, outs):
            b2.paged_decode_gqa(j[0], j[1], o, ws=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for (q, kv, k, v), o in zip(jobs, outs):
        want, mag = R.decode(q, k, v, kv.block_tables, [3000, 50])
        close(o, want, mag, q, k, v, 3000)


def test_pool_past_32_bits(cuda):
    """Blocks that lie more than 2^32 bytes into the pool (and 2^31 elements, of a 16-bit one)."""
    D, nkv, bs = 64, 1, 16
    q, kv, k, v = make(17, [40], 4, nkv, D, bs, "fp16")
    block = kv.pool[0].numel()
    far = -(-(2 ** 32 + 2 ** 20) // block)
    big = torch.empty(far + kv.num_blocks, *kv.pool.shape[1:], dtype=torch.uint8, device="cuda")
    big[far:] = kv.pool
    kv2 = b2.PagedKV4(big, kv.block_tables + far, kv.seq_lens, D, torch.float16)
    a, b = torch.empty_like(q), torch.empty_like(q)
    b2.paged_decode_gqa(q, kv, a, ws=ws_for(kv, 4))
    b2.paged_decode_gqa(q, kv2, b, ws=ws_for(kv, 4))
    assert torch.equal(a, b)
    want, mag = R.decode(q, k, v, kv.block_tables, [40])
    close(a, want, mag, q, k, v, 40)
