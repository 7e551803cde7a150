"""The paged append, with rotation, into caches of 16-bit and of 4-bit rows, and
rows of a 4-bit cache read back, on the GPU against 64-bit references
(kv4_ref.py).

Bounds.  16-bit rows: half a step of the type, u |x|, and the sine and cosine in
32 bits, off by less than 2^-22 each (the angle as turns in 64 bits, rounded to
32: 2^-25 of pi; the functions: 2^-23), with the products' roundings 2^-21 (|x1|
+ |x2|).  4-bit rows hold exactly what the reference holds.  Rows read back: one
rounding of m + u s to 32 bits (u s is exact there) and one to 16: u (1 + 2^-12)
|x| + 2^-25."""
import math

import pytest
import torch

import b2engine as b2
import kv4_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def empty_cache(bits, B, mb, bs, nkv, D, dt, lens, seed=0, extra=2):
    """A cache of anything, its tables in random order."""
    g = gen(seed)
    nb = B * mb + extra
    tables = torch.randperm(nb, generator=g, device="cuda")[: B * mb].to(torch.int32).view(B, mb)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if bits == 4:
        pool = torch.randint(0, 256, (nb, nkv, bs // 16, R.tile_bytes(D)), generator=g, device="cuda", dtype=torch.uint8)
        return b2.PagedKV4(pool, tables, sl, D, DT[dt])
    k = torch.randn(nb, bs, nkv, D, generator=g, device="cuda").to(DT[dt])
    return b2.PagedKV(k, torch.randn(nb, bs, nkv, D, generator=g, device="cuda").to(DT[dt]), tables, sl)


def rounded(got, want, x, rot):
    """got against want in 64 bits; x: what was rotated, of want's shape."""
    u = torch.finfo(got.dtype).eps / 2
    a = x.double().abs()
    both = torch.cat((a[..., :rot // 2] + a[..., rot // 2:rot],) * 2 + (0 * a[..., rot:],), -1)
    tol = u * want.abs() + 2.0 ** -21 * both + 2.0 ** -25
    ok = (got.double() - want).abs() <= tol
    assert ok.all(), (~ok).nonzero()[0].tolist()


def check(kv, before, q, k, v, qo, counts=None, positions=None, freq=(), q_before=None):
    """The cache and qo after an append against the reference; everything else as it was."""
    bits = 4 if isinstance(kv, b2.PagedKV4) else 16
    rot, D = 2 * len(freq), kv.head_dim
    want_q, rows = R.append(q, k, v, kv.block_tables.cpu(), kv.seq_lens.tolist(),
                            None if counts is None else counts.tolist(),
                            None if positions is None else positions.tolist(), list(freq), kv.block_size, kv.num_blocks)
    if q is not None:
        B, S = q.shape[:2]
        for b in range(B):
            n = S if counts is None else max(0, min(S, int(counts[b])))
            if n:
                rounded(qo[b, :n], want_q[b, :n], q[b, :n], rot)
            assert torch.equal(qo[b, n:], q_before[b, n:])
    touched = torch.zeros(kv.num_blocks, kv.block_size, dtype=torch.bool, device="cuda")
    for blk, slot, _, _ in rows:
        touched[blk, slot] = True
    if bits == 16:
        for blk, slot, kr, vr in rows:
            assert torch.equal(kv.v[blk, slot].double(), vr)
        if rows:
            at = torch.tensor([r[:2] for r in rows], device="cuda")
            src = torch.cat([k[b, :(k.shape[1] if counts is None else max(0, min(k.shape[1], int(counts[b]))))]
                             for b in range(k.shape[0])])
            if len(src) == len(rows):
                rounded(kv.k[at[:, 0], at[:, 1]], torch.stack([r[2] for r in rows]), src, rot)
            else:
                assert torch.allclose(kv.k[at[:, 0], at[:, 1]].double(), torch.stack([r[2] for r in rows]),
                                      rtol=torch.finfo(kv.dtype).eps, atol=2e-5)
        assert torch.equal(kv.k[~touched], before[0][~touched]) and torch.equal(kv.v[~touched], before[1][~touched])
        return
    ka, va = R.pool_rows(kv.pool, D)
    kb, vb = R.pool_rows(before, D)
    for x, y in ((ka, kb), (va, vb)):
        assert torch.equal(x[~touched].nan_to_num(7e7, 8e8, 9e9), y[~touched].nan_to_num(7e7, 8e8, 9e9))
    if rows:
        at = torch.tensor([r[:2] for r in rows], device="cuda")
        for x, i in ((ka, 2), (va, 3)):
            want = R.held(torch.stack([r[i] for r in rows]))
            got = x[at[:, 0], at[:, 1]]
            assert torch.equal(got.nan_to_num(7e7), want.nan_to_num(7e7)), (got != want).nonzero()[:3].tolist()


def keep(kv):
    return kv.pool.clone() if isinstance(kv, b2.PagedKV4) else (kv.k.clone(), kv.v.clone())


CASES = [
    # B, S, lens, counts, nq, nkv, D, bs, rot, dtype
    (1, 1, [1], None, 14, 2, 64, 16, 64, "fp16"),
    (3, 1, [1, 17, 32], None, 32, 8, 128, 16, 128, "bf16"),
    (2, 40, [40, 43], None, 4, 2, 128, 16, 128, "fp16"),
    (4, 33, [33, 60, 5, 40], [33, 0, 5, 17], 4, 2, 64, 32, 64, "bf16"),
    (2, 50, [50, 60], [50, 49], 3, 1, 80, 16, 80, "fp16"),
    (2, 20, [20, 90], None, 8, 1, 96, 48, 96, "bf16"),
    (2, 20, [20, 30], None, 4, 2, 72, 16, 72, "fp16"),
    (2, 9, [9, 30], None, 4, 4, 256, 16, 256, "bf16"),
    (2, 9, [9, 30], None, 2, 2, 192, 16, 64, "fp16"),
    (2, 9, [9, 30], None, 2, 1, 136, 16, 40, "fp16"),
    (2, 9, [9, 30], None, 2, 2, 8, 16, 8, "bf16"),
    (2, 30, [30, 30], None, 4, 2, 128, 16, 32, "bf16"),
    (1, 300, [300], None, 2, 2, 64, 16, 64, "fp16"),
    (1, 1, [100], None, 40, 5, 64, 128, 64, "fp16"),
    # several tokens in one place: 2, 4 and 8 at a time, the last ones of a sequence fewer
    (3, 301, [301, 400, 301], [301, 150, 1], 3, 2, 64, 16, 64, "bf16"),
    (3, 611, [611, 611, 700], [3, 611, 610], 2, 1, 72, 16, 72, "fp16"),
    (60, 61, [61 + i for i in range(60)], [61 - i for i in range(60)], 5, 2, 128, 16, 128, "bf16"),
    (60, 61, [61 + i for i in range(60)], [i + 1 for i in range(60)], 2, 3, 96, 32, 64, "fp16"),
    (1, 4003, [4003], None, 2, 1, 256, 64, 256, "bf16"),
]


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("B,S,lens,counts,nq,nkv,D,bs,rot,dt", CASES)
def test_append(cuda, bits, B, S, lens, counts, nq, nkv, D, bs, rot, dt):
    g = gen(1)
    kv = empty_cache(bits, B, -(-max(lens) // bs) + 1, bs, nkv, D, dt, lens)
    qkv = torch.randn(B, S, nq + 2 * nkv, D, generator=g, device="cuda").to(DT[dt])
    q, k, v = qkv[:, :, :nq], qkv[:, :, nq:nq + nkv], qkv[:, :, nq + nkv:]
    rope = b2.Rope(rot, theta=10000.0)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    pos = torch.tensor([5 + 100000 * b for b in range(B)], dtype=torch.int32, device="cuda")
    for positions in (None, pos):
        before, out = keep(kv), torch.randn(B, S, nq, D, device="cuda").to(DT[dt])
        q_before = out.clone()
        assert b2.paged_kv_append(kv, k, v, q=q, q_out=out, rope=rope, counts=n, positions=positions) is out
        check(kv, before, q, k, v, out, n, positions, rope.inv_freq, q_before)
    # in place, and without rotation
    before, q2 = keep(kv), q.clone()
    src = qkv.clone()
    b2.paged_kv_append(kv, src[:, :, nq:nq + nkv], src[:, :, nq + nkv:], q=src[:, :, :nq], rope=rope, counts=n)
    check(kv, before, q, k, v, src[:, :, :nq], n, None, rope.inv_freq, q2)
    assert torch.equal(src[:, :, nq:], qkv[:, :, nq:])
    before = keep(kv)
    b2.paged_kv_append(kv, k, v, counts=n)
    check(kv, before, None, k, v, None, n)


@pytest.mark.parametrize("bits", [4, 16])
def test_far_positions(cuda, bits):
    """Angles of positions up to 2^31 are as exact as those of near ones."""
    at = [0, 131071, 2 ** 24 + 1, 2 ** 31 - 9, -5]
    kv = empty_cache(bits, 5, 1, 16, 2, 128, "fp16", [3] * 5)
    q, k, v = (torch.randn(5, 3, 2, 128, generator=gen(2), device="cuda").half() for _ in "qkv")
    pos = torch.tensor(at, dtype=torch.int32, device="cuda")
    rope = b2.Rope(128, theta=500000.0)
    before, out = keep(kv), torch.empty_like(q)
    b2.paged_kv_append(kv, k, v, q=q, q_out=out, rope=rope, positions=pos)
    check(kv, before, q, k, v, out, None, pos, rope.inv_freq, out)


@pytest.mark.parametrize("bits", [4, 16])
def test_rows_that_have_no_place(cuda, bits):
    """Positions below zero and past the table, entries that are none, counts past S and below zero."""
    kv = empty_cache(bits, 5, 2, 16, 2, 64, "bf16", [2, 40, 20, 20, 20])
    kv.block_tables[2, 0], kv.block_tables[2, 1] = -1, kv.num_blocks
    q, k, v = (torch.randn(5, 12, 2, 64, generator=gen(3), device="cuda").bfloat16() for _ in "qkv")
    n = torch.tensor([12, 12, 12, 100, -4], dtype=torch.int32, device="cuda")
    rope = b2.Rope(64)
    before, out = keep(kv), torch.randn_like(q)
    q_before = out.clone()
    b2.paged_kv_append(kv, k, v, q=q, q_out=out, rope=rope, counts=n)
    check(kv, before, q, k, v, out, n, None, rope.inv_freq, q_before)


def test_any_block_size_and_layout_of_16_bit_rows(cuda):
    for bs in (1, 5, 8):
        nb = 30
        k, v = (torch.randn(nb, 2, bs, 64, generator=gen(4), device="cuda").half().transpose(1, 2) for _ in "kv")
        tables = torch.randperm(nb, generator=gen(5), device="cuda")[:24].to(torch.int32).view(2, 12)
        kv = b2.PagedKV(k, v, tables, torch.tensor([12, 7], dtype=torch.int32, device="cuda"))
        before = keep(kv)
        kn, vn = (torch.randn(2, 7, 2, 64, generator=gen(6), device="cuda").half() for _ in "kv")
        b2.paged_kv_append(kv, kn, vn, rope=b2.Rope(64))
        check(kv, before, None, kn, vn, None, None, None, b2.Rope(64).inv_freq)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_odd_values(cuda, dt):
    """Equal numbers, zeros, the smallest and the largest, NaN and infinities, numbers past half's range."""
    x = torch.randn(1, 16, 2, 128, generator=gen(7), device="cuda").to(DT[dt])
    big = torch.finfo(DT[dt]).max
    x[0, 0], x[0, 1], x[0, 2, 0], x[0, 2, 1] = 0, 3.5, 1e-7, -6e-8
    x[0, 3, 0, 7], x[0, 4, 1, 100], x[0, 5, 0, 64] = math.nan, math.inf, -math.inf
    x[0, 6], x[0, 7] = 65504.0 / 2, -65504.0 / 2
    x[0, 8, 0, ::2], x[0, 8, 0, 1::2] = 65504.0, -65504.0
    if dt == "bf16":
        x[0, 9, 0] = big / 2
        x[0, 10, 0, :64] = 1e6
        x[0, 11, 0, ::3] = -3e5
    x[0, 12, 0, 1:] = x[0, 12, 0, 0]
    for turn in (False, True):
        kv = empty_cache(4, 1, 1, 16, 2, 128, dt, [16])
        before = keep(kv)
        rope = b2.Rope(128) if turn else None
        b2.paged_kv_append(kv, x, x, rope=rope)
        if not turn:
            check(kv, before, None, x, x, None)
        else:  # (rotated numbers past a 32-bit one's range are not the cache's matter)
            ka, va = R.pool_rows(kv.pool, 128)
            at = int(kv.block_tables[0, 0])
            assert torch.isnan(ka[at, 3, 0, :64]).all() and torch.isnan(ka[at, 3, 0, 64:]).all()  # pairs (7, 71)
            assert torch.isfinite(ka[at, 3, 1]).all() and torch.isnan(va[at, 3, 0, :64]).all()
            assert torch.isfinite(va[at, 3, 0, 64:]).all() and torch.isfinite(ka[at, 13:]).all()


def test_codes_at_borders(cuda):
    """Numbers half way between two codes go to the even one, as 64-bit arithmetic has it."""
    x = torch.empty(1, 64, 1, 64, dtype=torch.float64, device="cuda")
    for i in range(64):
        s = 2.0 ** (i % 8 - 4) * (1 + (i // 8) / 8)
        x[0, i, 0] = torch.arange(64, device="cuda").double() * s / 4 + (i % 3 - 1) * s
        x[0, i, 0, 61:] = x[0, i, 0, 60]
    v = x.half()
    kv = empty_cache(4, 1, 4, 16, 1, 64, "fp16", [64])
    before = keep(kv)
    b2.paged_kv_append(kv, v, v)
    check(kv, before, None, v, v, None)


@pytest.mark.parametrize("D", [8, 64, 72, 96, 128, 192, 256])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_read(cuda, D, dt):
    g = gen(8)
    nkv, bs, mb = 3, 32, 5
    rows = torch.randn(11, bs, nkv, D, generator=g, device="cuda")
    pool = R.fill_pool(rows, rows.flip(0))
    k, v = R.pool_rows(pool, D)
    tables = torch.randperm(11, generator=g, device="cuda")[:10].to(torch.int32).view(2, mb)
    for lens, counts, T in (([150, 3], None, 200), ([150, 3], [40, 7], 50), ([160, 0], [160, 5], 160),
                            ([1000, 77], None, 30), ([17, -2], [-1, 4], 8), ([33, 16], [1, 16], 16)):
        kv = b2.PagedKV4(pool, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), D, DT[dt])
        wide = torch.randn(2, T, 2 * nkv, D, generator=g, device="cuda").to(DT[dt])
        was = wide.clone()
        n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
        b2.paged_kv_read(kv, wide[:, :, :nkv], wide[:, :, nkv:], counts=n)
        for b in range(2):
            L = max(0, min(lens[b], mb * bs))
            m = max(0, min(L, T, T if counts is None else counts[b]))
            pos = torch.arange(L - m, L, device="cuda")
            at = tables[b].long()[pos // bs], pos % bs
            for got, want in ((wide[b, :m, :nkv], k[at]), (wide[b, :m, nkv:], v[at])):
                tol = torch.finfo(DT[dt]).eps / 2 * (1 + 2.0 ** -12) * want.abs() + 2.0 ** -25
                assert ((got.double() - want).abs() <= tol).all()
            assert torch.equal(wide[b, m:], was[b, m:])


def test_read_leaves_rows_without_a_block(cuda):
    kv = empty_cache(4, 1, 3, 16, 2, 64, "fp16", [48])
    kv.pool.copy_(R.fill_pool(*(torch.randn(kv.num_blocks, 16, 2, 64, device="cuda") for _ in "kv")))
    kv.block_tables[0, 1] = kv.num_blocks
    k = torch.full((1, 48, 2, 64), 9.0, dtype=torch.float16, device="cuda")
    v = k.clone()
    b2.paged_kv_read(kv, k, v)
    assert (k[0, 16:32] == 9).all() and (v[0, 16:32] == 9).all() and not (k[0, :16] == 9).all()


def test_binding_refuses(cuda):
    kv = empty_cache(4, 2, 2, 16, 2, 64, "fp16", [3, 3])
    x = torch.zeros(2, 3, 2, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [dict(k=x[:1]), dict(k=x.bfloat16()), dict(k=x[:, :, :1]), dict(v=x[:, :2]), dict(v=x.cpu()),
           dict(q=q[:1]), dict(q=q, q_out=q[:, :, :2]), dict(q_out=q), dict(counts=n.long()), dict(counts=n[:1]),
           dict(positions=n.cpu()), dict(q=q.float())]
    for more in bad:
        with pytest.raises(ValueError):
            b2.paged_kv_append(kv, **{**dict(k=x, v=x), **more})
    for more in (dict(rope=b2.Rope(128)), dict(k=x.transpose(1, 3).contiguous().transpose(1, 3))):
        with pytest.raises(b2.B2Error) as e:
            b2.paged_kv_append(kv, **{**dict(k=x, v=x), **more})
        assert e.value.status == -2
    wide = q[:, :, :1].expand(-1, -1, 4, -1)  # four heads in one place: may be read, not written
    for call in (lambda: b2.paged_kv_append(kv, x, x, q=wide), lambda: b2.paged_kv_append(kv, x, x, q=q, q_out=wide),
                 lambda: b2.paged_kv_read(kv, x[:, :, :1].expand(-1, -1, 2, -1), x)):
        with pytest.raises(b2.B2Error) as e:
            call()
        assert e.value.status == -1
    b2.paged_kv_append(kv, x, x, q=wide, q_out=q)
    for more in (dict(k_out=x[:1]), dict(v_out=x[:, :2]), dict(k_out=x.float()), dict(counts=n.long())):
        with pytest.raises(ValueError):
            b2.paged_kv_read(kv, **{**dict(k_out=x, v_out=x), **more})
    with pytest.raises(ValueError):
        b2.paged_kv_read(empty_cache(16, 2, 2, 16, 2, 64, "fp16", [3, 3]), x, x)


def test_pool_past_32_bits(cuda):
    for bits in (4, 16):
        small = empty_cache(bits, 1, 1, 16, 1, 64, "fp16", [16], extra=0)
        block = small.pool[0].numel() if bits == 4 else 16 * 64
        far = -(-(2 ** 32 + 2 ** 20) // block) if bits == 4 else -(-(2 ** 31 + 2 ** 20) // block)
        table = small.block_tables + far
        if bits == 4:
            pool = torch.empty(far + 1, *small.pool.shape[1:], dtype=torch.uint8, device="cuda")
            kv = b2.PagedKV4(pool, table, small.seq_lens, 64, torch.float16)
        else:
            pool = torch.empty(far + 1, 16, 1, 64, dtype=torch.float16, device="cuda")
            kv = b2.PagedKV(pool, torch.empty_like(pool), table, small.seq_lens)
        x = torch.randn(1, 16, 1, 64, device="cuda").half()
        b2.paged_kv_append(kv, x, x)
        if bits == 4:
            b2.paged_kv_append(small, x, x)
            assert torch.equal(pool[far], small.pool[0])
            k, v = torch.empty_like(x), torch.empty_like(x)
            b2.paged_kv_read(kv, k, v)
            assert torch.equal(k, v) and (k - x).abs().max() < 0.5
        else:
            assert torch.equal(pool[far], x[0]) and torch.equal(kv.v[far], x[0])
        del kv, pool
        torch.cuda.empty_cache()
