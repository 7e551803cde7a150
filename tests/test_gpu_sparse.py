"""Block bounds, the choice of blocks and a decode over the chosen ones on the
GPU, against references that they have to equal (kv4_ref.py), and the operators
together, as a server would use them."""
import math

import pytest
import torch

import b2engine as b2
import kv4_ref as R
from test_gpu_append import empty_cache
from test_gpu_kv4 import close, make, make16, ws_for

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def want_bounds(kv, k, lens, newest, codes, scale):
    """codes and scale (CPU clones) with the touched blocks' bounds written."""
    bs = kv.block_size
    for b, n in enumerate(lens):
        n = max(0, min(n, kv.block_tables.shape[1] * bs))
        since = 0 if newest is None else n - max(0, min(n, newest[b]))
        if since >= n:
            continue
        for j in range(since // bs, -(-n // bs)):
            at = int(kv.block_tables[b, j])
            if 0 <= at < kv.num_blocks:
                codes[at], scale[at] = R.bounds(k[at, : min(bs, n - j * bs)])
    return codes, scale


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("lens,nkv,D,bs,dt,newest", [
    ([1], 1, 64, 16, "fp16", None),
    ([100, 16, 0, 33], 2, 128, 16, "bf16", None),
    ([100, 16, 0, 33], 2, 128, 16, "fp16", [1, 1, 1, 2]),
    ([100, 64, 90], 3, 80, 64, "fp16", [40, 0, 1000]),
    ([300, 5], 1, 256, 128, "bf16", [-3, 5]),
    ([70, 40], 4, 72, 32, "bf16", None),
    ([20, 17], 2, 8, 16, "fp16", None),
    ([40] * 140, 1, 64, 16, "fp16", [1] * 140),
    ([30] * 300, 2, 64, 16, "bf16", None),
])
def test_bounds(cuda, bits, lens, nkv, D, bs, dt, newest):
    _, kv, k, _ = (make if bits == 4 else make16)(1, lens, nkv, nkv, D, bs, dt)
    bd = b2.BlockBounds(codes=torch.randint(-128, 128, (kv.num_blocks, nkv, 2, D), device="cuda").to(torch.int8),
                        scale=torch.randn(kv.num_blocks, nkv, device="cuda"))
    want = want_bounds(kv, k, lens, newest, bd.codes.cpu(), bd.scale.cpu())
    n = None if newest is None else torch.tensor(newest, dtype=torch.int32, device="cuda")
    b2.paged_block_bounds(kv, bd, newest=n)
    assert torch.equal(bd.codes.cpu(), want[0]) and torch.equal(bd.scale.cpu(), want[1])


def test_bounds_of_odd_values(cuda):
    big = torch.finfo(torch.bfloat16).max
    k = torch.randn(10, 16, 2, 64, generator=gen(2), device="cuda").bfloat16()
    k[0], k[1, 3, 0, 5], k[2, 15, 1, 63], k[3] = 0, math.nan, -math.inf, big
    k[4], k[5], k[6] = -big, 1e-38, 127.0
    k[7], k[8, :, 0], k[8, :, 1] = 127.5, 1e-30, -254.0
    kv = b2.PagedKV(k, k.clone(), torch.arange(10, dtype=torch.int32, device="cuda")[None],
                    torch.tensor([160], dtype=torch.int32, device="cuda"))
    kv.block_tables[0, 9] = -1
    bd = b2.BlockBounds(10, 2, 64)
    want = want_bounds(kv, k.double(), [160], None, bd.codes.cpu(), bd.scale.cpu())
    b2.paged_block_bounds(kv, bd)
    assert torch.equal(bd.scale.cpu(), want[1]) and torch.equal(bd.codes.cpu(), want[0])
    v = bd.codes.double() * bd.scale.double()[..., None, None]
    fine = torch.isfinite(bd.scale)
    assert (v[:9, :, 0] <= k[:9].double().amin(1))[fine[:9]].all() and (v[:9, :, 1] >= k[:9].double().amax(1))[fine[:9]].all()


def want_blocks(q, kv, bd, lens, n, first, last):
    B, nkv = q.shape[0], kv.nkv
    out = torch.full((B, nkv, n), -1, dtype=torch.int32)
    for b in range(B):
        L = max(0, min(lens[b], kv.block_tables.shape[1] * kv.block_size))
        nb = -(-L // kv.block_size)
        at = kv.block_tables[b, :nb].long().cpu()
        there = (at >= 0) & (at < kv.num_blocks)
        for h in range(nkv):
            g = q.shape[1] // nkv
            s = R.score(q[b, h * g:(h + 1) * g].cpu(), bd.codes[:, h].cpu()[at.clamp(0, kv.num_blocks - 1)],
                        bd.scale[:, h].cpu()[at.clamp(0, kv.num_blocks - 1)])
            s = torch.where(there, s, -math.inf)
            pick = R.choose(s.tolist(), n, first, last)
            out[b, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return out


def chosen(q, kv, bd, n, first, last):
    out = torch.full((q.shape[0], kv.nkv, n), 77, dtype=torch.int32, device="cuda")
    ws = b2.Workspace(b2.paged_block_select_workspace_bytes(q.shape[0], kv.nkv, kv.block_tables.shape[1]))
    assert b2.paged_block_select(q, kv, bd, out, first=first, last=last, ws=ws) is out
    again = torch.empty_like(out)
    b2.paged_block_select(q, kv, bd, again, first=first, last=last, ws=ws)
    assert torch.equal(out, again)
    return out.cpu()


def bare(seed, lens, nkv, D, bs, dt, group, blocks=None):
    """A cache of no rows to speak of, and bounds of their own."""
    g = gen(seed)
    B, mb = len(lens), max(1, -(-max(lens) // bs))
    nb = blocks or B * mb
    tables = torch.randint(0, nb, (B, mb), generator=g, device="cuda").to(torch.int32)
    x = torch.randint(-127, 128, (nb, nkv, 2, D), generator=g, device="cuda")
    x = torch.sort(x, 2).values.to(torch.int8)
    scale = 2.0 ** torch.randint(-7, -4, (nb, nkv), generator=g, device="cuda").float()
    pool = torch.zeros(nb, nkv, bs // 16, R.tile_bytes(D), dtype=torch.uint8, device="cuda")
    kv = b2.PagedKV4(pool, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), D, DT[dt])
    q = torch.randn(B, nkv * group, D, generator=g, device="cuda").to(DT[dt])
    return q, kv, b2.BlockBounds(codes=x, scale=scale)


@pytest.mark.parametrize("lens,nkv,D,group,dt,n,first,last", [
    ([1], 1, 64, 1, "fp16", 1, 0, 0),
    ([1000, 300, 16, 0], 2, 128, 4, "bf16", 5, 1, 2),
    ([1000, 300, 16, 0], 2, 128, 4, "fp16", 62, 1, 1),
    ([1000, 999], 3, 80, 3, "fp16", 7, 0, 0),
    ([1000, 999], 1, 72, 17, "bf16", 9, 9, 0),
    ([1000, 999], 1, 8, 2, "bf16", 9, 4, 5),
    ([600, 90], 2, 256, 8, "fp16", 11, 1, 1),
    ([20000, 7777, 30], 2, 64, 4, "fp16", 64, 1, 2),
    ([140000], 1, 64, 2, "bf16", 300, 4, 4),
    ([131072], 2, 64, 2, "fp16", 40, 1, 2),
    ([100000, 70000], 1, 8, 1, "bf16", 64, 0, 0),
    ([33] * 600, 8, 64, 1, "fp16", 2, 0, 1),
])
def test_choice(cuda, lens, nkv, D, group, dt, n, first, last):
    q, kv, bd = bare(3, lens, nkv, D, 16, dt, group, blocks=min(4000, sum(-(-x // 16) for x in lens) + 5))
    assert torch.equal(chosen(q, kv, bd, n, first, last), want_blocks(q, kv, bd, lens, n, first, last))


@pytest.mark.parametrize("L", [65536, 131072, 300000])
def test_ties_of_long_sequences(cuda, L):
    """Scores of three values: the best of the best one's blocks, then the first of the next one's."""
    q, kv, bd = bare(5, [L], 1, 64, 16, "fp16", 2)
    nb = L // 16
    kv.block_tables.copy_(torch.arange(nb, device="cuda")[None])
    bd.scale.fill_(1.0)
    bd.codes.fill_(3)
    bd.codes[::10, :, 1], bd.codes[5::1000, :, 1] = 20, 90
    q.fill_(1.0)
    n = nb // 1000 + 1 + nb // 20
    assert torch.equal(chosen(q, kv, bd, n, 1, 1), want_blocks(q, kv, bd, [L], n, 1, 1))


@pytest.mark.parametrize("what", ["ties", "zero query", "nan query", "infinite query", "infinite scale", "no block",
                                  "large scales", "tiny query", "nan scale"])
def test_choice_of_odd_values(cuda, what):
    lens = [5000, 400]
    q, kv, bd = bare(4, lens, 2, 64, 16, "bf16", 4)
    if what == "ties":
        bd.codes.fill_(5)
        bd.codes[::7] = 6
        bd.scale.fill_(1.0)
    elif what == "zero query":
        q.zero_()
    elif what == "nan query":
        q[0, 3, 5] = math.nan
    elif what == "infinite query":
        q[0, 3, 5], q[1, 0, 0] = math.inf, -math.inf
    elif what == "infinite scale":
        bd.scale[::5] = math.inf
    elif what == "no block":
        kv.block_tables[:, ::3] = -1
        kv.block_tables[1, 1::3] = kv.num_blocks
    elif what == "large scales":
        bd.scale[::2] = 2.0 ** 110
        bd.scale[1::4] = 2.0 ** -120
    elif what == "tiny query":
        q *= 2.0 ** -100
    if what == "nan scale":  # never written: any choice, but inside the sequence, ascending, of full length
        bd.scale.fill_(math.nan)
        got = chosen(q, kv, bd, 6, 1, 2)
        for b, L in enumerate(lens):
            for row in got[b].tolist():
                assert row == sorted(set(row)) and row[0] == 0 and row[-1] == -(-L // 16) - 1
        return
    for n, first, last in ((6, 1, 2), (40, 0, 0)):
        assert torch.equal(chosen(q, kv, bd, n, first, last), want_blocks(q, kv, bd, lens, n, first, last))


def test_refusals(cuda):
    q, kv, bd = bare(5, [100, 50], 2, 64, 16, "fp16", 2)
    out = torch.zeros(2, 2, 3, dtype=torch.int32, device="cuda")
    ws = b2.Workspace(b2.paged_block_select_workspace_bytes(2, 2, kv.block_tables.shape[1]))
    other = b2.BlockBounds(kv.num_blocks + 1, 2, 64)
    for args in ((q.bfloat16(), kv, bd, out), (q[:1], kv, bd, out), (q, kv, other, out), (q, kv, bd, out.long()),
                 (q, kv, bd, out[:, :1]), (q, kv, bd, out.cpu())):
        with pytest.raises(ValueError):
            b2.paged_block_select(*args, ws=ws)
    for more, status in ((dict(first=2, last=2, ws=ws), -1), (dict(), -3), (dict(ws=b2.Workspace(16)), -3)):
        with pytest.raises(b2.B2Error) as e:
            b2.paged_block_select(q, kv, bd, out, **more)
        assert e.value.status == status
    for more in (dict(first=2 ** 32), dict(last=2 ** 32 + 1), dict(first=-2 ** 32), dict(last=-1)):  # no bits are dropped
        with pytest.raises(b2.B2Error) as e:
            b2.paged_block_select(q, kv, bd, out, ws=ws, **more)
        assert e.value.status == -1
    with pytest.raises(ValueError):
        b2.paged_block_bounds(kv, other)
    with pytest.raises(ValueError):
        b2.paged_block_bounds(kv, bd, newest=out)


@pytest.mark.parametrize("bits", [4, 16])
def test_together(cuda, bits):
    """Prompts appended in two chunks, the second one's attention over all rows, then decode steps over chosen blocks:
    append, bounds, choice and attention captured once and replayed with new tokens."""
    dt, B, nq, nkv, D, bs, n = torch.bfloat16, 2, 8, 2, 64, 16, 5
    u = 2.0 ** -8
    g = gen(6)
    S = [90, 70]
    kv = empty_cache(bits, B, 10, bs, nkv, D, "bf16", [0, 0])
    rope = b2.Rope(D, theta=10000.0)
    qkv = torch.randn(B, 90, nq + 2 * nkv, D, generator=g, device="cuda").to(dt)
    q, k, v = qkv[:, :, :nq], qkv[:, :, nq:nq + nkv], qkv[:, :, nq + nkv:]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    # 60 tokens of each, then what is left
    turned = torch.empty(B, 90, nq, D, dtype=dt, device="cuda")
    kv.seq_lens.copy_(i32([60, 60]))
    b2.paged_kv_append(kv, k[:, :60], v[:, :60], q=q[:, :60], q_out=turned[:, :60], rope=rope)
    kv.seq_lens.copy_(i32(S))
    b2.paged_kv_append(kv, k[:, 60:], v[:, 60:], q=q[:, 60:], q_out=turned[:, 60:], rope=rope, counts=i32([30, 10]))
    if bits == 4:
        kr, vr = (torch.zeros(B, 90, nkv, D, dtype=dt, device="cuda") for _ in "kv")
        b2.paged_kv_read(kv, kr, vr, counts=kv.seq_lens)
    else:
        at = kv.block_tables.long()[:, torch.arange(90, device="cuda") // bs], torch.arange(90, device="cuda") % bs
        kr, vr = kv.k[at].contiguous(), kv.v[at].contiguous()
    out = torch.empty(B, 30, nq, D, dtype=dt, device="cuda")
    b2.window_prefill_gqa(turned[:, 60:].contiguous(), kr, vr, out, seq_lens=kv.seq_lens)
    for b, L in enumerate(S):
        for t in (60, L - 1):
            for h in range(nq):
                want, mag = R.attend(turned[b, t, h][None], kr[b, :, h // 4], vr[b, :, h // 4],
                                     torch.arange(90, device="cuda") <= t)
                assert ((out[b, t - 60, h].double() - want[0]).abs() <= (2 * u + 1e-4) * mag[0] + 1e-6).all()
    bd = b2.BlockBounds(kv.num_blocks, nkv, D)
    b2.paged_block_bounds(kv, bd)
    ws = ws_for(kv, nq)
    sws = b2.Workspace(b2.paged_block_select_workspace_bytes(B, nkv, 10))
    tok = torch.empty(B, 1, nq + 2 * nkv, D, dtype=dt, device="cuda")
    qt, o = torch.empty(B, 1, nq, D, dtype=dt, device="cuda"), torch.empty(B, nq, D, dtype=dt, device="cuda")
    blocks, one = torch.empty(B, nkv, n, dtype=torch.int32, device="cuda"), i32([1, 1])

    def step():
        kv.seq_lens.add_(1)
        b2.paged_kv_append(kv, tok[:, :, nq:nq + nkv], tok[:, :, nq + nkv:], q=tok[:, :, :nq], q_out=qt, rope=rope)
        b2.paged_block_bounds(kv, bd, newest=one)
        b2.paged_block_select(qt[:, 0], kv, bd, blocks, first=1, last=1, ws=sws)
        b2.paged_decode_gqa(qt[:, 0], kv, o, blocks=blocks, ws=ws)

    tok.copy_(torch.randn(tok.shape, generator=g, device="cuda"))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens = [s + 1 for s in S]
    assert kv.seq_lens.tolist() == lens  # capturing runs nothing
    for _ in range(20):
        tok.copy_(torch.randn(tok.shape, generator=g, device="cuda"))
        graph.replay()
        lens = [x + 1 for x in lens]
        if bits == 4:
            kk, vv = R.pool_rows(kv.pool, D)
        else:
            kk, vv = kv.k.double(), kv.v.double()
        want = want_bounds(kv, kk, lens, None, bd.codes.cpu(), bd.scale.cpu())
        assert torch.equal(bd.codes.cpu(), want[0]) and torch.equal(bd.scale.cpu(), want[1])
        assert torch.equal(blocks.cpu(), want_blocks(qt[:, 0], kv, bd, lens, n, 1, 1))
        want, mag = R.decode(qt[:, 0], kk, vv, kv.block_tables, lens, blocks=blocks.cpu())
        held = torch.isfinite(kk).all(-1, keepdim=True) & (kk.abs() < 100).all(-1, keepdim=True)
        close(o, want, mag, qt[:, 0], torch.where(held, kk, 0.0), torch.where(held, vv, 0.0), n * bs)
