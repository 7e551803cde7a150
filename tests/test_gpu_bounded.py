"""Bounded-cache attention on the GPU against 64-bit references
(bounded_ref.py): windowed prefill, paged decode with window, sinks and
accumulated weights, and eviction.

Bounds.  With u the unit roundoff of the 16-bit type (2^-11 half, 2^-8 bf16)
and A = sum_j p_j |v_j|: rounding the weights to 16 bits before the product
with V moves an output by at most u A, rounding the result by at most u |o| <=
u A.  Scores are sums of D exact products in 32 bits: with |q| |k| below 32
sqrt(D) (the inputs here) a logit is off by less than 2^-24 D^(1/2) 32 < 3e-5
for D <= 256, which changes every weight by that relative amount, the sum
likewise: 6e-5 A covers both and the 2^-22 of the exponential.  fp16 results
below its normal range round by up to 2^-25.  Weights added to a score: 6e-5 of
the weight, and 2^-23 of the score for the addition."""
import numpy as np
import pytest
import torch

import b2engine as b2
import bounded_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
U = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
NAN = float("nan")


def close(got, want, mag, dt):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    tol = (2 * U[dt] + 6e-5) * mag + 2.0 ** -25
    bad = err > tol
    assert not bad.any(), (int(bad.sum()), float((err - tol).max()), bad.nonzero()[0].tolist())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


# ---------------------------------------------------------------------------
# windowed prefill
# ---------------------------------------------------------------------------

def prefill_case(seed, B, S, start, nq, nkv, D, dt, window, sinks, lens=None):
    g = gen(seed)
    T = S + start
    q, k, v = (randn(g, B, n, h, D) for n, h in ((S, nq), (T, nkv), (T, nkv)))
    if lens is not None:
        for b, n in enumerate(lens):
            k[b, n:], v[b, n:] = NAN, NAN
    q, k, v = (t.to(DT[dt]) for t in (q, k, v))
    L = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((B, S, nq, D), NAN, dtype=DT[dt], device="cuda")
    b2.window_prefill_gqa(q, k, v, out, window=window, sinks=sinks, seq_lens=L)
    assert b2.device_status() == 0
    close(out, *R.window_prefill(q, k, v, lens, window, sinks), dt)


@pytest.mark.parametrize("D", [8, 40, 64, 80, 128, 160, 256])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_prefill_head_dims(cuda, D, dt):
    prefill_case(1, 2, 150, 0, 4, 2, D, dt, 40, 3)


@pytest.mark.parametrize("S", [1, 2, 16, 127, 128, 129, 255, 256, 257, 400])
@pytest.mark.parametrize("D", [64, 128])
def test_prefill_lengths(cuda, S, D):
    prefill_case(2, 1, S, 0, 2, 1, D, "fp16", 0, 0)
    prefill_case(3, 1, S, 0, 2, 1, D, "bf16", 100, 4)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (1, 200), (2, 0), (127, 0), (128, 4), (129, 128), (129, 129),
                                          (300, 1), (300, 300), (512, 4), (1000, 4), (0, 7), (1 << 40, 3)])
def test_prefill_masks(cuda, window, sinks):
    prefill_case(4, 1, 700, 0, 2, 1, 128, "bf16", window, sinks)
    prefill_case(5, 1, 700, 0, 2, 1, 64, "fp16", window, sinks)


@pytest.mark.parametrize("nq,nkv", [(32, 8), (28, 4), (36, 36), (33, 11), (40, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 200), (300, 4), (512, 130), (129, 129)])
def test_prefill_more_tiles_than_sms(cuda, nq, nkv, window, sinks):
    """Pairs of tiles: two heads at the same rows, or (odd groups) the next rows; several pairs per CTA."""
    prefill_case(13, 1, 700, 0, nq, nkv, 128, "bf16", window, sinks)
    prefill_case(14, 2, 401, 77, nq, nkv, 64, "fp16", window, sinks, lens=[478, 300])


def test_prefill_many_ragged_sequences(cuda):
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(0, 260, 70)]
    prefill_case(15, 70, 260, 0, 6, 2, 64, "bf16", 50, 3, lens=lens)
    prefill_case(16, 70, 200, 60, 3, 1, 128, "fp16", 0, 0, lens=lens)


@pytest.mark.parametrize("S,start", [(1, 0), (1, 500), (1, 511), (5, 123), (128, 128), (200, 333), (300, 1),
                                     (130, 1200)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 4), (257, 130)])
def test_prefill_chunks(cuda, S, start, window, sinks):
    prefill_case(6, 1, S, start, 4, 2, 128, "fp16", window, sinks)
    prefill_case(7, 2, S, start, 2, 2, 64, "bf16", window, sinks, lens=[start + S, start + max(0, S - 3)])


@pytest.mark.parametrize("lens", [[400, 399, 1, 0], [256, 128, 129, 257], [0, 0, 0, 400], [272, 255, 127, 130]])
def test_prefill_ragged_padding_is_never_seen(cuda, lens):
    """Rows past a sequence's length are NaN; outputs there are zero."""
    for dt, D in (("fp16", 128), ("bf16", 64), ("fp16", 72), ("bf16", 144)):
        prefill_case(8, 4, 400, 0, 4, 1, D, dt, 150, 5, lens=lens)


def test_prefill_pieces_equal_the_whole(cuda):
    """A prompt in chunks gives what one call gives (same tiles' arithmetic up to rounding)."""
    g = gen(9)
    S, nq, nkv, D = 600, 4, 2, 128
    q, k, v = (randn(g, 1, S, h, D).half() for h in (nq, nkv, nkv))
    whole = torch.empty_like(q)
    b2.window_prefill_gqa(q, k, v, whole, window=200, sinks=4)
    at = 0
    for n in (256, 1, 300, 43):
        part = torch.empty(1, n, nq, D, dtype=q.dtype, device="cuda")
        b2.window_prefill_gqa(q[:, at:at + n], k[:, :at + n], v[:, :at + n], part, window=200, sinks=4)
        assert (part.float() - whole[:, at:at + n].float()).abs().max() < 4e-3
        at += n


@pytest.mark.parametrize("D", [64, 128])
def test_prefill_strided_views(cuda, D):
    """q, k, v inside one fused projection, a head-major cache, and rows that 16-byte copies cannot take."""
    g = gen(10)
    B, S, nq, nkv = 2, 200, 4, 2
    fused = randn(g, B, S, nq + 2 * nkv, D).bfloat16()
    q, k, v = fused[:, :, :nq], fused[:, :, nq:nq + nkv], fused[:, :, nq + nkv:]
    out = torch.empty(B, S, nq, D, dtype=q.dtype, device="cuda")
    b2.window_prefill_gqa(q, k, v, out, window=77, sinks=2)
    close(out, *R.window_prefill(q, k, v, None, 77, 2), "bf16")
    kh = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    vh = v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    b2.window_prefill_gqa(q, kh, vh, out, window=77, sinks=2)
    close(out, *R.window_prefill(q, k, v, None, 77, 2), "bf16")
    odd = torch.empty(B * S * nkv * (D + 1) + 1, dtype=q.dtype, device="cuda")[1:].view(B, S, nkv, D + 1)[..., :D]
    odd.copy_(k)
    b2.window_prefill_gqa(q, odd, v, out, window=77, sinks=2)
    close(out, *R.window_prefill(q, k, v, None, 77, 2), "bf16")


def test_prefill_large_logits(cuda):
    """Logits of some hundreds: the running maximum moves far, nothing overflows."""
    g = gen(11)
    q, k, v = (randn(g, 1, 500, h, 128) for h in (2, 1, 1))
    k *= torch.linspace(0.1, 8, 500, device="cuda")[None, :, None, None]
    q, k, v = (8 * q).half(), k.half(), v.half()
    out = torch.empty_like(q)
    b2.window_prefill_gqa(q, k, v, out, window=300, sinks=4)
    want, mag = R.window_prefill(q, k, v, None, 300, 4)
    # |q||k| up to 64 times the bound's: a logit off by 2e-3
    err = (out.double() - want).abs()
    assert (err <= (2 * U["fp16"] + 4e-3) * mag + 2.0 ** -25).all()


def test_prefill_runs_on_the_stream_it_is_given(cuda):
    g = gen(12)
    q, k, v = (randn(g, 1, 300, h, 64).half() for h in (4, 2, 2))
    want, mag = R.window_prefill(q, k, v, None, 64, 1)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(20):
        out.zero_()
    s.wait_stream(torch.cuda.current_stream())
    b2.window_prefill_gqa(q, k, v, out, window=64, sinks=1, stream=s.cuda_stream)
    s.synchronize()
    close(out, want, mag, "fp16")


# ---------------------------------------------------------------------------
# paged decode
# ---------------------------------------------------------------------------

class Cache:
    """Pools of B sequences with scattered blocks; rows past a sequence's end, spare blocks and, with a window,
    everything the window has left behind are NaN."""

    def __init__(self, seed, lens, bs, nkv, D, dt, layout="slot", max_blocks=None, spare=3):
        g = gen(seed)
        self.lens, self.bs, self.nkv, self.D, self.dt = lens, bs, nkv, D, dt
        mb = max_blocks or max(1, max(-(-n // bs) for n in lens))
        nb = len(lens) * mb + spare
        shape = (nb, bs, nkv, D) if layout == "slot" else (nb, nkv, bs, D)
        self.k, self.v = randn(g, *shape).to(DT[dt]), randn(g, *shape).to(DT[dt])
        if layout == "head":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
        self.tables = perm[:len(lens) * mb].view(len(lens), mb).contiguous()
        self.free = perm[len(lens) * mb:]
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.scores = torch.rand(nb, nkv, bs, generator=g, device="cuda")
        self.poison(lambda b, pos: pos >= lens[b])
        self.k[self.free.long()], self.v[self.free.long()] = NAN, NAN
        self.kv = b2.PagedKV(self.k, self.v, self.tables, self.seq_lens)

    def poison(self, where):
        for b in range(len(self.lens)):
            pos = torch.arange(self.tables.shape[1] * self.bs, device="cuda")
            pos = pos[where(b, pos)]
            blk = self.tables[b].long()[pos // self.bs]
            ok = (blk >= 0) & (blk < self.k.shape[0])
            self.k[blk[ok], (pos % self.bs)[ok]] = NAN
            self.v[blk[ok], (pos % self.bs)[ok]] = NAN


def decode_case(seed, lens, bs, nq, nkv, D, dt, window=0, sinks=0, scored=True, layout="slot", ws=True, cache=None):
    c = cache or Cache(seed, lens, bs, nkv, D, dt, layout)
    B = len(lens)
    q = randn(gen(seed + 1), B, nq, D).to(DT[dt])
    if window:
        c.poison(lambda b, pos: (pos < lens[b] - window) & (pos >= sinks))
    before = c.scores.clone()
    want, mag, new, add = R.paged_decode(q, c.k, c.v, c.tables, lens, window, sinks, before)
    out = torch.full((B, nq, D), NAN, dtype=DT[dt], device="cuda")
    span = c.tables.shape[1] * c.bs
    w = b2.Workspace(b2.paged_decode_workspace_bytes(B, nq, nkv, D, min(span, window + sinks) if window else span,
                                                     scored)) if ws else None
    b2.paged_decode_gqa(q, c.kv, out, window=window, sinks=sinks, scores=c.scores if scored else None, ws=w)
    assert b2.device_status() == 0
    close(out, want, mag, dt)
    if not scored:
        assert torch.equal(c.scores, before)
        return c
    err = (c.scores.double() - new).abs()
    assert (err <= 6e-5 * add + 2.0 ** -23 * new.abs()).all(), float(err.max())
    assert torch.equal(c.scores[add == 0], before[add == 0])  # invisible positions keep their bits
    return c


@pytest.mark.parametrize("D", [8, 32, 48, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_decode_head_dims(cuda, D, dt):
    decode_case(20, [100, 333], 16, 6, 2, D, dt)


@pytest.mark.parametrize("nq,nkv", [(1, 1), (2, 1), (7, 1), (8, 1), (9, 1), (16, 1), (17, 1), (40, 1), (14, 2), (12, 12)])
def test_decode_group_sizes(cuda, nq, nkv):
    for scored in (False, True):
        decode_case(21, [70, 200, 1], 16, nq, nkv, 64, "fp16", scored=scored)
        decode_case(22, [70, 200, 1], 16, nq, nkv, 128, "bf16", scored=scored, window=50, sinks=3)


@pytest.mark.parametrize("bs", [1, 5, 8, 16, 24, 32, 128])
@pytest.mark.parametrize("layout", ["slot", "head"])
def test_decode_block_sizes(cuda, bs, layout):
    decode_case(23, [1, 2, 15, 16, 17, 63, 64, 65, 130, 259], bs, 4, 2, 128, "fp16", layout=layout)
    decode_case(24, [1, 2, 15, 16, 17, 63, 64, 65, 130, 259], bs, 4, 2, 64, "bf16", layout=layout, window=37, sinks=6)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (1, 64), (15, 17), (16, 16), (64, 0), (64, 4), (65, 100),
                                          (500, 4), (5000, 1), (0, 9)])
def test_decode_masks(cuda, window, sinks):
    lens = [1, 64, 65, 128, 700, 1000]
    decode_case(25, lens, 16, 8, 2, 128, "bf16", window, sinks)
    decode_case(26, lens, 16, 8, 2, 64, "fp16", window, sinks)


def test_decode_empty_sequences(cuda):
    decode_case(27, [0, 5, 0], 16, 4, 2, 64, "fp16")
    decode_case(28, [0], 16, 4, 2, 128, "bf16", scored=False)


@pytest.mark.parametrize("B,L", [(1, 5000), (3, 20000), (40, 300), (2, 40000)])
def test_decode_long_and_many(cuda, B, L):
    lens = [max(1, L - 977 * b) for b in range(B)]
    for scored in (False, True):
        decode_case(29, lens, 16, 8, 2, 128, "fp16", scored=scored)
    decode_case(30, lens, 32, 8, 2, 64, "bf16", scored=True)
    decode_case(31, lens, 32, 8, 2, 128, "bf16", scored=False, ws=False)


def test_decode_batch_above_a_thousand(cuda):
    rng = np.random.default_rng(3)
    decode_case(32, [int(x) for x in rng.integers(0, 40, 1500)], 16, 2, 1, 64, "fp16")


def test_decode_missing_blocks_are_left_out(cuda):
    c = Cache(33, [200, 90], 16, 2, 64, "fp16")
    c.tables[0, 3], c.tables[0, 7], c.tables[1, 0] = -1, 10 ** 6, -5
    decode_case(33, [200, 90], 16, 4, 2, 64, "fp16", cache=c)
    c = Cache(34, [40], 16, 2, 64, "fp16")
    c.tables.fill_(-1)
    decode_case(34, [40], 16, 4, 2, 64, "fp16", cache=c)


def test_decode_entries_of_blocks_left_behind_are_not_used(cuda):
    c = Cache(35, [1000], 16, 2, 128, "bf16")
    c.tables[0, 1:40] = 2 ** 31 - 1
    decode_case(35, [1000], 16, 4, 2, 128, "bf16", window=200, sinks=4, cache=c)


def test_decode_lengths_above_the_table_are_cut(cuda):
    c = Cache(36, [64], 16, 2, 64, "fp16")
    c.seq_lens.fill_(100)
    decode_case(36, [64], 16, 4, 2, 64, "fp16", cache=c)


def test_decode_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 elements, the sequence in its last blocks."""
    nb, bs, nkv, D = 70000, 64, 8, 128
    k = torch.zeros(nb, bs, nkv, D, dtype=torch.float16, device="cuda")
    assert k.numel() > 2 ** 32
    v = torch.zeros_like(k)
    n = 150
    tables = torch.tensor([[nb - 1, nb - 3, nb - 2]], dtype=torch.int32, device="cuda")
    g = gen(37)
    for t in (k, v):
        t[nb - 3:] = randn(g, 3, bs, nkv, D).half()
    q = randn(g, 1, 16, D).half()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = torch.empty(1, 16, D, dtype=torch.float16, device="cuda")
    scores = torch.zeros(nb, nkv, bs, device="cuda")
    w = b2.Workspace(b2.paged_decode_workspace_bytes(1, 16, nkv, D, 3 * bs, True))
    b2.paged_decode_gqa(q, b2.PagedKV(k, v, tables, lens), out, scores=scores, ws=w)
    want, mag, new, _ = R.paged_decode(q, k[nb - 3:], v[nb - 3:], tables - (nb - 3), [n], 0, 0, scores[nb - 3:] * 0)
    close(out, want, mag, "fp16")
    assert ((scores[nb - 3:].double() - new).abs() <= 1e-4 * new).all()


def test_decode_strided_queries_and_repeatable_bits(cuda):
    """q as the head of fused q|k|v rows; two runs give the same bits, scores included."""
    g = gen(38)
    c = Cache(38, [3000, 1234, 7], 16, 8, 128, "fp16")
    fused = randn(g, 3, 48, 128).half()
    q = fused[:, :32]
    ws = b2.Workspace(b2.paged_decode_workspace_bytes(3, 32, 8, 128, c.tables.shape[1] * 16, True))
    got = []
    for _ in range(2):
        sc, out = c.scores.clone(), torch.empty(3, 32, 128, dtype=torch.float16, device="cuda")
        b2.paged_decode_gqa(q, c.kv, out, scores=sc, ws=ws)
        got.append((out, sc))
    want, mag, _, _ = R.paged_decode(q, c.k, c.v, c.tables, [3000, 1234, 7], 0, 0)
    close(got[0][0], want, mag, "fp16")
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_decode_in_a_graph_follows_lengths_and_tables(cuda):
    c = Cache(39, [400, 90], 16, 2, 64, "fp16")
    q = randn(gen(40), 2, 4, 64).half()
    out = torch.empty(2, 4, 64, dtype=torch.float16, device="cuda")
    ws = b2.Workspace(b2.paged_decode_workspace_bytes(2, 4, 2, 64, c.tables.shape[1] * 16))
    b2.paged_decode_gqa(q, c.kv, out, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b2.paged_decode_gqa(q, c.kv, out, ws=ws)
    for lens in ([400, 90], [33, 1], [1, 90]):
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        want, mag, _, _ = R.paged_decode(q, c.k, c.v, c.tables, lens, 0, 0)
        close(out, want, mag, "fp16")


def test_all_three_in_one_graph(cuda):
    """Prefill, decode and eviction captured together and replayed on new contents."""
    c = Cache(42, [300, 200], 16, 2, 64, "bf16")
    g = gen(43)
    q, k, v = (randn(g, 1, 200, h, 64).bfloat16() for h in (4, 2, 2))
    out, q1, o1 = torch.empty_like(q), randn(g, 2, 4, 64).bfloat16(), torch.empty(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    kept = torch.empty(2, 2, 64, dtype=torch.int32, device="cuda")
    ws = b2.Workspace(b2.paged_decode_workspace_bytes(2, 4, 2, 64, c.tables.shape[1] * 16, True))

    def calls():
        b2.window_prefill_gqa(q, k, v, out, window=30, sinks=2)
        b2.paged_decode_gqa(q1, c.kv, o1, scores=c.scores, ws=ws)
        b2.paged_kv_evict(c.kv, c.scores, 64, kept, c.seq_lens, sinks=2, recent=10)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        calls()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for seed in (1, 2):
        d = Cache(44 + seed, [300, 200], 16, 2, 64, "bf16")
        for t in (c.k, c.v, c.scores, c.seq_lens, c.tables):
            src = d.k if t is c.k else d.v if t is c.v else d.scores if t is c.scores else d.seq_lens if t is c.seq_lens else d.tables
            t.copy_(src)
        q.copy_(randn(gen(seed), 1, 200, 4, 64))
        graph.replay()
        torch.cuda.synchronize()
        close(out, *R.window_prefill(q, k, v, None, 30, 2), "bf16")
        want, mag, score, add = R.paged_decode(q1, d.k, d.v, d.tables, [300, 200], 0, 0, d.scores)
        close(o1, want, mag, "bf16")
        assert c.seq_lens.tolist() == [64, 64]
        # the choice goes by the scores the decode call left, which the reference gives to within their rounding
        for b in range(2):
            for h in range(2):
                i = kept[b, h].long()
                assert i[:2].tolist() == [0, 1] and i[-10:].tolist() == list(range([300, 200][b] - 10, [300, 200][b]))
                at = lambda p: score[d.tables[b].long()[p // 16], h, p % 16]  # noqa: E731
                mid = torch.arange(2, [300, 200][b] - 10, device="cuda")
                out_of = mid[~torch.isin(mid, i)]
                assert at(i[2:-10]).min() >= at(out_of).max() - 1e-4


def test_decode_workspace_too_small(cuda):
    c = Cache(41, [400], 16, 2, 64, "fp16")
    q = randn(gen(41), 1, 4, 64).half()
    with pytest.raises(b2.B2Error) as e:
        b2.paged_decode_gqa(q, c.kv, torch.empty_like(q), scores=c.scores, ws=b2.Workspace(16))
    assert e.value.status == -3


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------

def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def evict_case(seed, lens, bs, nkv, D, dt, budget, sinks, recent, scores=None, layout="slot", in_place=False,
               alias=False, mangle=None):
    B = len(lens)
    need = -(-budget // bs)
    c = Cache(seed, lens, bs, nkv, D, dt, layout, spare=B * need + 2)
    if scores is not None:
        c.scores = scores(c.scores)
    dst = None if in_place else c.free[:B * need].view(B, need).contiguous()
    if mangle:
        mangle(c, dst)
    want = R.paged_evict(c.k, c.v, c.scores, c.tables, lens, budget, sinks, recent, dst)
    kept = torch.full((B, nkv, budget), -7, dtype=torch.int32, device="cuda")
    new = c.seq_lens if alias else torch.full((B,), -7, dtype=torch.int32, device="cuda")
    b2.paged_kv_evict(c.kv, c.scores, budget, kept, new, sinks=sinks, recent=recent, dst_tables=dst)
    torch.cuda.synchronize()
    k2, v2, s2, kept2, new2 = want
    assert torch.equal(new.cpu(), new2)
    assert torch.equal(kept.cpu(), kept2)
    assert torch.equal(bits(c.k), bits(k2)) and torch.equal(bits(c.v), bits(v2))
    assert torch.equal(bits(c.scores), bits(s2))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bs,layout", [(1, "slot"), (5, "slot"), (16, "slot"), (16, "head"), (128, "slot")])
def test_evict_blocks(cuda, in_place, bs, layout):
    evict_case(50, [1, 40, 41, 100, 517], bs, 2, 64, "fp16", 40, 4, 8, layout=layout, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("D,dt", [(8, "fp16"), (40, "bf16"), (64, "bf16"), (128, "fp16"), (144, "fp16"), (256, "bf16")])
def test_evict_head_dims(cuda, in_place, D, dt):
    evict_case(51, [300, 90], 16, 3, D, dt, 100, 2, 30, in_place=in_place)


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (7, 0, 0), (64, 64, 0), (64, 0, 64),
                                                 (64, 32, 32), (64, 31, 32), (299, 4, 4), (300, 4, 4), (301, 4, 4)])
def test_evict_budgets(cuda, budget, sinks, recent):
    for in_place in (False, True):
        evict_case(52, [300, 299, 64, 65, 0], 16, 2, 64, "fp16", budget, sinks, recent, in_place=in_place)


SCORES = {
    "equal": lambda s: torch.ones_like(s),
    "zero": lambda s: torch.zeros_like(s),
    "signed zeros": lambda s: torch.where(s < 0.5, 0.0, -0.0),
    "few values": lambda s: (s * 4).floor(),
    "negative": lambda s: -s,
    "mixed": lambda s: s - 0.5,
    "infinities": lambda s: torch.where(s < 0.2, -float("inf"), torch.where(s > 0.8, float("inf"), s)),
    "nan": lambda s: torch.where(s < 0.1, NAN, s),
    "all nan": lambda s: torch.full_like(s, NAN),
    "tiny": lambda s: s * 1e-42,
    "rising": lambda s: s * 0 + torch.arange(s.numel(), device=s.device).view(s.shape),
}


@pytest.mark.parametrize("kind", sorted(SCORES))
def test_evict_scores(cuda, kind):
    for in_place in (False, True):
        evict_case(53, [500, 333, 64], 16, 2, 64, "fp16", 64, 3, 5, scores=SCORES[kind], in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_long(cuda, in_place):
    evict_case(54, [9000, 20000, 2049], 16, 2, 128, "fp16", 2048, 4, 500, in_place=in_place)
    evict_case(55, [70001], 16, 1, 64, "bf16", 30000, 4, 500, in_place=in_place)
    evict_case(56, [70001], 16, 1, 8, "bf16", 69000, 4, 500, scores=SCORES["few values"], in_place=in_place)


def test_evict_lengths_may_be_updated_in_place(cuda):
    evict_case(57, [500, 20, 64], 16, 4, 64, "fp16", 64, 3, 5, in_place=True, alias=True)


def test_evict_many_sequences(cuda):
    rng = np.random.default_rng(4)
    evict_case(58, [int(x) for x in rng.integers(0, 200, 300)], 16, 1, 16, "fp16", 50, 2, 7, in_place=True)


def test_evict_then_decode(cuda):
    """Decode over the shrunk cache equals attention over the kept rows."""
    c = Cache(59, [900, 400], 16, 2, 64, "fp16")
    kept = torch.empty(2, 2, 128, dtype=torch.int32, device="cuda")
    k0, v0 = c.k.clone(), c.v.clone()
    b2.paged_kv_evict(c.kv, c.scores, 128, kept, c.seq_lens, sinks=4, recent=32)
    q = randn(gen(60), 2, 4, 64).half()
    out = torch.empty_like(q)
    b2.paged_decode_gqa(q, c.kv, out, ws=b2.Workspace(b2.paged_decode_workspace_bytes(2, 4, 2, 64, 57 * 16)))
    assert c.seq_lens.tolist() == [128, 128]
    for b in range(2):
        for h in range(4):
            i = kept[b, h // 2].long()
            blk, slot = c.tables[b].long()[i // 16], i % 16
            o, a, _ = R.attend(q[b, h][None], k0[blk, slot, h // 2], v0[blk, slot, h // 2],
                               torch.ones(1, 128, dtype=torch.bool, device="cuda"))
            close(out[b, h][None], o, a, "fp16")
