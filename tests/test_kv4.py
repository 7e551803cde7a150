"""The 4-bit paged cache, the paged append and sparse decoding without a GPU:
what they refuse, and the 64-bit references of the GPU tests on small cases
worked by hand."""
import ctypes as C
import math

import pytest
import torch

import b2engine as b2
import kv4_ref as R

FAKE = 1 << 20  # a non-null, 16-byte-aligned address that nothing reads


def cache16(**over):
    f = dict(k=FAKE, v=FAKE, block_tables=FAKE, seq_lens=FAKE, stride_block=16 * 2 * 64, stride_slot=2 * 64,
             stride_head=64, num_blocks=8, block_size=16, max_blocks=4, bf16=0)
    f.update(over)
    return b2.PagedKVStruct(**f)


def cache4(**over):
    f = dict(pool=FAKE, block_tables=FAKE, seq_lens=FAKE, stride_block=2 * R.tile_bytes(64), num_blocks=8,
             block_size=16, max_blocks=4, bf16=0)
    f.update(over)
    return b2.PagedKV4Struct(**f)


def ref(x):
    return C.byref(x) if x is not None else None


def view(stride=64, data=FAKE, d=1):
    return b2.KVView(data, 4096, stride, 512, d)


def decode4(kv, q=FAKE, ldq=256, blocks=None, listed=0, out=FAKE, batch=1, nq=4, nkv=2, D=64, window=0, sinks=0,
            ws=None):
    return b2.lib().b2_paged_kv4_decode_gqa(q, ldq, ref(kv), blocks, listed, out, batch, nq, nkv, D, window, sinks, ws,
                                            None)


def listed16(kv, blocks=FAKE, listed=2, q=FAKE, ldq=256, out=FAKE, batch=1, nq=4, nkv=2, D=64, ws=None):
    return b2.lib().b2_paged_decode_gqa_blocks(q, ldq, ref(kv), blocks, listed, out, batch, nq, nkv, D, ws, None)


FREQ = (C.c_double * 32)(*([1.0] * 32))


def append(kv, k=None, v=None, q=None, q_out=None, freq=FREQ, rot=64, batch=1, S=1, nq=4, nkv=2, D=64):
    fn = b2.lib().b2_paged_kv4_append if isinstance(kv, b2.PagedKV4Struct) else b2.lib().b2_paged_kv_append
    none = view(data=None)
    rows = b2.AppendStruct(k or view(), v or view(), q or none, q_out or none, C.addressof(freq) if freq else None, None, None,
                           S, batch, nq, nkv, D, rot)
    return fn(ref(kv), ref(rows), None)


def read(kv, k=None, v=None, batch=1, T=1, nkv=2, D=64):
    return b2.lib().b2_paged_kv4_read(ref(kv), ref(k or view()), ref(v or view()), None, batch, T, nkv, D, None)


def bounds(kv, codes=FAKE, scale=FAKE, batch=1, nkv=2, D=64):
    fn = b2.lib().b2_paged_kv4_block_bounds if isinstance(kv, b2.PagedKV4Struct) else b2.lib().b2_paged_block_bounds
    return fn(ref(kv), None, codes, scale, batch, nkv, D, None)


def select(q=FAKE, ldq=256, tables=FAKE, lens=FAKE, num_blocks=8, bs=16, mb=4, codes=FAKE, scale=FAKE, blocks=FAKE, n=2,
           first=1, last=1, batch=1, nq=4, nkv=2, D=64, ws=None):
    what = b2.BlockSelectStruct(q, ldq, tables, lens, codes, scale, blocks, 0, num_blocks, bs, mb, n, first, last, batch, nq,
                                nkv, D)
    return b2.lib().b2_paged_block_select(ref(what), ws, None)


def test_decode_refuses():
    assert decode4(None, batch=0) == 0
    assert decode4(None) == -1
    assert decode4(cache4(), q=None) == -1 and decode4(cache4(), out=None) == -1
    assert decode4(cache4(pool=None)) == -1 and decode4(cache4(block_tables=None)) == -1
    assert decode4(cache4(seq_lens=None)) == -1
    assert decode4(cache4(block_size=0)) == -1 and decode4(cache4(max_blocks=0)) == -1
    assert decode4(cache4(num_blocks=0)) == -1
    assert decode4(cache4(), nq=5) == -1 and decode4(cache4(), window=-1) == -1 and decode4(cache4(), sinks=-1) == -1
    assert decode4(cache4(stride_block=R.tile_bytes(64))) == -1  # blocks would overlap
    assert decode4(cache4(), D=60) == -2 and decode4(cache4(), D=264) == -2
    assert decode4(cache4(block_size=8)) == -2 and decode4(cache4(block_size=24)) == -2
    assert decode4(cache4(stride_block=2 * R.tile_bytes(64) + 8)) == -2 and decode4(cache4(pool=FAKE + 8)) == -2
    assert decode4(cache4(), q=FAKE + 2) == -2 and decode4(cache4(), ldq=260) == -2
    assert decode4(cache4(max_blocks=2 ** 27)) == -2
    assert decode4(cache4(), blocks=FAKE, listed=0) == -1  # an empty list
    assert decode4(cache4(), blocks=FAKE, listed=2, window=4) == -1
    assert decode4(cache4(), blocks=FAKE, listed=2 ** 30) == -2


def test_listed_decode_refuses():
    assert listed16(None, batch=0) == 0
    assert listed16(None) == -1 and listed16(cache16(), blocks=None) == -1 and listed16(cache16(), listed=0) == -1
    assert listed16(cache16(), q=None) == -1 and listed16(cache16(), out=None) == -1
    assert listed16(cache16(), listed=2 ** 30) == -2 and listed16(cache16(), D=60) == -2


@pytest.mark.parametrize("make", [cache16, cache4])
def test_append_refuses(make):
    fn = b2.lib().b2_paged_kv_append if make is cache16 else b2.lib().b2_paged_kv4_append
    assert fn(ref(make()), None, None) == -1 and fn(None, ref(b2.AppendStruct(batch=0, S=1)), None) == 0
    assert append(make(), S=0) == 0 and append(make(), batch=0) == 0
    assert append(make(block_tables=None)) == -1 and append(make(num_blocks=0)) == -1
    assert append(make(), k=view(data=None)) == -1 and append(make(), v=view(data=None)) == -1
    assert append(make(), q=view()) == -1 and append(make(), q_out=view()) == -1  # one without the other
    assert append(make(), q=view(data=None), q_out=view()) == -1
    assert append(make(), q=view(), q_out=view(), nq=0) == -1
    assert append(make(), freq=None) == -1 and append(make(), rot=-8) == -1
    assert append(make(), rot=72) == -2 and append(make(), rot=12) == -2
    assert append(make(), k=view(data=FAKE + 8)) == -2 and append(make(), v=view(stride=60)) == -2
    assert append(make(), k=view(d=2)) == -2
    assert append(make(), q=view(data=FAKE + 4), q_out=view()) == -2
    assert append(make(), q=view(), q_out=view(stride=0)) == -1  # heads written to one place
    assert append(make(), D=60) == -2 and append(make(), S=2 ** 31) == -2 and append(make(), batch=65536) == -2


def test_read_refuses():
    assert read(cache4(), T=0) == 0 and read(None, batch=0) == 0
    assert read(None) == -1 and read(cache4(), k=view(data=None)) == -1
    assert read(cache4(), k=view(d=2)) == -2 and read(cache4(), v=view(stride=4)) == -2
    assert read(cache4(), k=view(stride=0)) == -1 and read(cache4(), v=view(stride=0)) == -1  # heads to one place
    assert read(cache4(), T=2 ** 31) == -2 and read(cache4(), batch=65536) == -2


@pytest.mark.parametrize("make", [cache16, cache4])
def test_bounds_refuse(make):
    assert bounds(make(), batch=0) == 0
    assert bounds(make(), codes=None) == -1 and bounds(make(), scale=None) == -1 and bounds(make(seq_lens=None)) == -1
    assert bounds(make(), codes=FAKE + 8) == -2 and bounds(make(), D=4) == -2
    assert bounds(make(max_blocks=2 ** 20), batch=2 ** 12) == -2


def test_select_refuses():
    assert select(batch=0) == 0 and b2.lib().b2_paged_block_select(None, None, None) == -1
    for name in ("q", "tables", "lens", "codes", "scale", "blocks"):
        assert select(**{name: None}) == -1, name
    assert select(n=0, first=0, last=0) == -1 and select(first=2, last=1) == -1 and select(first=-1) == -1
    assert select(first=2 ** 31 - 1, last=2 ** 31 - 1) == -1
    assert select(nq=5) == -1 and select(num_blocks=0) == -1 and select(bs=0) == -1 and select(mb=0) == -1
    assert select(codes=FAKE + 8) == -2 and select(D=60) == -2 and select(mb=2 ** 27) == -2
    assert select() == -3  # a workspace is needed


def test_sizes():
    f = b2.lib().b2_kv4_tile_bytes
    assert [f(d) for d in (8, 64, 72, 96, 128, 136, 256)] == [R.tile_bytes(d) for d in (8, 64, 72, 96, 128, 136, 256)]
    assert f(0) == 0 and f(60) == 0 and f(264) == 0
    assert b2.paged_block_select_workspace_bytes(2, 3, 5) >= 2 * 3 * 5 * 4
    assert b2.paged_block_select_workspace_bytes(0, 3, 5) == 0
    assert b2.paged_decode_workspace_bytes(2, 8, 2, 128, 4096) >= b2.lib().b2_paged_kv4_decode_workspace_bytes(8, 2, 128)
    assert b2.lib().b2_paged_kv4_decode_workspace_bytes(3, 2, 64) == 0


def cpu_cache4(D=64, nkv=2, blocks=8, bs=16, B=1, mb=4, dtype=torch.float16):
    pool = torch.zeros(blocks, nkv, bs // 16, R.tile_bytes(D), dtype=torch.uint8)
    return b2.PagedKV4(pool, torch.zeros(B, mb, dtype=torch.int32), torch.zeros(B, dtype=torch.int32), D, dtype)


def test_binding_refuses():
    kv = cpu_cache4(bs=32)
    t, n = kv.block_tables, kv.seq_lens
    for bad in (kv.pool.float(), kv.pool[..., :-16], kv.pool[0], kv.pool.transpose(1, 2)):
        with pytest.raises(ValueError):
            b2.PagedKV4(bad, t, n, 64, torch.float16)
    with pytest.raises(ValueError):
        b2.PagedKV4(kv.pool, t.long(), n, 64, torch.float16)
    with pytest.raises(ValueError):
        b2.PagedKV4(kv.pool, t, n, 64, torch.float32)
    with pytest.raises(ValueError):
        b2.PagedKV4(kv.pool, t, n, 60, torch.float16)
    with pytest.raises(ValueError):
        b2.kv4_pool(4, 24, 2, 64)
    for rot in (0, 12, 264):
        with pytest.raises(ValueError):
            b2.Rope(rot)
    with pytest.raises(ValueError):
        b2.Rope(16, inv_freq=[1.0] * 7)
    x = torch.zeros(1, 3, 2, 64, dtype=torch.float16)
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    kv = cpu_cache4()
    bd = b2.BlockBounds(codes=torch.zeros(8, 2, 2, 64, dtype=torch.int8), scale=torch.ones(8, 2))
    # everything fits, but no kernel may read it
    for call in (lambda: b2.paged_kv_append(kv, x, x), lambda: b2.paged_kv_read(kv, x, x),
                 lambda: b2.paged_decode_gqa(q, kv, q.clone()), lambda: b2.paged_block_bounds(kv, bd),
                 lambda: b2.paged_block_select(q, kv, bd, torch.zeros(1, 2, 3, dtype=torch.int32))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError):
        b2.BlockBounds(codes=torch.zeros(8, 2, 2, 64, dtype=torch.int8), scale=torch.ones(8, 3))
    with pytest.raises(ValueError):
        b2.BlockBounds(codes=torch.zeros(8, 2, 3, 64, dtype=torch.int8), scale=torch.ones(8, 2))


def test_binding_refuses_what_does_not_go_together():
    kv = cpu_cache4()
    with pytest.raises(ValueError, match="4 bits"):
        b2.paged_kv_evict(kv, torch.zeros(8, 2, 16), 4, torch.zeros(1, 2, 4, dtype=torch.int32), kv.seq_lens)
    for alone in (dict(codes=torch.zeros(8, 2, 2, 64, dtype=torch.int8)), dict(scale=torch.ones(8, 2))):
        with pytest.raises(ValueError, match="together"):
            b2.BlockBounds(**alone)


def test_rope_frequencies():
    r = b2.Rope(16, theta=500000.0)
    assert list(r.inv_freq) == [500000.0 ** (-2.0 * i / 16) for i in range(8)]
    assert list(b2.Rope(8, inv_freq=torch.arange(4.0)).inv_freq) == [0, 1, 2, 3]


@pytest.mark.parametrize("D", [8, 64, 72, 128, 136, 256])
def test_layout_places_are_all_different(D):
    seen = set()
    for p in range(16):
        for c in range(R.padded(D)):
            for place in (R.k_place, R.v_place):
                at = place(D, p, c)
                assert at not in seen and at[0] < 16 * R.padded(D)
                seen.add(at)
        for g in range(-(-R.padded(D) // 64)):
            for value in (0, 1):
                at = R.scale_place(D, p, g, value)
                assert at % 4 == 0 and 16 * R.padded(D) <= at < R.tile_bytes(D) and (at, 9) not in seen
                seen.add((at, 9))


def test_references_by_hand():
    # codes of a row from 0 to 15 are its numbers; equal numbers have no scale; ties go to even
    codes, s, m = R.quantise(torch.arange(16.0).double())
    assert codes.tolist() == list(range(16)) and s.tolist() == [1] and m.tolist() == [0]
    codes, s, m = R.quantise(torch.full((8,), 3.0).double())
    assert codes.tolist() == [0] * 8 and s.tolist() == [0] and m.tolist() == [3]
    assert R.quantise(torch.tensor([0.0, 0.5, 1.5, 2.5, 15.0]).double())[0].tolist() == [0, 0, 2, 2, 15]
    assert torch.isnan(R.held(torch.tensor([1.0, math.inf]).double())).all()
    x = torch.randn(3, 16, 2, 72, dtype=torch.float64)
    k, v = R.pool_rows(R.fill_pool(x, x + 1), 72)
    assert torch.equal(k, R.held(x)) and torch.equal(v, R.held(x + 1))
    assert (k - x).abs().max() < 0.25
    # a quarter turn
    y = R.rotate(torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0]).double(), torch.tensor(1), [math.pi / 2, 0.0])
    assert torch.allclose(y, torch.tensor([-3.0, 2, 1, 4, 5]).double())
    qo, rows = R.append(None, torch.ones(1, 3, 1, 2), torch.zeros(1, 3, 1, 2), torch.tensor([[4, 9]]), [3], [2], None,
                        [0.0], 2, 8)
    assert [(r[0], r[1]) for r in rows] == [(4, 1)]  # position 1; position 2's block is none
    codes, scale = R.bounds(torch.tensor([[[1.0, -2.0]], [[3.0, 127.0]]]))
    assert scale.tolist() == [1] and codes.tolist() == [[[1, -2], [3, 127]]]
    codes, scale = R.bounds(torch.tensor([[[0.3, 128.0]]]))
    assert scale.tolist() == [2] and codes.tolist() == [[[0, 64], [1, 64]]]
    assert R.bounds(torch.tensor([[[math.nan, 1.0]]]))[1].tolist() == [math.inf]
    assert R.score(torch.tensor([[1.0, -1.0], [1.0, 0.0]]), torch.tensor([[[1, 2], [3, 4]]], dtype=torch.int8),
                   torch.ones(1)).tolist() == [16384 * 3 - 8192 * 2]
    assert R.choose([5, 1, 3, 3, 0, 9], 4, 1, 1) == [0, 2, 3, 5] and R.choose([1, 2], 3, 1, 1) == [0, 1]
    assert R.choose([1.0, 1.0, 1.0], 2, 0, 0) == [0, 1]
