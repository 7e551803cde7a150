"""Bounded-cache attention operators without a GPU: what they refuse, and the
64-bit references of the GPU tests against small cases worked by hand."""
import ctypes as C
import math

import pytest
import torch

import b2engine as b2
import bounded_ref as R

FAKE = 1 << 20  # a non-null, 16-byte-aligned address that nothing reads


def view(stride=64):
    return b2.KVView(FAKE, 4096, stride, 512, 1)


def cache(**over):
    f = dict(k=FAKE, v=FAKE, block_tables=FAKE, seq_lens=FAKE, stride_block=16 * 2 * 64, stride_slot=2 * 64,
             stride_head=64, num_blocks=8, block_size=16, max_blocks=4, bf16=0)
    f.update(over)
    return b2.PagedKVStruct(**f)


def prefill(q=None, S=4, start=0, nq=4, nkv=2, D=64, batch=1, window=0, sinks=0, out=FAKE):
    v = view()
    return b2.lib().b2_window_prefill_gqa(q if q is not None else v, v, v, out, None, S, start, nq, nkv, D, batch,
                                          window, sinks, 0, None)


def decode(kv, q=FAKE, ldq=256, out=FAKE, scores=None, batch=1, nq=4, nkv=2, D=64, window=0, sinks=0, ws=None):
    return b2.lib().b2_paged_decode_gqa(q, ldq, C.byref(kv) if kv is not None else None, out, scores, batch, nq, nkv,
                                        D, window, sinks, ws, None)


def evict(kv, scores=FAKE, dst=None, mdb=0, batch=1, nkv=2, D=64, budget=32, sinks=4, recent=4, kept=FAKE, new=FAKE):
    return b2.lib().b2_paged_kv_evict(C.byref(kv) if kv is not None else None, scores, dst, mdb, batch, nkv, D, budget,
                                      sinks, recent, kept, new, None)


def test_prefill_refuses():
    assert prefill(S=0) == 0 and prefill(batch=0) == 0  # nothing to do
    assert prefill(q=b2.KVView()) == -1
    assert prefill(out=None) == -1
    assert prefill(nq=3) == -1  # not a multiple of the K/V heads
    assert prefill(window=-1) == -1 and prefill(sinks=-1) == -1 and prefill(start=-1) == -1
    assert prefill(D=264) == -2
    assert prefill(q=b2.KVView(FAKE, 4096, 64, 512, 2)) == -2  # rows must be contiguous


def test_decode_refuses():
    assert decode(None, batch=0) == 0
    assert decode(None) == -1
    assert decode(cache(), q=None) == -1 and decode(cache(), out=None) == -1
    assert decode(cache(k=None)) == -1 and decode(cache(block_tables=None)) == -1
    assert decode(cache(seq_lens=None)) == -1
    assert decode(cache(block_size=0)) == -1 and decode(cache(max_blocks=0)) == -1 and decode(cache(num_blocks=0)) == -1
    assert decode(cache(), nq=5) == -1
    assert decode(cache(), window=-1) == -1 and decode(cache(), sinks=-1) == -1
    assert decode(cache(), D=60) == -2 and decode(cache(), D=264) == -2
    assert decode(cache(stride_slot=100)) == -2 and decode(cache(k=FAKE + 8)) == -2
    assert decode(cache(), q=FAKE + 2) == -2 and decode(cache(), ldq=260) == -2
    assert decode(cache(), scores=FAKE) == -3  # weights need a workspace


def test_evict_refuses():
    assert evict(None, batch=0) == 0
    assert evict(None) == -1
    assert evict(cache(), scores=None) == -1 and evict(cache(), kept=None) == -1 and evict(cache(), new=None) == -1
    assert evict(cache(), budget=0) == -1
    assert evict(cache(), sinks=20, recent=13) == -1  # more than the budget stays in any case
    assert evict(cache(), dst=FAKE, mdb=1) == -1  # 16 positions cannot hold a budget of 32
    assert evict(cache(), D=60) == -2 and evict(cache(stride_head=60)) == -2


def test_binding_refuses_tensors_that_do_not_fit():
    k = torch.zeros(8, 16, 2, 64, dtype=torch.float16)
    t = torch.zeros(1, 4, dtype=torch.int32)
    n = torch.zeros(1, dtype=torch.int32)
    kv = b2.PagedKV(k, k, t, n)
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        b2.PagedKV(k, k[:4], t, n)
    with pytest.raises(ValueError):
        b2.PagedKV(k, k, t.long(), n)
    with pytest.raises(ValueError):
        b2.PagedKV(k.float(), k.float(), t, n)
    with pytest.raises(ValueError):
        b2.paged_decode_gqa(q.bfloat16(), kv, q.bfloat16())
    with pytest.raises(ValueError):
        b2.paged_decode_gqa(q, kv, q.transpose(1, 2))
    with pytest.raises(ValueError):
        b2.paged_decode_gqa(q, kv, q, scores=torch.zeros(8, 2, 16, dtype=torch.float64))
    with pytest.raises(ValueError):
        b2.paged_kv_evict(kv, torch.zeros(8, 2, 16), 4, torch.zeros(1, 2, 5, dtype=torch.int32), n)
    x = torch.zeros(1, 6, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        b2.window_prefill_gqa(x, x[:, :4, :2], x[:, :4, :2], x)  # fewer keys than queries
    with pytest.raises(ValueError):
        b2.window_prefill_gqa(x, x[:, :, :2].bfloat16(), x[:, :, :2].bfloat16(), x)


def test_workspace_sizes():
    f = b2.paged_decode_workspace_bytes
    assert f(0, 4, 2, 64, 100) == 0 and f(1, 3, 2, 64, 100) == 0
    assert f(2, 4, 2, 64, 4096, scored=True) >= max(1, f(2, 4, 2, 64, 4096))


def test_references_by_hand():
    assert R.visible(5, 8, 2, 1).tolist() == [True, False, False, False, True, True, False, False]
    assert R.visible(5, 6, 0, 0).all()
    # equal keys: the output is the mean of the visible values
    k = torch.ones(1, 6, 1, 8)
    v = torch.arange(6.0).view(1, 6, 1, 1).expand(1, 6, 1, 8)
    out, mag = R.window_prefill(torch.ones(1, 6, 1, 8), k, v, None, 2, 1)
    assert torch.allclose(out[0, :, 0, 0], torch.tensor([0, 0.5, 1, 5 / 3, 7 / 3, 3]).double())
    out, _ = R.window_prefill(torch.ones(1, 6, 1, 8), k, v, [3], 0, 0)
    assert out[0, 3:].abs().max() == 0
    assert R.evict_choice([0, 5, 1, 5, math.nan, 2, 0], 7, 4, 1, 1) == [0, 1, 4, 6]
    assert R.evict_choice([0, 5, 1, 5, 1, 2, 0], 7, 3, 0, 0) == [1, 3, 5]
    assert R.evict_choice([1, 1, 1, 1], 4, 2, 0, 1) == [0, 3]
    pool = torch.arange(4.0).view(4, 1, 1, 1).expand(4, 1, 1, 8).contiguous()
    sc = torch.tensor([3.0, 1, 2, 0]).view(4, 1, 1)
    k2, _, s2, kept, new = R.paged_evict(pool, pool, sc, torch.tensor([[0, 1, 2, 3]]), [4], 2, 0, 0)
    assert kept.tolist() == [[[0, 2]]] and new.tolist() == [2] and k2[:2, 0, 0, 0].tolist() == [0, 2]
    assert s2[:, 0, 0].tolist() == [3, 2, 2, 0]
