"""Views whose dimensions of one carry any stride: torch leaves them as they
come, and no element is reached through them."""
import pytest
import torch

import b2engine as b2
import bounded_ref as R
from test_gpu_bounded import Cache, close, gen, randn

pytestmark = pytest.mark.gpu


def restride(t, **strides):
    """t with the strides of its dimensions of one replaced (d0=.., d1=..)."""
    st = list(t.stride())
    for name, s in strides.items():
        assert t.shape[int(name[1:])] == 1
        st[int(name[1:])] = s
    return t.as_strided(t.shape, st)


@pytest.mark.parametrize("nq,change", [(4, dict(d0=3)), (4, dict(d0=0)), (1, dict(d1=5)), (1, dict(d0=7, d1=1))])
def test_decode_queries(cuda, nq, change):
    c = Cache(90, [70], 16, 1, 64, "fp16")
    q = randn(gen(91), 1, nq, 64).half()
    out = torch.empty_like(q)
    want, mag, _, _ = R.paged_decode(q, c.k, c.v, c.tables, [70], 0, 0)
    b2.paged_decode_gqa(restride(q, **change), c.kv, out)
    close(out, want, mag, "fp16")


def test_decode_one_head_of_a_transposed_batch(cuda):
    c = Cache(92, [70, 33, 5], 16, 1, 64, "bf16")
    q = randn(gen(93), 1, 3, 64).bfloat16().transpose(0, 1)
    assert q.stride(1) == 3 * 64
    out = torch.empty(3, 1, 64, dtype=q.dtype, device="cuda")
    b2.paged_decode_gqa(q, c.kv, out)
    close(out, *R.paged_decode(q, c.k, c.v, c.tables, [70, 33, 5], 0, 0)[:2], "bf16")


@pytest.mark.parametrize("blocks,bs,nkv,change", [(1, 16, 2, dict(d0=5)), (6, 1, 2, dict(d1=3)), (4, 16, 1, dict(d2=1)),
                                                  (1, 16, 1, dict(d0=1, d2=2))])
def test_pools(cuda, blocks, bs, nkv, change):
    g = gen(94)
    n = blocks * bs - (bs > 1)
    k, v = (randn(g, blocks, bs, nkv, 64).half() for _ in range(2))
    tables = torch.arange(blocks, dtype=torch.int32, device="cuda")[None]
    q = randn(g, 1, 4, 64).half()
    out = torch.empty_like(q)
    want, mag, _, _ = R.paged_decode(q, k, v, tables, [n], 0, 0)
    for kk, vv in ((restride(k, **change), restride(v, **change)), (k, restride(v, **change))):
        kv = b2.PagedKV(kk, vv, tables, torch.tensor([n], dtype=torch.int32, device="cuda"))
        b2.paged_decode_gqa(q, kv, out)
        close(out, want, mag, "fp16")
    scores = torch.rand(blocks, nkv, bs, generator=g, device="cuda")
    kept, new = torch.empty(1, nkv, 3, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    k2, v2, s2, kept2, _ = R.paged_evict(k, v, scores, tables, [n], 3, 1, 1)
    b2.paged_kv_evict(kv, scores, 3, kept, new, sinks=1, recent=1)
    assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(scores, s2) and torch.equal(kept.cpu(), kept2)


@pytest.mark.parametrize("B,S,nq,nkv", [(1, 30, 4, 1), (2, 1, 1, 1), (1, 1, 1, 1)])
@pytest.mark.parametrize("D", [64, 160])
def test_prefill(cuda, B, S, nq, nkv, D):
    g = gen(95)
    q, k, v = (randn(g, B, S, h, D).bfloat16() for h in (nq, nkv, nkv))
    out = torch.empty_like(q)
    odd = lambda t: restride(t, **{f"d{i}": 3 + 2 * i for i in range(3) if t.shape[i] == 1})  # noqa: E731
    b2.window_prefill_gqa(odd(q), odd(k), odd(v), out, window=9, sinks=2)
    close(out, *R.window_prefill(q, k, v, None, 9, 2), "bf16")
