"""Windows, sinks and recent counts past what C integers hold: more positions
than any sequence has, not their lower bits."""
import pytest
import torch

import b2engine as b2
import bounded_ref as R
from test_gpu_bounded import Cache, close, gen, randn

pytestmark = pytest.mark.gpu

PAST = [2 ** 31, 2 ** 32 + 5, 2 ** 40, 2 ** 63, 2 ** 64 + 5]


@pytest.mark.parametrize("n", PAST)
def test_windows_and_sinks(cuda, n):
    c = Cache(80, [300, 17], 16, 2, 64, "fp16")
    q = randn(gen(81), 2, 4, 64).half()
    out = torch.empty_like(q)
    x, k, v = (randn(gen(82), 1, m, h, 64).bfloat16() for m, h in ((200, 4), (230, 2), (230, 2)))
    y = torch.empty_like(x)
    for window, sinks in ((n, 0), (n, 3), (n, n), (20, n)):
        want, mag, _, _ = R.paged_decode(q, c.k, c.v, c.tables, c.lens, 0, 0)
        b2.paged_decode_gqa(q, c.kv, out, window=window, sinks=sinks)
        close(out, want, mag, "fp16")
        b2.window_prefill_gqa(x, k, v, y, window=window, sinks=sinks)
        close(y, *R.window_prefill(x, k, v, None, 0, 0), "bf16")


@pytest.mark.parametrize("n", PAST)
def test_negative_counts_are_refused(cuda, n):
    c = Cache(83, [40], 16, 2, 64, "fp16")
    q = randn(gen(84), 1, 4, 64).half()
    x, out = randn(gen(85), 1, 40, 4, 64).half(), torch.empty(1, 40, 4, 64, dtype=torch.float16, device="cuda")
    for args in (dict(window=-n), dict(sinks=-n)):
        with pytest.raises(b2.B2Error) as e:
            b2.paged_decode_gqa(q, c.kv, torch.empty_like(q), **args)
        assert e.value.status == -1
        with pytest.raises(b2.B2Error) as e:
            b2.window_prefill_gqa(x, x[:, :, :2], x[:, :, 2:], out, **args)
        assert e.value.status == -1


@pytest.mark.parametrize("n", PAST + [-m for m in PAST])
def test_eviction_keeps_no_more_than_the_budget(cuda, n):
    c = Cache(86, [40], 16, 2, 64, "fp16")
    kept, new = torch.full((1, 2, 8), -7, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for args in (dict(sinks=n), dict(recent=n), dict(sinks=n, recent=n)):
        with pytest.raises(b2.B2Error) as e:
            b2.paged_kv_evict(c.kv, c.scores, 8, kept, new, **args)
        assert e.value.status == -1
    torch.cuda.synchronize()
    assert (kept == -7).all()
