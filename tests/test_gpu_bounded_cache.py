"""The bounded-cache example: windowed prefill, paged decode with weights and
eviction as one layer, every call against the 64-bit references on what the
layer holds at that moment."""
import os
import subprocess
import sys

import pytest
import torch

import bounded_ref as R
from test_gpu_bounded import close

EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "serving-engine_b200", "examples")
sys.path.insert(0, EXAMPLES)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,dt", [(0, "bf16"), (48, "fp16")])
def test_layer_against_references(cuda, window, dt):
    from bounded_cache import BoundedLayer
    torch.manual_seed(7)
    B, nq, nkv, D, S = 2, 4, 2, 64, 150
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}[dt]
    lay = BoundedLayer(B, nq, nkv, D, capacity=160, budget=96, sinks=3, recent=20, window=window, dtype=dtype)
    new = lambda n, h: torch.randn(B, n, h, D, device="cuda").to(dtype)  # noqa: E731
    q, k, v = new(S, nq), new(S, nkv), new(S, nkv)
    out = lay.prefill(q, k, v, chunk=64, observe=8)
    close(out, *R.window_prefill(q, k, v, None, window, 3), dt)
    # the 8 probes left each of its weights: every sequence's scores sum to 8 per query head
    assert (lay.scores.double().sum() - B * nq * 8).abs() < 1e-3
    evictions = 0
    for _ in range(90):
        if max(lay.rows) == lay.capacity:
            want = R.paged_evict(lay.kv.k, lay.kv.v, lay.scores, lay.kv.block_tables, lay.rows, 96, 3, 20)
            lay.evict()
            evictions += 1
            assert torch.equal(lay.kept.cpu(), want[3]) and lay.seq_lens.tolist() == want[4].tolist() == lay.rows
            assert torch.equal(lay.kv.k, want[0]) and torch.equal(lay.kv.v, want[1]) and torch.equal(lay.scores, want[2])
        q1, before = new(1, nq)[:, 0], lay.scores.clone()
        got = lay.decode(q1, new(1, nkv)[:, 0], new(1, nkv)[:, 0])
        o, mag, score, add = R.paged_decode(q1, lay.kv.k, lay.kv.v, lay.kv.block_tables, lay.rows, window, 3, before)
        close(got, o, mag, dt)
        assert ((lay.scores.double() - score).abs() <= 6e-5 * add + 2.0 ** -23 * score.abs()).all()
    assert evictions == 2


def test_example_runs(cuda):
    r = subprocess.run([sys.executable, os.path.join(EXAMPLES, "bounded_cache.py")], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr
    assert "rows held now" in r.stdout
