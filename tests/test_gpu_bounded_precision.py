"""Paged decode attention loses nothing to 16-bit weights (bounded_precision.py)."""
import pytest
import torch

import b2engine as b2
import bounded_ref as R
from bounded_precision import bound
from test_gpu_bounded import DT, Cache, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("nq,nkv", [(8, 2), (16, 1)])
def test_weights_are_not_rounded(cuda, D, dt, nq, nkv):
    lens = [40, 100, 64, 700]
    c = Cache(120, lens, 16, nkv, D, dt)
    q = randn(gen(121), len(lens), nq, D).to(DT[dt])
    out = torch.empty_like(q)
    ws = b2.Workspace(b2.paged_decode_workspace_bytes(len(lens), nq, nkv, D, c.tables.shape[1] * 16))
    want, mag, _, _ = R.paged_decode(q, c.k, c.v, c.tables, lens, 0, 0)
    b2.paged_decode_gqa(q, c.kv, out, ws=ws)
    for b, n in enumerate(lens):
        i = torch.arange(n, device="cuda")
        v = c.v[c.tables[b].long()[i // 16], i % 16].double().abs().sum(0).repeat_interleave(nq // nkv, 0)
        over = (out[b].double() - want[b]).abs() - bound(want[b], mag[b], v, n, DT[dt])
        assert over.max() <= 0, (n, float(over.max()))
