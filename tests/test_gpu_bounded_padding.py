"""Paged decode where head_dim is below the 64, 128 or 256 elements a row takes
in shared memory: the rest of each row is multiplied by zero queries and has to
be zero itself, whatever the kernel before left in shared memory.  Against the
64-bit references and within the bounds of test_gpu_bounded.py."""
import pytest
import torch

import b2engine as b2
import bounded_ref as R
from test_gpu_bounded import DT, Cache, close, gen, randn

pytestmark = pytest.mark.gpu


class Nans:
    """A decode at a head_dim without such a rest over rows that are all NaN: every CTA of its grid fills its whole
    ring with them."""

    def __init__(self, D, dt):
        B, L, bs, nkv = 32, 4096, 16, 8
        pool = torch.full((L // bs, bs, nkv, D), float("nan"), dtype=DT[dt], device="cuda")
        tables = torch.arange(L // bs, dtype=torch.int32, device="cuda").expand(B, -1).contiguous()
        self.kv = b2.PagedKV(pool, pool, tables, torch.full((B,), L, dtype=torch.int32, device="cuda"))
        self.q = torch.ones(B, nkv, D, dtype=DT[dt], device="cuda")
        self.out = torch.zeros_like(self.q)
        self.ws = b2.Workspace(b2.paged_decode_workspace_bytes(B, nkv, nkv, D, L))

    def run(self):
        b2.paged_decode_gqa(self.q, self.kv, self.out, ws=self.ws)


@pytest.mark.parametrize("D,whole", [(8, 64), (40, 64), (72, 128), (80, 128), (96, 128), (120, 128), (136, 256), (192, 256)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_rest_of_a_row_is_zero(cuda, D, whole, dt):
    """Batches up to 32 and above, one and several segments per CTA, with and without a workspace."""
    nans = Nans(whole, dt)
    for lens, nq, nkv, bs, layout, window, ws in (
            ([700], 4, 2, 16, "slot", 0, True), ([1], 16, 1, 16, "slot", 0, True),
            ([300 - 9 * b for b in range(32)], 24, 12, 16, "slot", 0, True),
            ([200 - 4 * b for b in range(33)], 12, 3, 16, "slot", 0, True),
            ([900, 40, 333], 8, 2, 16, "head", 100, True), ([900, 40, 333], 8, 2, 5, "slot", 0, False)):
        c = Cache(70, lens, bs, nkv, D, dt, layout)
        q = randn(gen(71), len(lens), nq, D).to(DT[dt])
        w = b2.Workspace(b2.paged_decode_workspace_bytes(len(lens), nq, nkv, D, c.tables.shape[1] * bs, True))
        for scored in (False, True) if ws else (False,):
            before = c.scores.clone()
            want, mag, new, add = R.paged_decode(q, c.k, c.v, c.tables, lens, window, 5, before)
            out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
            torch.cuda.synchronize()
            nans.run()
            b2.paged_decode_gqa(q, c.kv, out, window=window, sinks=5, scores=c.scores if scored else None,
                                ws=w if ws else None)
            close(out, want, mag, dt)
            if scored:
                assert ((c.scores.double() - new).abs() <= 6e-5 * add + 2.0 ** -23 * new.abs()).all()
        assert nans.out.isnan().all()
