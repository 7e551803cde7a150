"""Windowed prefill over a K row that holds a NaN: the outputs that see the row
are not finite and the others are as without it, whichever column of a tile the
row is."""
import pytest
import torch

import b2engine as b2
import bounded_ref as R
from test_gpu_bounded import DT, close, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [40, 64, 96, 128, 160])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 2)])
def test_broken_key_shows_in_every_column(cuda, D, dt, window, sinks):
    S = 450
    q, k, v = (randn(gen(97), 1, S, h, D).to(DT[dt]) for h in (2, 1, 1))
    out = torch.empty_like(q)
    want, mag = R.window_prefill(q, k, v, None, window, sinks)
    for j in list(range(8)) + [63, 64, 127, 128, 190, 255, 446, 449]:
        broken = k.clone()
        broken[0, j, 0, D - 1] = float("nan")
        b2.window_prefill_gqa(q, broken, v, out, window=window, sinks=sinks)
        sees = torch.stack([R.visible(i, S, window, sinks)[j] for i in range(S)])
        assert not out[0, sees].isfinite().any(), j
        close(out[0, ~sees], want[0, ~sees], mag[0, ~sees], dt)
