"""Windowed prefill with several pairs of query tiles per SM: what carries over
from one pair to the next (the query buffer, the ring of K and V tiles, the
pairs handed out ahead, the output stage, the accumulators).  Against the 64-bit
references and within the bounds of test_gpu_bounded.py."""
import pytest
import torch

from test_gpu_bounded import prefill_case

pytestmark = pytest.mark.gpu


def pairs(S, start, nq, nkv, lens, B):
    """Pairs of 128-row tiles that hold a token; tiles of one K/V head are paired across its query heads."""
    rows = [min(S, max(0, n - start)) for n in (lens or [start + S] * B)]
    return sum(nkv * -(-(-(-r // 128) * (nq // nkv)) // 2) for r in rows)


@pytest.mark.parametrize("D", [128, 96, 64])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("B,S,start,nq,nkv,lens", [(3, 2000, 0, 36, 4, None), (3, 1990, 0, 32, 8, [1990, 1983, 1111]),
                                                   (2, 1500, 777, 45, 9, [2277, 2000]), (1, 4001, 130, 24, 8, None)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4), (100, 260)])
def test_several_pairs_per_sm(cuda, D, dt, B, S, start, nq, nkv, lens, window, sinks):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert pairs(S, start, nq, nkv, lens, B) > 2 * sms
    prefill_case(100, B, S, start, nq, nkv, D, dt, window, sinks, lens=lens)
