"""The choice of blocks where its border falls among blocks that rank above every
number: their scale is a NaN, as one that was never written may be.  They are
listed lowest first, and the first and last blocks stay in any case."""
import math

import pytest
import torch

import kv4_ref as R
from test_gpu_sparse import bare, chosen

pytestmark = pytest.mark.gpu


def want(q, kv, bd, L, n, first, last):
    """A NaN above an infinity, above every number; of equal ones the lowest block."""
    nb, out = -(-L // kv.block_size), []
    g = q.shape[1] // kv.nkv
    for h in range(kv.nkv):
        s = R.score(q[0, h * g:(h + 1) * g].cpu(), bd.codes[:nb, h].cpu(), bd.scale[:nb, h].cpu()).tolist()
        rank = lambda i: (-2, 0, i) if math.isnan(s[i]) else (-1, 0, i) if s[i] == math.inf else (0, -s[i], i)  # noqa: E731
        mid = sorted(range(first, nb - last), key=rank)[: n - first - last]
        out.append(sorted(list(range(first)) + mid + list(range(nb - last, nb))))
    return torch.tensor(out, dtype=torch.int32)[None]


@pytest.mark.parametrize("L", [300, 1600, 5000, 80000, 200000])
@pytest.mark.parametrize("every", [5, 37])
@pytest.mark.parametrize("infinite", [False, True])
def test_scales_that_are_no_numbers(cuda, L, every, infinite):
    """19 blocks to 12500 (more than the choice keeps in registers); fewer such blocks than are chosen, and up to 2500."""
    q, kv, bd = bare(7, [L], 2, 64, 16, "bf16", 4)
    kv.block_tables.copy_(torch.arange(-(-L // 16), device="cuda")[None])
    bd.scale[1::every] = math.nan
    if infinite:
        bd.scale[2::every] = math.inf
    for n, first, last in ((6, 1, 2), (3, 1, 1), (5, 0, 5), (12, 0, 0)):
        assert torch.equal(chosen(q, kv, bd, n, first, last), want(q, kv, bd, L, n, first, last)), (n, first, last)
