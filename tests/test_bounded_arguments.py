"""Bounded-cache attention without a GPU: arguments at the edges of their types
and tensors that no kernel may be given."""
import pytest
import torch

import b2engine as b2
from test_bounded import prefill


@pytest.mark.parametrize("S,start", [(4, 2 ** 63 - 2), (2 ** 63 - 1, 2 ** 63 - 1), (2 ** 62, 2 ** 62), (2 ** 30, 1),
                                     (1, 2 ** 30)])
def test_prefill_refuses_more_positions_than_it_counts(S, start):
    assert prefill(S=S, start=start) == -2
    assert prefill(S=S, start=start, D=160) == -2


@pytest.mark.parametrize("nbytes", [2 ** 64 - 1, 2 ** 64 - 256, 2 ** 64 - 16384])
def test_workspace_refuses_sizes_that_wrap(nbytes):
    """The lent bytes are rounded up and the counters' follow: cudaErrorMemoryAllocation, not a small workspace."""
    with pytest.raises(b2.B2Error) as e:
        b2.Workspace(nbytes)
    assert e.value.status == 2


def cpu_cache():
    k = torch.zeros(8, 16, 2, 64, dtype=torch.float16)
    return b2.PagedKV(k, k.clone(), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_binding_refuses_tensors_in_host_memory():
    """Everything fits, but no kernel may read it."""
    x = torch.zeros(1, 6, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        b2.window_prefill_gqa(x, x[:, :, :2], x[:, :, :2], torch.zeros_like(x))
    kv = cpu_cache()
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        b2.paged_decode_gqa(q, kv, torch.zeros_like(q))
    with pytest.raises(ValueError, match="GPU"):
        b2.paged_kv_evict(kv, torch.zeros(8, 2, 16), 4, torch.zeros(1, 2, 4, dtype=torch.int32),
                          torch.zeros(1, dtype=torch.int32))
