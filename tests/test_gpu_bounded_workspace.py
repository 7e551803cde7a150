"""Making a workspace while the caller's streams are busy."""
import pytest
import torch

import b2engine as b2

pytestmark = pytest.mark.gpu


def test_workspace_does_not_wait_for_queued_work(cuda):
    b2.Workspace(1 << 20)
    x = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    y = torch.matmul(x, x)
    torch.cuda.synchronize()
    for _ in range(300):  # some 200 ms of the default stream
        torch.matmul(x, x, out=y)
    done = torch.cuda.Event()
    done.record()
    ws = b2.Workspace(1 << 20)
    assert not done.query()
    assert ws.nbytes == 1 << 20
    torch.cuda.synchronize()
