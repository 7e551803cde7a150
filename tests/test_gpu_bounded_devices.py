"""The bounded-cache binding takes tensors of the current GPU only."""
import pytest
import torch

import b2engine as b2

pytestmark = pytest.mark.gpu


def cache(device, **other):
    at = lambda name: other.get(name, device)  # noqa: E731
    k = torch.zeros(8, 16, 2, 64, dtype=torch.float16, device=at("k"))
    v = torch.zeros(8, 16, 2, 64, dtype=torch.float16, device=at("v"))
    return b2.PagedKV(k, v, torch.zeros(1, 4, dtype=torch.int32, device=at("tables")),
                      torch.ones(1, dtype=torch.int32, device=at("lens")))


def test_one_tensor_in_host_memory(cuda):
    for name in ("k", "v", "tables", "lens"):
        with pytest.raises(ValueError, match="on"):
            cache("cuda", **{name: "cpu"})
    kv = cache("cuda")
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    scores = torch.zeros(8, 2, 16, device="cuda")
    ws = b2.Workspace(b2.paged_decode_workspace_bytes(1, 4, 2, 64, 64, True))
    b2.paged_decode_gqa(q, kv, torch.empty_like(q), scores=scores, ws=ws)
    for args in (dict(q=q.cpu()), dict(out=q.cpu()), dict(scores=scores.cpu()), dict(kv=cache("cpu"))):
        a = dict(q=q, kv=kv, out=torch.empty_like(q), scores=scores, ws=ws) | args
        with pytest.raises(ValueError, match="on"):
            b2.paged_decode_gqa(**a)
    kept, new = torch.empty(1, 2, 4, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    dst = torch.tensor([[7]], dtype=torch.int32, device="cuda")
    b2.paged_kv_evict(kv, scores, 4, kept, new, dst_tables=dst)
    for args in (dict(scores=scores.cpu()), dict(kept=kept.cpu()), dict(new_lens=new.cpu()), dict(dst_tables=dst.cpu())):
        a = dict(kv=kv, scores=scores, budget=4, kept=kept, new_lens=new, dst_tables=dst) | args
        with pytest.raises(ValueError, match="on"):
            b2.paged_kv_evict(**a)
    x = torch.zeros(1, 6, 4, 64, dtype=torch.float16, device="cuda")
    lens = torch.full((1,), 6, dtype=torch.int32, device="cuda")
    b2.window_prefill_gqa(x, x[:, :, :2], x[:, :, 2:], torch.empty_like(x), seq_lens=lens)
    for args in (dict(q=x.cpu()), dict(k=x[:, :, :2].cpu()), dict(v=x[:, :, :2].cpu()), dict(out=x.cpu()),
                 dict(seq_lens=lens.cpu())):
        a = dict(q=x, k=x[:, :, :2], v=x[:, :, 2:], out=torch.empty_like(x), seq_lens=lens) | args
        with pytest.raises(ValueError, match="on"):
            b2.window_prefill_gqa(**a)


def test_tensors_of_another_gpu(cuda, monkeypatch):
    """The current device is another one than the tensors' (told so: one GPU is enough)."""
    kv = cache("cuda")
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    x = torch.zeros(1, 6, 4, 64, dtype=torch.float16, device="cuda")
    scores = torch.zeros(8, 2, 16, device="cuda")
    ws = b2.Workspace(b2.paged_decode_workspace_bytes(1, 4, 2, 64, 64))
    ws.device += 1
    with pytest.raises(ValueError, match="workspace"):
        b2.paged_decode_gqa(q, kv, torch.empty_like(q), ws=ws)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        b2.paged_decode_gqa(q, kv, torch.empty_like(q))
    with pytest.raises(ValueError, match="current device"):
        b2.window_prefill_gqa(x, x[:, :, :2], x[:, :, 2:], torch.empty_like(x))
    with pytest.raises(ValueError, match="current device"):
        b2.paged_kv_evict(kv, scores, 4, torch.empty(1, 2, 4, dtype=torch.int32, device="cuda"), kv.seq_lens)
