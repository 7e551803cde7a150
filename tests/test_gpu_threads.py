"""Calls from several Python threads at once: the arguments of one are not another's."""
import threading

import pytest
import torch

import b2engine as b2
import kv4_ref as R
from test_gpu_append import empty_cache, gen
from test_gpu_sparse import bare, want_blocks


def test_every_thread_has_room_of_its_own():
    mine, seen = b2._views(), []
    assert b2._views() is mine

    def look():
        seen.append(b2._views())
    threads = [threading.Thread(target=look) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len({at for _, at in seen + [mine]}) == 4


@pytest.mark.gpu
def test_appends_reads_and_choices_at_once(cuda):
    """Four threads, each with a cache, a stream and sizes of its own, start together and call in turn."""
    jobs = []
    for i in range(4):
        bits, D, nkv, B = (4, 16)[i % 2], (64, 128)[i // 2], 1 + i, 2 + i
        kv = empty_cache(bits, B, 8, 16, nkv, D, "fp16", [100] * B, seed=i)
        k, v = (torch.randn(B, 20 + i, nkv, D, generator=gen(10 * i + j), device="cuda").half() for j in range(2))
        sq, skv, bd = bare(20 + i, [900 + 100 * i, 300], nkv, D, 16, "fp16", 2)
        jobs.append((kv, k, v, sq, skv, bd, torch.zeros(2, nkv, 5 + i, dtype=torch.int32, device="cuda"),
                     b2.Workspace(b2.paged_block_select_workspace_bytes(2, nkv, skv.block_tables.shape[1])),
                     torch.zeros_like(k), torch.zeros_like(v), torch.cuda.Stream()))
    torch.cuda.synchronize()
    together, wrong = threading.Barrier(4), []

    def work(kv, k, v, sq, skv, bd, blocks, ws, k_back, v_back, s):
        try:
            together.wait(30)
            for _ in range(200):
                b2.paged_kv_append(kv, k, v, stream=s.cuda_stream)
                if kv.four:
                    b2.paged_kv_read(kv, k_back, v_back, stream=s.cuda_stream)
                b2.paged_block_select(sq, skv, bd, blocks, first=1, last=2, ws=ws, stream=s.cuda_stream)
        except Exception as e:
            wrong.append(e)
    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
    for i, (kv, k, v, sq, skv, bd, blocks, _, k_back, v_back, _) in enumerate(jobs):
        S = k.shape[1]
        pos = torch.arange(100 - S, 100, device="cuda")
        at = kv.block_tables.long()[:, pos // 16], pos % 16
        for new, held, back in ((k, 0, k_back), (v, 1, v_back)):
            if kv.four:
                want = R.held(new.double())
                assert torch.equal(R.pool_rows(kv.pool, kv.head_dim)[held][at], want)
                assert ((back.double() - want).abs() <= 2.0 ** -11 * (1 + 2.0 ** -12) * want.abs() + 2.0 ** -25).all()
            else:
                assert torch.equal((kv.k, kv.v)[held][at], new)
        assert torch.equal(blocks.cpu(), want_blocks(sq, skv, bd, [900 + 100 * i, 300], 5 + i, 1, 2))
