"""One attention layer served from a K/V cache of bounded size.

  python serving-engine_b200/examples/bounded_cache.py

A prompt runs through windowed prefill in chunks while its K/V rows go into a
block pool; the last prompt queries are then run over the pool once more so
that every row has an attention weight; from there on each new token is one
paged decode call that also accumulates weights, and whenever a sequence
reaches its capacity the cache is cut back to its budget: sinks, the most
recent rows, and the rows with the most weight.  Rows keep the position
encoding they were written with, so q and k come in already rotated.  A decode
window counts the rows held: once something above `recent` has been evicted it
reaches further back in tokens than its number says.  Rows are appended in one
launch for all sequences."""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import b2engine as b2  # noqa: E402


def whole_rows(t):
    """t with its rows as an append takes them, contiguous and 16-byte aligned: t itself, or a copy."""
    fits = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and \
        all(n == 1 or step % 8 == 0 for n, step in zip(t.shape[:-1], t.stride()[:-1]))
    return t if fits else t.clone(memory_format=torch.contiguous_format)


class BoundedLayer:
    """K/V pool, block tables, lengths and scores of `batch` sequences of one
    layer.  A sequence holds at most `capacity` rows; eviction leaves
    `budget` of them, `sinks` first and `recent` last ones among them."""

    def __init__(self, batch, nq, nkv, head_dim, capacity, budget, sinks=4, recent=64, window=0, block_size=16,
                 dtype=torch.bfloat16):
        if not 0 < budget < capacity or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError(f"a capacity of {capacity} needs a budget below it that holds the sinks and the recent "
                             f"rows, got {budget}, {sinks} and {recent}")
        blocks = -(-capacity // block_size)
        self.capacity, self.budget, self.sinks, self.recent, self.window = capacity, budget, sinks, recent, window
        self.nq = nq
        k = torch.zeros(batch * blocks, block_size, nkv, head_dim, dtype=dtype, device="cuda")
        tables = torch.randperm(batch * blocks, device="cuda").to(torch.int32).view(batch, blocks)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.kv = b2.PagedKV(k, torch.zeros_like(k), tables, self.seq_lens)
        self.scores = torch.zeros(batch * blocks, nkv, block_size, device="cuda")
        self.kept = torch.empty(batch, nkv, budget, dtype=torch.int32, device="cuda")
        self.ws = b2.Workspace(b2.paged_decode_workspace_bytes(batch, nq, nkv, head_dim, blocks * block_size,
                                                               scored=True))
        self.rows = [0] * batch  # the lengths as the host knows them

    def _append(self, k, v):
        """Rows of new tokens, which seq_lens counts already; rows that are refused leave the layer as it was."""
        try:
            b2.paged_kv_append(self.kv, whole_rows(k), whole_rows(v))
        except Exception:
            self.seq_lens.copy_(torch.tensor(self.rows, dtype=torch.int32))
            raise

    def prefill(self, q, k, v, chunk=512, observe=16):
        """Prompts [B, S, heads, head_dim] of one length S <= capacity;
        returns the attention outputs [B, S, nq, head_dim]."""
        B, S = q.shape[:2]
        if S > self.capacity:
            raise ValueError(f"a prompt of {S} tokens does not fit a capacity of {self.capacity}")
        out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
        for at in range(0, S, chunk):
            end = min(S, at + chunk)
            part = torch.empty(B, end - at, *q.shape[2:], dtype=q.dtype, device="cuda")
            b2.window_prefill_gqa(q[:, at:end], k[:, :end], v[:, :end], part, window=self.window, sinks=self.sinks)
            out[:, at:end] = part
        self.seq_lens.fill_(S)
        self._append(k, v)
        self.rows = [S] * B
        self.scores.zero_()
        # what the last prompt queries look at ranks the rows of the prompt
        probe = torch.empty(B, self.nq, q.shape[3], dtype=q.dtype, device="cuda")
        for i in range(max(0, S - observe), S):
            self.seq_lens.fill_(i + 1)
            b2.paged_decode_gqa(q[:, i], self.kv, probe, window=self.window, sinks=self.sinks, scores=self.scores,
                                ws=self.ws)
        return out

    def decode(self, q, k, v):
        """One new token per sequence: q [B, nq, head_dim], k and v [B, nkv,
        head_dim].  Returns the attention outputs [B, nq, head_dim]."""
        if max(self.rows) == self.capacity:
            self.evict()
        self.seq_lens += 1
        self._append(k[:, None], v[:, None])
        self.rows = [n + 1 for n in self.rows]
        out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
        return b2.paged_decode_gqa(q, self.kv, out, window=self.window, sinks=self.sinks, scores=self.scores,
                                   ws=self.ws)

    def evict(self):
        """Cut every longer sequence back to the budget, in place."""
        b2.paged_kv_evict(self.kv, self.scores, self.budget, self.kept, self.seq_lens, sinks=self.sinks,
                          recent=self.recent)
        self.rows = [min(n, self.budget) for n in self.rows]


def main():
    torch.manual_seed(0)
    B, nq, nkv, D, S, steps = 4, 32, 8, 128, 1500, 200
    layer = BoundedLayer(B, nq, nkv, D, capacity=1600, budget=512, recent=128, window=0)
    new = lambda n, h: torch.randn(B, n, h, D, device="cuda").bfloat16()  # noqa: E731
    layer.prefill(new(S, nq), new(S, nkv), new(S, nkv))
    for _ in range(steps):
        out = layer.decode(new(1, nq)[:, 0], new(1, nkv)[:, 0], new(1, nkv)[:, 0])
    torch.cuda.synchronize()
    print(f"{S} prompt tokens and {steps} new ones; rows held now: {layer.seq_lens.tolist()}; "
          f"|out| {out.float().abs().mean():.4f}")


if __name__ == "__main__":
    main()
