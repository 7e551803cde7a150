"""The operators of the 4-bit paged cache and of sparse decoding, as cases to
time and compare.

Long-context serving that reads few bytes per token:

  append  rotates the queries and keys of new tokens and writes their K and V
          rows into a paged cache, of 16-bit rows or of 4-bit ones; after a
          4-bit append the rows are read back as 16-bit ones, as the attention
          of a prompt's next chunk needs them;
  attend  GQA attention of one new token per sequence over a paged cache held
          in 4 bits, whole or with window and sinks;
  bounds  channel-wise lower and upper bounds, in 8 bits, of the keys of the
          blocks that the newest positions touch;
  sparse  the choice of `n` blocks per (sequence, K/V head) by an upper bound
          of their logits, and the attention of one new token per sequence
          over the chosen blocks alone, 4-bit or 16-bit.

`own` False computes them with elementary torch operations; `own` True calls
serving-engine_b200 (b2engine).

The 4-bit cache.  pool is uint8 [num_blocks, nkv, block_size / 16, tile]: 16
positions of one K/V head are a tile of 16 Dp bytes of codes and 128 NG of
scales, Dp the head dim rounded up to 64, 96, 128, 192 or 256, NG = ceil(Dp /
64).  Channels go in groups of 64; a group of a row holds x as m + u s with u in
0..15, m = half(min x), s = half((max x - m) / 15), u = (x - m) / s rounded to
even and clamped.  In a tile:
  K codes  row p at p Dp / 2: words (8 channels, channel 8 j + e at bits 4 e of
           word j) in the order j % 4, then j / 4;
  V codes  at 8 Dp: channels 32 x + 4 r + i (i at bits 4 i) of position p are
           16 bits at ((32 x + 4 r + p % 8 / 2) 4 + p / 8 2 + p % 2) 2;
  K scales at 16 Dp: (s, m) halves of group g of position p at
           ((p % 8 / 2 4 + p / 8 2 + p % 2) NG + g) 4; V scales after them."""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one token of a chat turn of a small model (14/2 heads of 64) into a 16-bit cache: what a call costs
        dict(name="append_one", op="append", bits=16, B=1, S=1, L=301, bs=16, nq=14, nkv=2, D=64, rot=64, theta=1e6,
             dtype="fp16", ragged=0.0, shift=0),
        # one token each of a full batch of long sequences, some of them cut back earlier, into a 4-bit cache
        dict(name="append_batch", op="append", bits=4, B=32, S=1, L=32768, bs=16, nq=32, nkv=8, D=128, rot=128,
             theta=5e5, dtype="bf16", ragged=0.6, shift=70001),
        # prompts of different lengths, padded to the longest, into a 16-bit cache
        dict(name="append_ragged", op="append", bits=16, B=4, S=1001, L=1001, bs=16, nq=12, nkv=4, D=128, rot=128,
             theta=1e4, dtype="fp16", ragged=0.6, shift=0),
        # a long prompt in one call into a 4-bit cache
        dict(name="append_prompt", op="append", bits=4, B=1, S=8192, L=8192, bs=64, nq=32, nkv=8, D=128, rot=128,
             theta=5e5, dtype="bf16", ragged=0.0, shift=0),
        # one chat turn of a small model: the latency of a step
        dict(name="attend_single", op="attend", B=1, L=301, bs=16, nq=14, nkv=2, D=64, dtype="fp16", window=0,
             sinks=0, ragged=0.0),
        # an ordinary batch
        dict(name="attend_batch", op="attend", B=8, L=4096, bs=16, nq=32, nkv=8, D=128, dtype="bf16", window=0,
             sinks=0, ragged=0.5),
        # a full batch of long contexts, everything read
        dict(name="attend_full", op="attend", B=32, L=32768, bs=16, nq=32, nkv=8, D=128, dtype="bf16", window=0,
             sinks=0, ragged=0.3),
        # one sequence with a very long context at 70B widths
        dict(name="attend_long", op="attend", B=1, L=131001, bs=64, nq=64, nkv=8, D=128, dtype="fp16", window=0,
             sinks=0, ragged=0.0),
        # the bounds of the newest block of each sequence of a batch, after a decode step
        dict(name="bounds_step", op="bounds", bits=4, B=8, L=4096, new=1, bs=64, nkv=8, D=128, dtype="bf16",
             ragged=0.5),
        # the bounds of a whole prompt's blocks
        dict(name="bounds_prompt", op="bounds", bits=16, B=1, L=32768, new=32768, bs=64, nkv=8, D=128, dtype="fp16",
             ragged=0.0),
        # a full batch of long contexts reading 128 blocks of 16 of their 4-bit caches
        dict(name="sparse_batch", op="sparse", bits=4, B=32, L=32768, bs=16, nq=32, nkv=8, D=128, dtype="bf16", n=128,
             first=1, last=2, ragged=0.3),
        # one sequence with a very long context at 70B widths reading 64 blocks of 32 of a 16-bit cache
        dict(name="sparse_long", op="sparse", bits=16, B=1, L=131001, bs=32, nq=64, nkv=8, D=128, dtype="fp16", n=64,
             first=1, last=2, ragged=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sparse", "bounds"])
    nq, nkv, D = rng.choice([(14, 2, 64), (32, 8, 128), (64, 8, 128), (8, 8, 64), (12, 4, 128), (16, 2, 80),
                             (32, 32, 128), (8, 1, 96), (16, 1, 128), (8, 4, 256)])
    c = dict(op=op, B=_log(rng, 1, 32), bs=rng.choice([16, 16, 16, 32, 64, 128]), nkv=nkv, D=D,
             dtype=rng.choice(["fp16", "bf16"]), ragged=rng.choice([0.0, 0.3, 0.9]))
    wide = nkv * D
    if op == "append":
        S = rng.choice([1, 1, _log(rng, 1, 8192)])
        c.update(bits=rng.choice([4, 16]), nq=nq, S=max(1, min(S, 8192 * 6144 // (c["B"] * (nq + 2 * nkv) * D))),
                 rot=rng.choice([D, D, D // 2]), theta=rng.choice([1e4, 5e5, 1e6]),
                 shift=rng.choice([0, 0, rng.randrange(1, 200000)]))
        c["L"] = c["S"] + rng.choice([0, min(_log(rng, 1, 16384), 32 * 8192 * 1024 // (c["B"] * wide))])
        return c
    L = max(1, min(_log(rng, 1, 131072), 32 * 27000 * 1024 // (c["B"] * wide)))
    if op == "attend":
        c.update(nq=nq, L=L, window=rng.choice([0, 0, _log(rng, 1, 8192)]), sinks=rng.choice([0, 1, 4, 4, 64, 133]))
    elif op == "sparse":
        n, first = _log(rng, 1, 256), rng.choice([0, 1, 1, 4])
        first = min(first, n)
        c.update(bits=rng.choice([4, 16]), nq=nq, L=L, n=n, first=first, last=min(n - first, rng.choice([0, 1, 2])))
        if c["bits"] == 16:
            c["L"] = max(1, min(L, 8 * 27000 * 1024 // (c["B"] * wide)))
    else:
        L = max(1, min(L, 32768 * 1024 // (c["B"] * wide)))
        c.update(bits=rng.choice([4, 16]), L=L, new=rng.choice([1, 1, L, rng.randrange(1, L + 1)]))
    return c


def _lens(case):
    """Length of each sequence: the longest first, the others up to `ragged` shorter."""
    L = case["L"]
    return [max(1, L - int(L * case["ragged"] * ((b * 0.6180339887) % 1.0))) for b in range(case["B"])]


def _counts(case, lens):
    """New tokens of each sequence of an append."""
    S = case["S"]
    return [min(n, max(1, S - int(S * case["ragged"] * ((b * 0.6180339887) % 1.0)))) for b, n in enumerate(lens)]


def _padded(D):
    return next(p for p in (64, 96, 128, 192, 256) if D <= p)


def _row4(D):
    """Bytes of a K or V row of one head in the 4-bit cache, without padding."""
    return D // 2 + 4 * -(-D // 64)


def work(case):
    op, D, nkv, B, bs = case["op"], case["D"], case["nkv"], case["B"], case["bs"]
    lens = _lens(case)
    blocks = sum(-(-n // bs) for n in lens)
    if op == "append":
        t, nq = sum(_counts(case, lens)), case["nq"]
        touched = sum(-(-n // bs) - (n - c) // bs for n, c in zip(lens, _counts(case, lens)))
        back = t * nkv * (2 * _row4(D) + 4 * D) if case["bits"] == 4 else 0
        row = _row4(D) if case["bits"] == 4 else 2 * D
        return {"bytes": t * (4 * nq * D + 4 * nkv * D + 2 * nkv * row) + back + 4 * touched + 8 * B,
                "flops": 3 * t * (nq + nkv) * case["rot"] + 8 * t * nkv * D * (case["bits"] == 4)}
    if op == "attend":
        nq, W, K = case["nq"], case["window"], case["sinks"]
        vis = sum(n if W == 0 or W >= n else W + min(K, n - W) for n in lens)
        return {"bytes": 2 * vis * nkv * _row4(D) + 4 * B * nq * D + 4 * (vis // bs + B), "flops": 4 * D * nq * vis}
    if op == "bounds":
        touched = sum(-(-n // bs) - max(0, n - case["new"]) // bs for n in lens)
        rows = sum(n - max(0, n - case["new"]) // bs * bs for n in lens)
        row = _row4(D) if case["bits"] == 4 else 2 * D
        return {"bytes": rows * nkv * row + touched * nkv * (2 * D + 4) + 4 * touched + 4 * B, "flops": 2 * rows * nkv * D}
    nq, n = case["nq"], case["n"]
    seen = sum(min(m, n * bs) for m in lens)
    row = 2 * _row4(D) if case["bits"] == 4 else 4 * D
    return {"bytes": blocks * nkv * (2 * D + 4) + 4 * blocks + 4 * B * nkv * n + seen * nkv * row + 4 * B * nq * D,
            "flops": 4 * blocks * nkv * D + 4 * D * nq * seen}


# ---------------------------------------------------------------------------
# the 4-bit layout
# ---------------------------------------------------------------------------

def _quantise(x):
    """x [..., D] in 32 or 64 bits: codes uint8 [..., Dp], scales and minima half [..., NG]."""
    D = x.shape[-1]
    Dp = _padded(D)
    ng = -(-Dp // 64)
    pad = ng * 64 - D
    lo = torch.nn.functional.pad(x, (0, pad), value=math.inf).unflatten(-1, (ng, 64))
    hi = torch.nn.functional.pad(x, (0, pad), value=-math.inf).unflatten(-1, (ng, 64)).amax(-1)
    m = lo.amin(-1).clamp(-65504.0, 65504.0).half()
    s = ((hi - m.to(x.dtype)) / 15).clamp(0.0, 65504.0).half()
    sx, mx = s.to(x.dtype)[..., None], m.to(x.dtype)[..., None]
    u = torch.where(sx > 0, (lo - mx) / torch.where(sx > 0, sx, 1.0), 0.0)
    u = u.nan_to_num(posinf=0.0).round_().clamp_(0.0, 15.0).to(torch.uint8).flatten(-2)[..., :Dp]
    u[..., D:] = 0
    return u, s, m


def _pack(ku, ks, km, vu, vs, vm):
    """Codes [..., 16, Dp], scales and minima [..., 16, NG] of K and V: tiles uint8 [..., tile]."""
    lead, Dp = ku.shape[:-2], ku.shape[-1]
    at = lambda *d: tuple(range(len(lead))) + tuple(len(lead) + i for i in d)  # noqa: E731
    k = ku[..., 0::2] | ku[..., 1::2] << 4
    k = k.reshape(*lead, 16, Dp // 32, 4, 4).permute(at(0, 2, 1, 3)).reshape(*lead, 8 * Dp)
    v = vu[..., 0::2] | vu[..., 1::2] << 4
    v = v.reshape(*lead, 2, 4, 2, Dp // 32, 8, 2).permute(at(3, 4, 1, 0, 2, 5)).reshape(*lead, 8 * Dp)
    out = [k, v]
    for s, m in ((ks, km), (vs, vm)):
        x = torch.stack((s, m), -1).reshape(*lead, 2, 4, 2, -1).permute(at(1, 0, 2, 3))
        out.append(x.reshape(*lead, -1).contiguous().view(torch.uint8))
    return torch.cat(out, -1)


def _unpack(tiles, D):
    """Tiles uint8 [..., tile]: K and V values in 32 bits, [..., 16, D]."""
    lead, Dp = tiles.shape[:-1], _padded(D)
    ng = -(-Dp // 64)
    at = lambda *d: tuple(range(len(lead))) + tuple(len(lead) + i for i in d)  # noqa: E731
    nib = lambda x: torch.stack((x & 15, x >> 4), -1)  # noqa: E731
    k = nib(tiles[..., : 8 * Dp]).reshape(*lead, 16, 4, Dp // 32, 8).permute(at(0, 2, 1, 3)).reshape(*lead, 16, Dp)
    v = nib(tiles[..., 8 * Dp: 16 * Dp]).reshape(*lead, Dp // 32, 8, 4, 2, 2, 4).permute(at(3, 2, 4, 0, 1, 5))
    v = v.reshape(*lead, 16, Dp)
    meta = tiles[..., 16 * Dp:].contiguous().view(torch.float16).reshape(*lead, 2, 4, 2, 2, ng, 2)
    meta = meta.permute(at(0, 2, 1, 3, 4, 5)).reshape(*lead, 2, 16, ng, 1, 2).expand(*lead, 2, 16, ng, 64, 2)
    meta = meta.reshape(*lead, 2, 16, ng * 64, 2)[..., :D, :].float()
    return (k[..., :D].float() * meta[..., 0, :, :, 0] + meta[..., 0, :, :, 1],
            v[..., :D].float() * meta[..., 1, :, :, 0] + meta[..., 1, :, :, 1])


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _b2():
    path = os.path.join(os.getcwd(), "serving-engine_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b2engine
    return b2engine


def _cache(case, gen, lens, toward):
    """A paged cache of the case's sequences: keys of a block share a direction, the first four tokens' keys are
    pushed along `toward`, and what lies past a sequence's end was never written (NaN)."""
    B, bs, nkv, D, dt = case["B"], case["bs"], case["nkv"], case["D"], DTYPES[case["dtype"]]
    mb = -(-case["L"] // bs)
    n = B * mb
    tables = torch.randperm(n, generator=gen, device="cuda").to(torch.int32).view(B, mb)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    first = torch.zeros(n, dtype=torch.bool, device="cuda")
    first[tables[:, 0].long()] = True
    left = torch.zeros(n, dtype=torch.long, device="cuda")  # rows that a block holds
    left[tables.long()] = (seq_lens[:, None] - torch.arange(mb, device="cuda") * bs).clamp(0, bs)
    held = torch.arange(bs, device="cuda") < left[:, None]
    four = case.get("bits", 4) == 4
    if four:
        Dp = _padded(D)
        tile = 16 * Dp + 128 * -(-Dp // 64)
        pool = torch.empty(n, nkv, bs // 16, tile, dtype=torch.uint8, device="cuda")
    else:
        k = torch.empty(n, bs, nkv, D, dtype=dt, device="cuda")
        v = torch.empty_like(k)
    step = max(1, (1 << 26) // (bs * nkv * D))
    for i in range(0, n, step):
        j = min(n, i + step)
        kk = torch.randn(j - i, bs, nkv, D, generator=gen, device="cuda")
        kk += 0.5 * torch.randn(j - i, 1, nkv, D, generator=gen, device="cuda")
        kk[:, :4] += 0.7 * toward * first[i:j, None, None, None]
        vv = torch.randn(j - i, bs, nkv, D, generator=gen, device="cuda")
        gone = ~held[i:j, :, None, None]
        if not four:
            k[i:j] = kk.masked_fill_(gone, math.nan).to(dt)
            v[i:j] = vv.masked_fill_(gone, math.nan).to(dt)
            continue
        parts = []
        for x in (kk, vv):
            u, s, m = _quantise(x.transpose(1, 2).reshape(j - i, nkv, bs // 16, 16, D))
            none = gone.reshape(j - i, 1, bs // 16, 16, 1)
            parts += [u, s.masked_fill_(none, math.nan), m.masked_fill_(none, math.nan)]
        pool[i:j] = _pack(*parts)
    st = dict(tables=tables, seq_lens=seq_lens)
    if four:
        st["pool"] = pool
        if own:
            st["kv"] = _b2().PagedKV4(pool, tables, seq_lens, D, dt)
    else:
        st.update(k=k, v=v)
        if own:
            st["kv"] = _b2().PagedKV(k, v, tables, seq_lens)
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, B, nkv, D, dt = case["op"], case["B"], case["nkv"], case["D"], DTYPES[case["dtype"]]
    lens = _lens(case)
    toward = torch.randint(0, 2, (nkv, D), generator=gen, device="cuda").float() * 2 - 1
    st = dict(case)
    if op == "append":
        S, nq = case["S"], case["nq"]
        st.update(_cache(case, gen, [n - c for n, c in zip(lens, _counts(case, lens))], toward))
        st["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        # q, k and v as one projection leaves them: heads of one token side by side
        qkv = torch.randn(B, S, nq + 2 * nkv, D, generator=gen, device="cuda").to(dt)
        st.update(q=qkv[:, :, :nq], knew=qkv[:, :, nq:nq + nkv], vnew=qkv[:, :, nq + nkv:],
                  qout=torch.zeros(B, S, nq, D, dtype=dt, device="cuda"),
                  counts=torch.tensor(_counts(case, lens), dtype=torch.int32, device="cuda"))
        # where the first new token of each sequence stands: further on than its cache holds rows after an eviction
        st["positions"] = st["seq_lens"] - st["counts"] + case["shift"]
        if case["bits"] == 4:
            st.update(kback=torch.zeros(B, S, nkv, D, dtype=dt, device="cuda"),
                      vback=torch.zeros(B, S, nkv, D, dtype=dt, device="cuda"))
        if own:
            st["rope"] = _b2().Rope(case["rot"], theta=case["theta"])
        return st
    st.update(_cache(case, gen, lens, toward))
    if op != "bounds":
        nq = case["nq"]
        q = torch.randn(B, nq, D, generator=gen, device="cuda") + 0.5 * toward.repeat_interleave(nq // nkv, 0)
        st.update(q=q.to(dt), out=torch.empty(B, nq, D, dtype=dt, device="cuda"))
        if own:
            b2 = _b2()
            st["ws"] = b2.Workspace(b2.paged_decode_workspace_bytes(B, nq, nkv, D, st["tables"].shape[1] * case["bs"]))
    if op != "attend":
        n = st["tables"].numel()
        codes = torch.zeros(n, nkv, 2, D, dtype=torch.int8, device="cuda")
        scale = torch.ones(n, nkv, device="cuda")
        st.update(codes=codes, scale=scale)
        if op == "sparse":
            _bounds(st, torch.zeros(B, dtype=torch.long, device="cuda"))
        if own:
            st["bounds"] = _b2().BlockBounds(codes=codes, scale=scale)
    if op == "bounds" and case["new"] < case["L"]:
        st["newest"] = torch.full((B,), case["new"], dtype=torch.int32, device="cuda")
    if op == "sparse":
        st["blocks"] = torch.empty(B, nkv, case["n"], dtype=torch.int32, device="cuda")
        if own:
            st["sws"] = b2.Workspace(b2.paged_block_select_workspace_bytes(B, nkv, st["tables"].shape[1]))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return {"append": _append, "attend": _attend, "bounds": _bounds_pass, "sparse": _sparse}[state["op"]](state)


def _rotate(x, at, rot, theta):
    """x [B, S, H, D] of tokens at positions `at` [B, S]: the first `rot` channels turned, in 64 bits."""
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = (at.double()[..., None] * f)[:, :, None]
    x = x.double()
    x1, x2 = x[..., : rot // 2], x[..., rot // 2: rot]
    c, s = torch.cos(a), torch.sin(a)
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s, x[..., rot:]), -1)


def _append(s):
    if own:
        b2 = sys.modules.get("b2engine") or _b2()
        b2.paged_kv_append(s["kv"], s["knew"], s["vnew"], q=s["q"], q_out=s["qout"], rope=s["rope"],
                           counts=s["counts"], positions=s["positions"])
        if s["bits"] == 16:
            return s["qout"], s["k"], s["v"]
        b2.paged_kv_read(s["kv"], s["kback"], s["vback"], counts=s["counts"])
        return s["qout"], s["kback"], s["vback"]
    B, S, nkv, D = s["knew"].shape
    bs = s["bs"]
    i = torch.arange(S, device="cuda")
    at = s["positions"].long()[:, None] + i
    b, i = (i < s["counts"][:, None]).nonzero(as_tuple=True)
    s["qout"][b, i] = _rotate(s["q"], at, s["rot"], s["theta"])[b, i].to(s["qout"].dtype)
    k = _rotate(s["knew"], at, s["rot"], s["theta"])[b, i]
    pos = (s["seq_lens"] - s["counts"]).long()[b] + i
    blk = s["tables"].long()[b, pos // bs]
    if s["bits"] == 16:
        s["k"][blk, pos % bs] = k.to(s["k"].dtype)
        s["v"][blk, pos % bs] = s["vnew"][b, i]
        return s["qout"], s["k"], s["v"]
    parts = _quantise(k) + _quantise(s["vnew"][b, i].double())
    Dp, p = _padded(D), pos % 16
    ng = -(-Dp // 64)
    # one row of 16 equal ones packed as a tile, whose bytes for position p are then moved
    rows = _pack(*(x[:, :, None].expand(-1, -1, 16, -1) for x in parts))
    mine = _bytes_of(Dp, ng)[p]
    h = torch.arange(nkv, device="cuda")[None, :, None]
    s["pool"][blk[:, None, None], h, (pos % bs // 16)[:, None, None], mine[:, None]] = rows.gather(
        -1, mine[:, None].expand(-1, nkv, -1))
    kb, vb = _unpack(s["pool"][blk, :, pos % bs // 16], D)
    s["kback"][b, i] = kb[torch.arange(len(p), device="cuda"), :, p].to(s["kback"].dtype)
    s["vback"][b, i] = vb[torch.arange(len(p), device="cuda"), :, p].to(s["vback"].dtype)
    return s["qout"], s["kback"], s["vback"]


def _bytes_of(Dp, ng):
    """Bytes of a tile that belong to each of its 16 positions, [16, Dp + 8 NG]."""
    p = torch.arange(16, device="cuda")[:, None]
    slot = p % 8 // 2 * 4 + p // 8 * 2 + p % 2
    at = torch.arange(Dp // 2, device="cuda")[None]
    k = p * (Dp // 2) + at
    v = 8 * Dp + (at // 2 * 4 + p % 8 // 2) * 8 + p // 8 * 4 + p % 2 * 2 + at % 2
    g = slot * 4 * ng + torch.arange(4 * ng, device="cuda")[None]
    return torch.cat((k, v, 16 * Dp + g, 16 * Dp + 64 * ng + g), 1)


def _softmax(q, k, v, vis):
    """Attention in 32 bits: q [B, nkv, G, D], k and v [B, nkv, T, D], vis [B, 1 or nkv, 1, T]; zeros if nothing is
    seen."""
    z = torch.matmul(q, k.transpose(-1, -2))
    z *= 1.0 / math.sqrt(q.shape[-1])
    z.masked_fill_(~vis, -math.inf)
    m = z.amax(-1, keepdim=True).clamp_(min=-3e38)
    p = torch.exp_(z.sub_(m))
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    return torch.matmul(p, v)


def _attend(s):
    if own:
        b2 = sys.modules.get("b2engine") or _b2()
        return b2.paged_decode_gqa(s["q"], s["kv"], s["out"], window=s["window"], sinks=s["sinks"], ws=s["ws"])
    B, nq, D = s["q"].shape
    nkv, bs, W = s["nkv"], s["bs"], s["window"]
    lens = s["seq_lens"].long()[:, None]
    pos = torch.arange(s["tables"].shape[1] * bs, device="cuda")
    vis = pos < lens
    if W:
        vis = vis & ((pos >= lens - W) | (pos < s["sinks"]))
    k, v = _unpack(s["pool"][s["tables"].long()].transpose(1, 2), D)
    seen = vis[:, None, :, None]
    k = torch.where(seen, k.reshape(B, nkv, -1, D), 0.0)
    v = torch.where(seen, v.reshape(B, nkv, -1, D), 0.0)
    o = _softmax(s["q"].float().view(B, nkv, nq // nkv, D), k, v, vis[:, None, None, :])
    s["out"].copy_(o.reshape(B, nq, D))
    return s["out"]


def _bounds(s, since):
    """Bounds of the blocks that hold the positions from since[b] on, in place."""
    B, mb = s["tables"].shape
    bs, nkv, D = s["bs"], s["nkv"], s["D"]
    lens = s["seq_lens"].long()
    j = torch.arange(mb, device="cuda")
    b, j = ((j * bs < lens[:, None]) & ((j + 1) * bs > since[:, None])).nonzero(as_tuple=True)
    if "pool" in s:
        at = s["tables"].long()[b, j]
        half = len(at) // 2
        k = torch.cat([_unpack(s["pool"][x], D)[0] for x in (at[:half], at[half:])]).reshape(len(at), nkv, bs, D)
    else:
        at = s["tables"].long()[b, j]
        k = s["k"][at].transpose(1, 2).float()
    there = (torch.arange(bs, device="cuda") < (lens[b] - j * bs)[:, None])[:, None, :, None]
    lo = torch.where(there, k, math.inf).amin(2).double()
    hi = torch.where(there, k, -math.inf).amax(2).double()
    top = torch.maximum(lo.abs(), hi.abs()).amax(-1)
    fine = torch.isfinite(top)
    f, e = torch.frexp(torch.where(fine, top, 1.0))
    e = torch.where(f > 127 / 128, e - 6, e - 7).clamp(min=-126)
    e = torch.where(top == 0, 0, e)
    back = torch.ldexp(torch.ones_like(top), -e)[..., None]
    codes = torch.stack((torch.floor(lo * back), torch.ceil(hi * back)), 2)
    s["codes"][at] = torch.where(fine[..., None, None], codes, 0.0).to(torch.int8)
    s["scale"][at] = torch.where(fine, torch.ldexp(torch.ones_like(top), e), math.inf).float()


def _bounds_pass(s):
    if own:
        b2 = sys.modules.get("b2engine") or _b2()
        b2.paged_block_bounds(s["kv"], s["bounds"], newest=s.get("newest"))
    else:
        new = s["newest"].long() if "newest" in s else s["seq_lens"].long()
        _bounds(s, (s["seq_lens"].long() - new).clamp(min=0))
    return s["codes"].float() * s["scale"][:, :, None, None]


def _select(s):
    """Chosen blocks [B, nkv, n], ascending, -1 after the last."""
    B, mb = s["tables"].shape
    nkv, bs, n, D = s["nkv"], s["bs"], s["n"], s["D"]
    q = s["q"].double().view(B, nkv, -1, D)
    up = torch.stack((q.clamp(max=0).sum(2), q.clamp(min=0).sum(2)), 2)  # lower bounds meet negative parts
    top = up.abs().amax((2, 3))
    fine = torch.isfinite(top)
    f, e = torch.frexp(torch.where(fine, top, 1.0))
    e = torch.where(f > 32767 / 32768, e - 14, e - 15)
    up = torch.where(fine[..., None, None], torch.round(up * torch.ldexp(torch.ones_like(top), -e)[..., None, None]), 0.0)
    at = s["tables"].long()
    total = torch.einsum("bhx,bmhx->bhm", up.flatten(2), s["codes"][at].flatten(3).double())  # whole numbers: exact
    scale = s["scale"][at].transpose(1, 2)
    score = torch.where(torch.isinf(scale), math.inf, total.float() * scale)
    nb = (-(-s["seq_lens"].long() // bs))[:, None, None]
    j = torch.arange(mb, device="cuda")
    always = (j < s["first"]) | (j >= nb - s["last"])
    by = torch.sort(score, dim=-1, descending=True, stable=True).indices
    rest = torch.where(j >= nb, 2, torch.where(always, 0, 1)).expand_as(score)
    by = by.gather(-1, torch.sort(rest.gather(-1, by), dim=-1, stable=True).indices)
    count = nb.clamp(max=n)
    kept = torch.zeros_like(score, dtype=torch.bool)
    kept.scatter_(-1, by, (j < count).expand_as(by))
    out = torch.full((B, nkv, n + 1), -1, dtype=torch.long, device="cuda")
    out.scatter_(-1, torch.where(kept, kept.cumsum(-1) - 1, n), j.expand_as(by).contiguous())
    s["blocks"].copy_(torch.where(torch.arange(n, device="cuda") < count, out[..., :n], -1))


def _sparse(s):
    if own:
        b2 = sys.modules.get("b2engine") or _b2()
        b2.paged_block_select(s["q"], s["kv"], s["bounds"], s["blocks"], first=s["first"], last=s["last"], ws=s["sws"])
        b2.paged_decode_gqa(s["q"], s["kv"], s["out"], blocks=s["blocks"], ws=s["ws"])
        return s["blocks"], s["out"]
    _select(s)
    B, nq, D = s["q"].shape
    nkv, bs, n = s["nkv"], s["bs"], s["n"]
    blocks = s["blocks"].long()
    at = s["tables"].long()[torch.arange(B, device="cuda")[:, None, None], blocks.clamp(min=0)]
    h = torch.arange(nkv, device="cuda")[None, :, None]
    pos = blocks[..., None] * bs + torch.arange(bs, device="cuda")
    vis = ((pos >= 0) & (pos < s["seq_lens"].long()[:, None, None, None])).reshape(B, nkv, n * bs)
    if "pool" in s:
        k, v = _unpack(s["pool"][at, h], D)
    else:
        k, v = s["k"].transpose(1, 2)[at, h].float(), s["v"].transpose(1, 2)[at, h].float()
    k = torch.where(vis[..., None], k.reshape(B, nkv, n * bs, D), 0.0)
    v = torch.where(vis[..., None], v.reshape(B, nkv, n * bs, D), 0.0)
    o = _softmax(s["q"].float().view(B, nkv, nq // nkv, D), k, v, vis[:, :, None, :])
    s["out"].copy_(o.reshape(B, nq, D))
    return s["blocks"], s["out"]


# ---------------------------------------------------------------------------
# the definitions in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------

def _places(D):
    """Where a tile holds (position, channel): byte and shift of the K and V codes, byte of K's scale."""
    Dp = _padded(D)
    ng = -(-Dp // 64)
    p = torch.arange(16, device="cuda")[:, None]
    c = torch.arange(D, device="cuda")[None, :]
    kc = p * Dp // 2 + ((c // 8) % 4 * (Dp // 32) + c // 32) * 4 + c % 8 // 2
    vc = 8 * Dp + ((c // 32 * 8 + c % 32 // 4) * 4 + p % 8 // 2) * 8 + p // 8 * 4 + p % 2 * 2 + c % 4 // 2
    ks = 16 * Dp + ((p % 8 // 2 * 4 + p // 8 * 2 + p % 2) * ng + c // 64) * 4
    return kc, vc, (c % 2 * 4).expand(16, D), ks, ks + 64 * ng


def _rows4(st, b, t, h):
    """K and V rows of positions t (sequence b, K/V head h) of the 4-bit cache in 64 bits, each m + u s."""
    bs, D = st["bs"], st["D"]
    tiles = st["pool"][st["tables"][b, t // bs].long(), h, t % bs // 16]
    kc, vc, sh, ks, vs = _places(D)
    x = torch.arange(len(t), device="cuda")[:, None]
    got = []
    for code, at in ((kc, ks), (vc, vs)):
        u = (tiles[x, code[t % 16]].long() >> sh[t % 16]) & 15
        raw = [tiles[x, at[t % 16] + i].to(torch.int32) for i in range(4)]
        half = [(raw[i] | raw[i + 1] << 8).to(torch.int16).view(torch.float16).double() for i in (0, 2)]
        got.append(half[1] + u * half[0])
    return got


def _rows(st, b, t, h):
    if "pool" in st:
        return _rows4(st, b, t, h)
    blk, slot = st["tables"][b, t // st["bs"]].long(), t % st["bs"]
    return st["k"][blk, slot, h].double(), st["v"][blk, slot, h].double()


def _held(x):
    """Rows [R, D] in 64 bits as the 4-bit cache holds them."""
    out = torch.empty_like(x)
    for g in range(0, x.shape[1], 64):
        y = x[:, g: g + 64]
        m = y.min(1, keepdim=True).values.half().double()
        s = ((y.max(1, keepdim=True).values - m) / 15).half().double()
        u = torch.where(s > 0, torch.round((y - m) / s), 0.0).clamp(0, 15)
        out[:, g: g + 64] = m + u * s
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op, lens = case["op"], _lens(case)
    B, nkv, D, bs = case["B"], case["nkv"], case["D"], case["bs"]
    if op == "append":
        counts, rot = _counts(case, lens), case["rot"]
        qout = st["qout"].double()
        if case["bits"] == 16:
            k, v = st["k"].double(), st["v"].double()
        else:
            k, v = st["kback"].double(), st["vback"].double()
        half = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
        freq = torch.exp(-2 * half / rot * math.log(case["theta"]))
        for b, (n, c) in enumerate(zip(lens, counts)):
            t = torch.arange(n - c, n, device="cuda")
            turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), (t + case["shift"])[:, None, None] * freq)
            for src, heads in ((st["q"], "q"), (st["knew"], "k")):
                x = src[b, :c].double()
                z = torch.complex(x[..., : rot // 2].contiguous(), x[..., rot // 2: rot].contiguous()) * turn
                x = torch.cat((z.real, z.imag, x[..., rot:]), -1)
                if heads == "q":
                    qout[b, :c] = x
                elif case["bits"] == 4:
                    k[b, :c] = _held(x.reshape(-1, D)).view(c, nkv, D)
                else:
                    k[st["tables"][b, t // bs].long(), t % bs] = x
            x = st["vnew"][b, :c].double()
            if case["bits"] == 4:
                v[b, :c] = _held(x.reshape(-1, D)).view(c, nkv, D)
            else:
                v[st["tables"][b, t // bs].long(), t % bs] = x
        return qout, k, v
    if op == "bounds":
        if B * nkv * (case["L"] // bs) > 20000:
            return None
        val = st["codes"].double() * st["scale"].double()[:, :, None, None]
        for b, n in enumerate(lens):
            for j in range(max(0, n - case["new"]) // bs, -(-n // bs)):
                t = torch.arange(j * bs, min(n, (j + 1) * bs), device="cuda")
                k = torch.stack([_rows(st, b, t, h)[0].float().double() for h in range(nkv)])
                top = k.abs().amax((1, 2)).tolist()
                unit = torch.tensor([2.0 ** max(-126, math.ceil(math.log2(x / 127))) if x > 0 else 1.0 for x in top],
                                    dtype=torch.float64, device="cuda")[:, None]
                to = int(st["tables"][b, j])
                val[to, :, 0] = torch.floor(k.amin(1) / unit) * unit
                val[to, :, 1] = torch.ceil(k.amax(1) / unit) * unit
        return val
    nq = case["nq"]
    g = nq // nkv
    out = torch.zeros(B, nq, D, dtype=torch.float64, device="cuda")
    chosen = torch.full((B, nkv, case.get("n", 1)), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        if op == "attend":
            W, K = case["window"], case["sinks"]
            t = torch.arange(n, device="cuda")
            t = t[(t >= n - W) | (t < K)] if W else t
        for h in range(nkv):
            q = st["q"][b, h * g: (h + 1) * g].double()
            if op == "sparse":
                nb = -(-n // bs)
                pick = torch.arange(nb, device="cuda")
                if nb > case["n"]:
                    parts = torch.cat((q.clamp(max=0).sum(0), q.clamp(min=0).sum(0)))
                    unit = 2.0 ** math.ceil(math.log2(float(parts.abs().max()) / 32767))
                    at = st["tables"][b, :nb].long()
                    score = (st["codes"][at, h].flatten(1).double() * torch.round(parts / unit)).sum(1)
                    score = score.float() * st["scale"][at, h]
                    score[: case["first"]] = math.inf
                    score[nb - case["last"]:] = math.inf
                    pick = torch.argsort(-score, stable=True)[: case["n"]].sort().values
                chosen[b, h, : len(pick)] = pick.int()
                t = (pick[:, None] * bs + torch.arange(bs, device="cuda")).flatten()
                t = t[t < n]
            k, v = _rows(st, b, t, h)
            out[b, h * g: (h + 1) * g] = torch.softmax(q @ k.T / D ** 0.5, -1) @ v
    return (chosen, out) if op == "sparse" else out
