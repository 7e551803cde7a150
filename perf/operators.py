"""The bounded-cache attention operators, as cases to time and compare.

Three operators of long-context serving on a paged K/V cache that is kept
small:

  prefill  causal GQA attention of a chunk of prompt tokens in which a query
           sees the last `window` positions and the first `sinks` ones;
  decode   GQA attention of one new token per sequence over a block pool read
           through block tables, whole or with window and sinks, optionally
           adding every position's attention weight to a running score;
  evict    the choice of the `budget` positions of each (sequence, K/V head)
           that stay (sinks, the most recent, and the best scores between
           them) and the move of their K/V rows and scores to fresh blocks.

`own` False computes them with elementary torch operations in 32 bits; `own`
True calls serving-engine_b200 (b2engine)."""
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
        # a short prompt of a small model (14/2 heads of 64): what a call costs before it does any work
        dict(name="prefill_short", op="prefill", B=1, S=77, start=0, nq=14, nkv=2, D=64, dtype="fp16", window=32,
             sinks=4, ragged=0.0),
        # a batch of prompts of different lengths at 8B widths, padded to the longest
        dict(name="prefill_ragged", op="prefill", B=4, S=1001, start=0, nq=32, nkv=8, D=128, dtype="bf16", window=512,
             sinks=4, ragged=0.6),
        # one long prompt in one call
        dict(name="prefill_long", op="prefill", B=1, S=8192, start=0, nq=32, nkv=8, D=128, dtype="bf16", window=2048,
             sinks=4, ragged=0.0),
        # a later chunk of a long prompt at 70B widths: the chunk's queries against earlier keys too
        dict(name="prefill_chunk", op="prefill", B=1, S=512, start=5500, nq=64, nkv=8, D=128, dtype="fp16",
             window=4095, sinks=128, ragged=0.0),
        # one chat turn of a small model: the latency of a step
        dict(name="decode_single", op="decode", B=1, L=301, bs=16, nq=14, nkv=2, D=64, dtype="fp16", window=0,
             sinks=0, scores=False, ragged=0.0, layout="slot"),
        # an ordinary batch that also keeps attention weights for a later eviction
        dict(name="decode_scored", op="decode", B=8, L=4096, bs=16, nq=32, nkv=8, D=128, dtype="fp16", window=0,
             sinks=0, scores=True, ragged=0.5, layout="slot"),
        # a full batch of long contexts, everything read
        dict(name="decode_full", op="decode", B=32, L=32768, bs=16, nq=32, nkv=8, D=128, dtype="bf16", window=0,
             sinks=0, scores=False, ragged=0.3, layout="slot"),
        # the same batch reading only window and sinks, pool kept head-major inside a block
        dict(name="decode_window", op="decode", B=32, L=16384, bs=32, nq=32, nkv=8, D=128, dtype="bf16", window=1024,
             sinks=4, scores=False, ragged=0.9, layout="head"),
        # one sequence with a very long context at 70B widths
        dict(name="decode_long", op="decode", B=1, L=131001, bs=16, nq=64, nkv=8, D=128, dtype="fp16", window=0,
             sinks=0, scores=True, ragged=0.0, layout="slot"),
        # one sequence of a small model over its budget
        dict(name="evict_single", op="evict", B=1, L=601, bs=16, nkv=2, D=64, dtype="fp16", budget=256, sinks=4,
             recent=64, ragged=0.0, layout="slot"),
        # an ordinary batch, some of it still under the budget
        dict(name="evict_batch", op="evict", B=8, L=4096, bs=16, nkv=8, D=128, dtype="bf16", budget=1024, sinks=4,
             recent=256, ragged=0.9, layout="slot"),
        # a large batch of long contexts
        dict(name="evict_long", op="evict", B=16, L=32768, bs=16, nkv=8, D=128, dtype="fp16", budget=8192, sinks=4,
             recent=1023, ragged=0.4, layout="slot"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefill", "decode", "decode", "evict"])
    nq, nkv, D = rng.choice([(14, 2, 64), (32, 8, 128), (64, 8, 128), (8, 8, 64), (12, 4, 128), (16, 2, 80),
                             (32, 32, 128), (8, 1, 96)])
    dtype = rng.choice(["fp16", "bf16"])
    ragged = rng.choice([0.0, 0.3, 0.9])
    sinks = rng.choice([0, 1, 4, 4, 64, 133])
    if op == "prefill":
        B = rng.choice([1, 1, 2, 3, 5])
        most = 8192
        while True:  # the products of all pairs stay within the largest listed case's
            S, start = _log(rng, 1, most), rng.choice([0, 0, _log(rng, 1, most)])
            if B * nq * S * (S + start) <= 32 * 8192 * 8192:
                break
        window = rng.choice([0, _log(rng, 1, 4096), _log(rng, 16, 4096), _log(rng, 16, 4096)])
        if B * nq * D * S * min(S + start, window or S + start) > 32 * 128 * 8192 * 2048:
            window = 512
        return dict(op=op, B=B, S=S, start=start, nq=nq, nkv=nkv, D=D, dtype=dtype, window=window, sinks=sinks,
                    ragged=ragged)
    bs = rng.choice([8, 16, 16, 16, 32, 64, 128])
    layout = rng.choice(["slot", "slot", "head"])
    B = _log(rng, 1, 32)
    if op == "decode":
        L = _log(rng, 1, 131072)
        L = max(1, min(L, 32 * 20000 * 8 * 128 // (B * nkv * D)))
        window = rng.choice([0, 0, _log(rng, 1, 8192)])
        return dict(op=op, B=B, L=L, bs=bs, nq=nq, nkv=nkv, D=D, dtype=dtype, window=window, sinks=sinks,
                    scores=rng.random() < 0.5, ragged=ragged, layout=layout)
    B = min(B, 16)
    L = _log(rng, 1, 65536)
    L = max(1, min(L, 16 * 32768 * 8 * 128 // (B * nkv * D)))
    budget = max(1, min(_log(rng, 1, 2 * L), 16 * 8192 * 8 * 128 // (B * nkv * D)))
    sinks = min(sinks, budget // 4)
    return dict(op=op, B=B, L=L, bs=bs, nkv=nkv, D=D, dtype=dtype, budget=budget, sinks=sinks,
                recent=rng.randrange(0, budget - sinks + 1), ragged=ragged, layout=layout)


def _lens(case):
    """Length of each sequence: the longest first, the others up to `ragged` shorter."""
    T = case["L"] if "L" in case else case["start"] + case["S"]
    return [max(1, T - int(T * case["ragged"] * ((b * 0.6180339887) % 1.0))) for b in range(case["B"])]


def _visible(pos, n, window, sinks):
    """How many positions the query at `pos` sees of a sequence of n tokens."""
    if pos >= n:
        return 0
    if window == 0 or window > pos:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    D, nkv, B = case["D"], case["nkv"], case["B"]
    lens = _lens(case)
    if case["op"] == "prefill":
        nq, S, start, W, K = case["nq"], case["S"], case["start"], case["window"], case["sinks"]
        pairs = rows = 0
        for n in lens:
            pairs += sum(_visible(start + i, n, W, K) for i in range(S))
            if n <= start:
                continue
            first = max(0, start + 1 - W) if W else 0  # the first key that the first query's window holds
            rows += n - first + min(K, first)
        return {"bytes": 2 * (2 * B * S * nq * D + 2 * rows * nkv * D), "flops": 4 * D * nq * pairs}
    if case["op"] == "decode":
        nq = case["nq"]
        vis = sum(_visible(n - 1, n, case["window"], case["sinks"]) for n in lens)
        tables = sum(-(-n // case["bs"]) for n in lens) if case["window"] == 0 else vis // case["bs"]
        return {"bytes": 4 * vis * nkv * D + 4 * B * nq * D + 4 * (tables + B) + (8 * vis * nkv if case["scores"] else 0),
                "flops": 4 * D * nq * vis}
    kept = sum(min(n, case["budget"]) for n in lens)
    # scores of all positions read, rows and scores of the kept ones moved, their list and the lengths written
    return {"bytes": 4 * sum(lens) * nkv + 8 * kept * nkv * D + 4 * kept * nkv + 4 * B * nkv * case["budget"] + 8 * B,
            "flops": sum(lens) * nkv}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _b2():
    path = os.path.join(os.getcwd(), "serving-engine_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b2engine
    return b2engine


def _pool(case, gen, lens, extra, first_keys):
    """K and V pools, block tables and lengths of B sequences: rows ~ N(0, 1), the first four tokens' keys pushed
    along `first_keys` (attention sinks), and what lies past a sequence's end never written (NaN)."""
    B, bs, nkv, D = case["B"], case["bs"], case["nkv"], case["D"]
    dt = DTYPES[case["dtype"]]
    mb = -(-case["L"] // bs)
    n = B * mb
    shape = (n + extra, bs, nkv, D) if case["layout"] == "slot" else (n + extra, nkv, bs, D)
    k = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    if case["layout"] == "head":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    tables = torch.randperm(n, generator=gen, device="cuda").to(torch.int32).view(B, mb)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    tl = tables.long()
    for t in range(min(4, case["L"])):
        k[tl[:, t // bs], t % bs] += first_keys.to(dt)
    pos = torch.arange(mb * bs, device="cuda")
    b, p = (pos[None, :] >= seq_lens[:, None]).nonzero(as_tuple=True)
    k[tl[b, p // bs], p % bs] = float("nan")
    v[tl[b, p // bs], p % bs] = float("nan")
    return k, v, tables, seq_lens


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, nkv, D, dt = case["B"], case["nkv"], case["D"], DTYPES[case["dtype"]]
    lens = _lens(case)
    toward = torch.randint(0, 2, (nkv, D), generator=gen, device="cuda").float() * 2 - 1
    st = dict(case)
    if case["op"] == "prefill":
        S, T, nq = case["S"], case["start"] + case["S"], case["nq"]
        # q, k and v as a projection leaves them: heads of one token side by side
        q = torch.randn(B, S, nq, D, generator=gen, device="cuda")
        q += 0.5 * toward.repeat_interleave(nq // nkv, 0)
        k = torch.randn(B, T, nkv, D, generator=gen, device="cuda")
        k[:, :4] += 0.7 * toward
        v = torch.randn(B, T, nkv, D, generator=gen, device="cuda")
        for b, n in enumerate(lens):  # padding is never written
            k[b, n:] = float("nan")
            v[b, n:] = float("nan")
        st.update(q=q.to(dt), k=k.to(dt), v=v.to(dt), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                  out=torch.empty(B, S, nq, D, dtype=dt, device="cuda"))
        return st
    if case["op"] == "decode":
        nq = case["nq"]
        k, v, tables, seq_lens = _pool(case, gen, lens, 0, 0.7 * toward)
        q = torch.randn(B, nq, D, generator=gen, device="cuda") + 0.5 * toward.repeat_interleave(nq // nkv, 0)
        scores = None
        if case["scores"]:
            scores = torch.rand(k.shape[0], nkv, case["bs"], generator=gen, device="cuda")
        st.update(q=q.to(dt), k=k, v=v, tables=tables, seq_lens=seq_lens, scores=scores,
                  out=torch.empty(B, nq, D, dtype=dt, device="cuda"))
        if own:
            b2 = _b2()
            st["kv"] = b2.PagedKV(k, v, tables, seq_lens)
            st["ws"] = b2.Workspace(b2.paged_decode_workspace_bytes(B, nq, nkv, D, tables.shape[1] * case["bs"],
                                                                    scored=case["scores"]))
        return st
    bs, budget = case["bs"], case["budget"]
    db = -(-budget // bs)
    k, v, tables, seq_lens = _pool(case, gen, lens, B * db, 0.7 * toward)
    n = B * tables.shape[1]
    dst = (n + torch.randperm(B * db, generator=gen, device="cuda")).to(torch.int32).view(B, db)
    # accumulated weights: a long tail, and a fifth of the positions never looked at
    scores = -torch.log(torch.rand(k.shape[0], nkv, bs, generator=gen, device="cuda").clamp_(min=1e-6))
    scores *= torch.rand(scores.shape, generator=gen, device="cuda") < 0.8
    st.update(k=k, v=v, tables=tables, seq_lens=seq_lens, dst=dst, scores=scores, fresh=n,
              kept=torch.empty(B, nkv, budget, dtype=torch.int32, device="cuda"),
              new_lens=torch.empty(B, dtype=torch.int32, device="cuda"))
    if own:
        st["kv"] = _b2().PagedKV(k, v, tables, seq_lens)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return {"prefill": _prefill, "decode": _decode, "evict": _evict}[state["op"]](state)


def _attend(q, k, v, vis):
    """Softmax attention in 32 bits; q [B, nkv, R, D], k and v [B, nkv, T, D], vis (broadcast over [B, nkv, R, T]).
    Returns the weights and the outputs; rows that see nothing are zero."""
    s = torch.matmul(q, k.transpose(-1, -2))
    s *= 1.0 / math.sqrt(q.shape[-1])
    s.masked_fill_(~vis, float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    p = torch.exp_(s.sub_(m))
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    return p, torch.matmul(p, v)


def _prefill(s):
    W, K = s["window"], s["sinks"]
    if own:
        b2 = sys.modules.get("b2engine") or _b2()
        b2.window_prefill_gqa(s["q"], s["k"], s["v"], s["out"], window=W, sinks=K, seq_lens=s["lens"])
        return s["out"]
    B, S, nq, D = s["q"].shape
    T, nkv = s["k"].shape[1:3]
    g = nq // nkv
    at = torch.arange(T - S, T, device="cuda")[:, None]
    key = torch.arange(T, device="cuda")[None, :]
    vis = key <= at
    if W:
        vis = vis & ((key > at - W) | (key < K))
    vis = vis[None] & (at < s["lens"][:, None, None]) & (key < s["lens"][:, None, None])
    there = (torch.arange(T, device="cuda") < s["lens"][:, None])[:, :, None, None]
    q = s["q"].float().view(B, S, nkv, g, D).permute(0, 2, 3, 1, 4).reshape(B, nkv, g * S, D)
    k = torch.where(there, s["k"].float(), 0.0).transpose(1, 2)
    v = torch.where(there, s["v"].float(), 0.0).transpose(1, 2)
    _, o = _attend(q, k, v, vis.repeat(1, g, 1)[:, None])
    s["out"].copy_(o.view(B, nkv, g, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, nq, D))
    return s["out"]


def _decode(s):
    W, K = s["window"], s["sinks"]
    if own:
        b2 = sys.modules.get("b2engine") or _b2()
        b2.paged_decode_gqa(s["q"], s["kv"], s["out"], window=W, sinks=K, scores=s["scores"], ws=s["ws"])
        return (s["out"], s["scores"]) if s["scores"] is not None else s["out"]
    B, nq, D = s["q"].shape
    bs, nkv = s["k"].shape[1:3]
    lens = s["seq_lens"].long()
    pos = torch.arange(s["tables"].shape[1] * bs, device="cuda")
    blk = s["tables"].long()[:, pos // bs]
    slot = (pos % bs).expand_as(blk)
    vis = pos < lens[:, None]
    if W:
        vis = vis & ((pos >= lens[:, None] - W) | (pos < K))
    k = torch.where(vis[:, :, None, None], s["k"][blk, slot].float(), 0.0).transpose(1, 2)
    v = torch.where(vis[:, :, None, None], s["v"][blk, slot].float(), 0.0).transpose(1, 2)
    p, o = _attend(s["q"].float().view(B, nkv, nq // nkv, D), k, v, vis[:, None, None, :])
    s["out"].copy_(o.reshape(B, nq, D))
    if s["scores"] is None:
        return s["out"]
    heads = torch.arange(nkv, device="cuda")
    last = lens - 1
    b = torch.arange(B, device="cuda")
    # the newest position starts from nothing, whatever its slot held
    s["scores"][s["tables"].long()[b, last // bs][:, None], heads, (last % bs)[:, None]] = 0.0
    s["scores"].index_put_((blk[:, None, :], heads[None, :, None], slot[:, None, :]), p.sum(2), accumulate=True)
    return s["out"], s["scores"]


def _evict(s):
    budget, K, recent = s["budget"], s["sinks"], s["recent"]
    n = s["fresh"]
    if own:
        b2 = sys.modules.get("b2engine") or _b2()
        b2.paged_kv_evict(s["kv"], s["scores"], budget, s["kept"], s["new_lens"], sinks=K, recent=recent,
                          dst_tables=s["dst"])
        return s["kept"], s["new_lens"], s["k"][n:], s["v"][n:], s["scores"][n:]
    B, mb = s["tables"].shape
    bs, nkv = s["k"].shape[1:3]
    lens = s["seq_lens"].long()
    pos = torch.arange(mb * bs, device="cuda")
    blk = s["tables"].long()[:, pos // bs]
    slot = (pos % bs).expand_as(blk)
    heads = torch.arange(nkv, device="cuda")
    sc = s["scores"][blk[:, None, :], heads[None, :, None], slot[:, None, :]]
    rest = (pos >= lens[:, None]).long() * 2 + ((pos >= K) & (pos < lens[:, None] - recent)).long()
    by = torch.sort(sc, dim=-1, descending=True, stable=True).indices
    by = by.gather(-1, torch.sort(rest[:, None].expand_as(by).gather(-1, by), dim=-1, stable=True).indices)
    now = lens.clamp(max=budget)
    keep = torch.zeros_like(sc, dtype=torch.bool)
    keep.scatter_(-1, by, (pos < now[:, None])[:, None].expand_as(by))
    to = torch.where(keep, keep.cumsum(-1) - 1, budget)
    kept = torch.full((B, nkv, budget + 1), -1, dtype=torch.long, device="cuda")
    kept.scatter_(-1, to, pos.expand_as(to).contiguous())
    kept = kept[:, :, :budget]
    kept = torch.where(torch.arange(budget, device="cuda") < now[:, None, None], kept, -1)
    s["kept"].copy_(kept)
    s["new_lens"].copy_(now)
    # rows and scores of the kept positions, in order, into the fresh blocks
    j = torch.arange(budget, device="cuda")
    live = (j < now[:, None])[:, None]
    src = kept.clamp(min=0)
    h = heads[None, :, None]
    sb, ss = s["tables"].long()[torch.arange(B, device="cuda")[:, None, None], src // bs], src % bs
    db, ds = s["dst"].long()[:, j // bs][:, None], (j % bs)[None, None]
    for x in (s["k"], s["v"]):
        x[db, ds, h] = torch.where(live[..., None], x[sb, ss, h], x[db, ds, h])
    s["scores"][db, h, ds] = torch.where(live, s["scores"][sb, h, ss], s["scores"][db, h, ds])
    return s["kept"], s["new_lens"], s["k"][n:], s["v"][n:], s["scores"][n:]


# ---------------------------------------------------------------------------
# the definitions in 64 bits, one sequence and one K/V head at a time
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    lens = _lens(case)
    B, nkv, D = case["B"], case["nkv"], case["D"]
    if case["op"] == "prefill":
        S, T, nq = case["S"], case["start"] + case["S"], case["nq"]
        out = torch.zeros(B, S, nq, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            rows = min(S, n - case["start"])
            if rows <= 0:
                continue
            i = case["start"] + torch.arange(rows, device="cuda")
            j = torch.arange(n, device="cuda")
            back = i[:, None] - j[None, :]
            hidden = back < 0
            if case["window"]:
                hidden |= (back >= case["window"]) & (j >= case["sinks"])[None, :]
            for h in range(nq):
                kv = h * nkv // nq
                z = st["q"][b, :rows, h].double() @ st["k"][b, :n, kv].double().T / D ** 0.5
                z[hidden] = float("-inf")
                out[b, :rows, h] = torch.softmax(z, -1) @ st["v"][b, :n, kv].double()
        return out
    bs = case["bs"]
    if case["op"] == "decode":
        nq = case["nq"]
        out = torch.zeros(B, nq, D, dtype=torch.float64, device="cuda")
        scores = st["scores"].double() if case["scores"] else None
        for b, n in enumerate(lens):
            seen = [t for t in range(n) if case["window"] == 0 or t < case["sinks"] or n - t <= case["window"]]
            t = torch.tensor(seen, device="cuda")
            blk, slot = st["tables"][b, t // bs].long(), t % bs
            for kv in range(nkv):
                mine = slice(kv * nq // nkv, (kv + 1) * nq // nkv)
                z = st["q"][b, mine].double() @ st["k"][blk, slot, kv].double().T / D ** 0.5
                w = torch.softmax(z, -1)
                out[b, mine] = w @ st["v"][blk, slot, kv].double()
                if scores is not None:
                    w = w.sum(0)
                    w[:-1] += scores[blk[:-1], kv, slot[:-1]]
                    scores[blk, kv, slot] = w
        return (out, scores) if case["scores"] else out
    n0, budget = st["fresh"], case["budget"]
    kept = torch.full((B, nkv, budget), -1, dtype=torch.int32)
    pools = [st["k"], st["v"]]
    outs = [x[n0:].clone() for x in pools]
    outs.append(st["scores"][n0:].double())
    tables, dst = st["tables"].cpu(), st["dst"].cpu()
    for b, n in enumerate(lens):
        now = min(n, budget)
        where = torch.arange(n)
        stays = (where < case["sinks"]) | (where >= n - case["recent"])
        j = torch.arange(now)
        to_b, to_s = (dst[b, j // bs].long() - n0).cuda(), (j % bs).cuda()
        for kv in range(nkv):
            sc = st["scores"][tables[b, where // bs].long().cuda(), kv, (where % bs).cuda()].double().cpu()
            if n > budget:
                sc[stays] = float("inf")
                pick = torch.argsort(-sc, stable=True)[:budget].sort().values
            else:
                pick = where
            kept[b, kv, :now] = pick.int()
            fb, fs = tables[b, pick // bs].long().cuda(), (pick % bs).cuda()
            for x, y in zip(pools, outs):
                y[to_b, to_s, kv] = x[fb, fs, kv]
            outs[2][to_b, kv, to_s] = st["scores"][fb, kv, fs].double()
    return kept, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32), outs[0].double(), outs[1].double(), outs[2]
