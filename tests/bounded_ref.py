"""The bounded-cache attention operators in 64 bits, straight from their
definitions, one sequence and one head at a time (torch, any device).  Each
attention reference also returns sum_j p_ij |v_j|, which the rounding bounds of
the tests are stated in."""
import math

import torch


def visible(i, n, window, sinks, device="cpu"):
    """bool [n]: the positions that the query at position i sees."""
    j = torch.arange(n, device=device)
    back = i - j
    ok = back >= 0
    if window > 0:
        ok &= (back < window) | (j < sinks)
    return ok


def attend(q, k, v, ok):
    """q [R, D], k and v [n, D], ok bool [R, n]: outputs, sum p|v| and weights, all in 64 bits."""
    s = q.double() @ k.double().T / math.sqrt(q.shape[-1])
    s = s.masked_fill(~ok, -math.inf)
    some = ok.any(-1, keepdim=True)
    m = torch.where(some, s.amax(-1, keepdim=True), torch.zeros((), dtype=torch.float64, device=s.device))
    p = torch.exp(s - m) * ok
    p = p / torch.where(some, p.sum(-1, keepdim=True), torch.ones((), dtype=torch.float64, device=s.device))
    vd = v.double()
    return p @ vd, p @ vd.abs(), p


def window_prefill(q, k, v, lens, window, sinks):
    """q [B, S, nq, D], k and v [B, T, nkv, D]; the queries are the last S positions."""
    B, S, nq, D = q.shape
    T, nkv = k.shape[1:3]
    out = torch.zeros(B, S, nq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for b in range(B):
        n = T if lens is None else min(T, int(lens[b]))
        rows = min(S, n - (T - S))
        if rows <= 0:
            continue
        ok = torch.stack([visible(T - S + i, n, window, sinks, q.device) for i in range(rows)])
        for h in range(nq):
            kv = h // (nq // nkv)
            o, a, _ = attend(q[b, :rows, h], k[b, :n, kv], v[b, :n, kv], ok)
            out[b, :rows, h], mag[b, :rows, h] = o, a
    return out, mag


def paged_decode(q, k, v, tables, lens, window, sinks, scores=None):
    """q [B, nq, D], pools [blocks, bs, nkv, D]; scores [blocks, nkv, bs] or None (not modified).
    Returns outputs, sum p|v|, the new scores and what was added to each."""
    B, nq, D = q.shape
    nb, bs, nkv, _ = k.shape
    out = torch.zeros(B, nq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    new = None if scores is None else scores.double().clone()
    add = None if scores is None else torch.zeros_like(new)
    for b in range(B):
        n = min(int(lens[b]), tables.shape[1] * bs)
        if n <= 0:
            continue
        pos = visible(n - 1, n, window, sinks, q.device).nonzero()[:, 0]
        blk = tables[b].long()[pos // bs]
        there = (blk >= 0) & (blk < nb)
        pos, blk = pos[there], blk[there]
        if not len(pos):
            continue
        slot = pos % bs
        ok = torch.ones(nq // nkv, len(pos), dtype=torch.bool, device=q.device)
        for kv in range(nkv):
            hs = slice(kv * nq // nkv, (kv + 1) * nq // nkv)
            o, a, p = attend(q[b, hs], k[blk, slot, kv], v[blk, slot, kv], ok)
            out[b, hs], mag[b, hs] = o, a
            if new is not None:
                w = p.sum(0)
                old = torch.where(pos == n - 1, 0.0, new[blk, kv, slot])
                new[blk, kv, slot] = old + w
                add[blk, kv, slot] = w
    return out, mag, new, add


def evict_choice(score, n, budget, sinks, recent):
    """Kept positions of one (sequence, head): score [>= n] in the operator's order (NaN largest, ties low)."""
    if n <= budget:
        return list(range(n))
    key = lambda i: (0, 0.0, i) if math.isnan(score[i]) else (1, -score[i], i)  # noqa: E731
    mid = sorted(range(sinks, n - recent), key=key)[: budget - sinks - recent]
    return sorted(list(range(sinks)) + mid + list(range(n - recent, n)))


def paged_evict(k, v, scores, tables, lens, budget, sinks, recent, dst=None):
    """New pools and scores, kept [B, nkv, budget] and lengths (CPU loops over copies)."""
    nb, bs, nkv, D = k.shape
    B = tables.shape[0]
    k2, v2, s2 = k.clone(), v.clone(), scores.clone()
    kept = torch.full((B, nkv, budget), -1, dtype=torch.int32)
    tab, to = tables.long().cpu(), (tables if dst is None else dst).long().cpu()
    sc = scores.cpu()
    new = []
    for b in range(B):
        n = min(int(lens[b]), tables.shape[1] * bs)
        new.append(min(n, budget))
        if n <= 0:
            continue
        i = torch.arange(n)
        for h in range(nkv):
            keep = evict_choice(sc[tab[b, i // bs], h, i % bs].tolist(), n, budget, sinks, recent)
            kept[b, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            src = torch.tensor(keep)
            j = torch.arange(len(keep))
            sb, ss, db, ds = tab[b, src // bs], src % bs, to[b, j // bs], j % bs
            k2[db, ds, h], v2[db, ds, h] = k[sb, ss, h], v[sb, ss, h]
            s2[db, h, ds] = scores[sb, h, ss]
    return k2, v2, s2, kept, torch.tensor(new, dtype=torch.int32)
