"""The 4-bit paged cache, the append, block bounds and block choice in 64 bits,
straight from their definitions (torch, any device), one row or block at a time
where that is the plainest."""
import math

import torch


def padded(D):
    return next(p for p in (64, 96, 128, 192, 256) if D <= p)


def tile_bytes(D):
    Dp = padded(D)
    return 16 * Dp + 128 * -(-Dp // 64)


def k_place(D, p, c):
    """(byte, shift) of channel c of position p among a tile's K codes."""
    Dp = padded(D)
    word = c // 8
    return p * Dp // 2 + (word % 4 * (Dp // 32) + word // 4) * 4 + c % 8 // 2, c % 2 * 4


def v_place(D, p, c):
    """The same among the V codes."""
    unit = ((c // 32 * 8 + c % 32 // 4) * 4 + p % 8 // 2) * 4 + p // 8 * 2 + p % 2
    return 8 * padded(D) + unit * 2 + c % 4 // 2, c % 2 * 4


def scale_place(D, p, g, value):
    """Byte of the (s, m) halves of group g of position p: value 0 K, 1 V."""
    ng = -(-padded(D) // 64)
    return 16 * padded(D) + 64 * ng * value + ((p % 8 // 2 * 4 + p // 8 * 2 + p % 2) * ng + g) * 4


def quantise(x):
    """x [..., D] in 64 bits: codes, s and m (in 64 bits) of its groups of 64."""
    D = x.shape[-1]
    codes, ss, ms = torch.zeros(x.shape, dtype=torch.long, device=x.device), [], []
    for g in range(0, D, 64):
        y = x[..., g:g + 64]
        fine = torch.isfinite(y).all(-1, keepdim=True)
        m = y.amin(-1, keepdim=True).clamp(-65504, 65504).float().half().double()
        s = ((y.amax(-1, keepdim=True) - m) / 15).clamp(0, 65504).float().half().double()
        u = torch.where((s > 0) & fine, torch.round((y - m) / torch.where(s > 0, s, 1.0)), 0.0).clamp(0, 15)
        codes[..., g:g + 64] = u.nan_to_num().long()
        ss.append(torch.where(fine, s, math.nan))
        ms.append(torch.where(fine, m, math.nan))
    return codes, torch.cat(ss, -1), torch.cat(ms, -1)


def held(x):
    """x [..., D] as a 4-bit row holds it, in 64 bits."""
    codes, s, m = quantise(x)
    at = torch.arange(x.shape[-1], device=x.device) // 64
    return m[..., at] + codes * s[..., at]


def _index(D, place):
    at = [[place(D, p, c) for c in range(D)] for p in range(16)]
    return torch.tensor([[x[0] for x in r] for r in at]), torch.tensor([[x[1] for x in r] for r in at])


def _scale_index(D, value):
    return torch.tensor([[scale_place(D, p, c // 64, value) for c in range(D)] for p in range(16)])


def pool_rows(pool, D):
    """K and V rows of a pool [blocks, nkv, bs / 16, tile] in 64 bits: [blocks, bs, nkv, D]."""
    nb, nkv, nt, _ = pool.shape
    out = []
    for place, value in ((k_place, 0), (v_place, 1)):
        byte, shift = (x.to(pool.device) for x in _index(D, place))
        at = _scale_index(D, value).to(pool.device)
        u = (pool[..., byte].long() >> shift) & 15
        half = [(pool[..., at + i].to(torch.int32) | pool[..., at + i + 1].to(torch.int32) << 8).to(torch.int16)
                .view(torch.float16).double() for i in (0, 2)]
        rows = half[1] + u * half[0]
        out.append(rows.reshape(nb, nkv, nt * 16, D).transpose(1, 2))
    return out


def fill_pool(k, v):
    """A pool that holds k and v [blocks, bs, nkv, D]; padding is left zero."""
    nb, bs, nkv, D = k.shape
    pool = torch.zeros(nb, nkv, bs // 16, tile_bytes(D), dtype=torch.uint8, device=k.device)
    for x, place, value in ((k, k_place, 0), (v, v_place, 1)):
        u, s, m = quantise(x.double().transpose(1, 2).reshape(nb, nkv, bs // 16, 16, D))
        byte, shift = _index(D, place)
        for c in range(D):
            for p in range(16):
                pool[..., int(byte[p, c])] |= (u[..., p, c] << int(shift[p, c])).to(torch.uint8)
        for p in range(16):
            for g in range(s.shape[-1]):
                raw = torch.stack((s[..., p, g], m[..., p, g]), -1).half().view(torch.uint8)
                at = scale_place(D, p, g, value)
                pool[..., at:at + 4] = raw
    return pool


def rotate(x, at, inv_freq):
    """x [..., D] in 64 bits, positions `at` (of x's leading shape or broadcast to it)."""
    half = len(inv_freq)
    a = at.double()[..., None] * torch.tensor(inv_freq, dtype=torch.float64, device=x.device)
    x1, x2 = x[..., :half].double(), x[..., half:2 * half].double()
    return torch.cat((x1 * torch.cos(a) - x2 * torch.sin(a), x2 * torch.cos(a) + x1 * torch.sin(a),
                      x[..., 2 * half:].double()), -1)


def append(q, k, v, tables, lens, counts, positions, inv_freq, bs, num_blocks):
    """What an append leaves: rotated q, and a list of (block, slot, k row [nkv, D], v row) in 64 bits."""
    B, S = k.shape[:2]
    qo = None if q is None else q.double().clone()
    rows = []
    for b in range(B):
        n = S if counts is None else max(0, min(S, int(counts[b])))
        first = int(lens[b]) - n
        turn = first if positions is None else int(positions[b])
        for i in range(n):
            at = torch.tensor(turn + i, device=k.device)
            if qo is not None:
                qo[b, i] = rotate(q[b, i], at, inv_freq)
            pos = first + i
            if 0 <= pos < tables.shape[1] * bs and 0 <= int(tables[b, pos // bs]) < num_blocks:
                rows.append((int(tables[b, pos // bs]), pos % bs, rotate(k[b, i], at, inv_freq), v[b, i].double()))
    return qo, rows


def bounds(keys):
    """keys [rows, nkv, D] (as 32-bit numbers): codes [nkv, 2, D] and scales [nkv]."""
    keys = keys.float().double()
    codes = torch.zeros(keys.shape[1], 2, keys.shape[2], dtype=torch.int8)
    scale = torch.ones(keys.shape[1])
    for h in range(keys.shape[1]):
        x = keys[:, h].cpu()
        if not torch.isfinite(x).all():
            scale[h] = math.inf
            continue
        top = float(x.abs().max())
        e = 0
        if top > 0:
            e = -126
            while 127 * 2.0 ** e < top:
                e += 1
        codes[h, 0] = torch.floor(x.amin(0) / 2.0 ** e).to(torch.int8)
        codes[h, 1] = torch.ceil(x.amax(0) / 2.0 ** e).to(torch.int8)
        scale[h] = 2.0 ** e
    return codes, scale


def score(q, codes, scale):
    """q [group, D], codes [blocks, 2, D], scale [blocks]: the blocks' scores."""
    q = q.double()
    parts = torch.stack((q.clamp(max=0).sum(0), q.clamp(min=0).sum(0)))
    top = float(parts.abs().max())
    if not math.isfinite(top):
        parts = torch.zeros_like(parts)
    elif top > 0:
        e = -200
        while 32767 * 2.0 ** e < top:
            e += 1
        parts = torch.round(parts / 2.0 ** e)
    total = (codes.double() * parts).sum((1, 2))
    return torch.where(torch.isinf(scale), math.inf, total.float() * scale)


def choose(scores, n, first, last):
    """Chosen of the blocks with these scores (a list), ascending."""
    nb = len(scores)
    if nb <= n:
        return list(range(nb))
    mid = sorted(range(first, nb - last), key=lambda i: (-scores[i], i))[: n - first - last]
    return sorted(list(range(first)) + mid + list(range(nb - last, nb)))


def attend(q, k, v, ok):
    """q [R, D], k and v [n, D], ok bool [n]: outputs and sum p|v| in 64 bits; zeros if nothing is seen."""
    if not bool(ok.any()):
        z = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
        return z, z
    p = torch.softmax(q.double() @ k[ok].double().T / math.sqrt(q.shape[1]), -1)
    return p @ v[ok].double(), p @ v[ok].double().abs()


def decode(q, k, v, tables, lens, window=0, sinks=0, blocks=None):
    """q [B, nq, D], row pools [blocks, bs, nkv, D] in 64 bits: outputs and sum p|v|.  blocks [B, nkv, n] or None."""
    B, nq, D = q.shape
    nb, bs, nkv, _ = k.shape
    out = torch.zeros(B, nq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for b in range(B):
        n = max(0, min(int(lens[b]), tables.shape[1] * bs))
        for h in range(nkv):
            if blocks is None:
                pos = [t for t in range(n) if window == 0 or t < sinks or n - t <= window]
            else:
                pos = [j * bs + i for j in blocks[b, h].tolist()[:-(-n // bs)] if 0 <= j < tables.shape[1] for i in range(bs)
                       if j * bs + i < n]
            at = [(int(tables[b, t // bs]), t % bs) for t in pos]
            at = [(x, y) for x, y in at if 0 <= x < nb]
            if not at:
                continue
            x, y = (torch.tensor(i, device=q.device) for i in zip(*at))
            hs = slice(h * nq // nkv, (h + 1) * nq // nkv)
            out[b, hs], mag[b, hs] = attend(q[b, hs], k[x, y, h], v[x, y, h],
                                            torch.ones(len(at), dtype=torch.bool, device=q.device))
    return out, mag
