"""The cache in 4 bits restated plainly: rows bit by bit, attention over the values they stand for in float64, head norms and rotation.

A row keeps its entries in groups of 32 with a scale s and a centre c (bfloat16): s = (max - min) / 15, c = min + 8 s, and for each entry a
number n from 0 to 15, which stands for c + s (n - 8)."""

import torch

F64 = torch.float64


def groups(hd):
    return (hd + 31) // 32


def bit_of(which, d, hd):
    """The first bit of entry d's number in a row."""
    G, g, r = groups(hd), d // 32, d % 32
    return 32 * (r // 8 * G + g) + 4 * (r % 8) if which == "k" else 16 * (r // 4 * G + g) + 4 * (r % 4)


def quantise(x):
    """(numbers int, s, c) of float32 rows [..., hd] in 32-bit steps; s and c float32 [..., G], numbers [..., hd]."""
    hd = x.shape[-1]
    n, ss, cs = torch.empty(x.shape, dtype=torch.int64), [], []
    for g in range(groups(hd)):
        part = x[..., 32 * g:32 * g + 32]
        lo, hi = part.amin(-1), part.amax(-1)
        s = ((hi - lo) / 15).to(torch.bfloat16).float()
        s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
        c = (lo + 8 * s).to(torch.bfloat16).float()
        inverse = torch.where(s > 0, 1 / s, torch.zeros_like(s))
        n[..., 32 * g:32 * g + 32] = (torch.round((part - c[..., None]) * inverse[..., None]) + 8).clamp(0, 15).long()
        ss.append(s)
        cs.append(c)
    return n, torch.stack(ss, -1), torch.stack(cs, -1)


def pack(which, n, s, c):
    """uint8 rows [..., 20 G]; numbers that stand for nothing are 8."""
    hd, G = n.shape[-1], groups(n.shape[-1])
    out = torch.zeros((*n.shape[:-1], 20 * G), dtype=torch.int64)
    for d in range(32 * G):
        bit = bit_of(which, d, hd)
        out[..., bit // 8] += (n[..., d] if d < hd else torch.full(n.shape[:-1], 8)) << (bit % 8)
    pairs = torch.stack([s, c], -1).to(torch.bfloat16).contiguous().view(torch.uint8).reshape(*n.shape[:-1], 4 * G)
    out[..., 16 * G:] = pairs.long()
    return out.to(torch.uint8)


def unpack(which, rows, hd):
    """float64 values [..., hd] of uint8 rows (CPU)."""
    G = groups(hd)
    params = rows[..., 16 * G:].contiguous().view(torch.bfloat16).to(F64).reshape(*rows.shape[:-1], G, 2)
    out = torch.empty((*rows.shape[:-1], hd), dtype=F64)
    for d in range(hd):
        bit = bit_of(which, d, hd)
        n = (rows[..., bit // 8].long() >> (bit % 8)) & 15
        out[..., d] = params[..., d // 32, 1] + params[..., d // 32, 0] * (n - 8)
    return out


def prepare_heads(rows, bias, q_norm, k_norm, eps, positions, cos, sin, nq, nkv, hd, rotate=True, dtype=F64):
    """Queries, keys and values [tokens, heads, hd] behind bias, norms and rotation, in ``dtype``."""
    x = rows.to(dtype)
    if bias is not None:
        x = x + bias.to(dtype)
    q, k, v = x.view(-1, nq + 2 * nkv, hd).split([nq, nkv, nkv], dim=1)

    def norm(t, w):
        return t if w is None else t / ((t * t).mean(-1, keepdim=True) + eps).sqrt() * w.to(dtype)

    def turn(t):
        if not rotate:
            return t
        c, s = cos[positions.long()].to(dtype)[:, None], sin[positions.long()].to(dtype)[:, None]
        a, b = t[..., :hd // 2], t[..., hd // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    return turn(norm(q, q_norm)), turn(norm(k, k_norm)), v


def attention(q, keys, values, positions, seq, scale, window=0, softcap=0.0, sinks=None, slopes=None):
    """q [tokens, nq, hd]; keys and values: lists of [n, nkv, hd] per request. Returns (out float64 [tokens, nq, hd], the largest sum of
    absolute products behind a score, the largest value)."""
    out = torch.zeros(q.shape, dtype=F64)
    nq = q.shape[1]
    largest = 0.0
    for t in range(q.shape[0]):
        r = int(seq[t])
        if r < 0:
            continue
        p = int(positions[t])
        lo = max(0, p - window + 1) if window else 0
        for h in range(nq):
            kv = h // (nq // keys[r].shape[1])
            k, v = keys[r][lo:p + 1, kv].to(F64), values[r][lo:p + 1, kv].to(F64)
            s = k @ q[t, h].to(F64) * scale
            largest = max(largest, float((k.abs() @ q[t, h].to(F64).abs()).max()) * scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[h]) * (p - torch.arange(lo, p + 1, dtype=F64))
            e = torch.cat([s, sinks[h:h + 1].to(F64)]) if sinks is not None else s
            w = torch.softmax(e, 0)[:len(s)]
            out[t, h] = w @ v
    return out, largest, max(float(v.abs().max()) for v in values)
