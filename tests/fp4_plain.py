"""Four-bit blocks, the cache in them, attention over it and products with them, in plain 64-bit operations on the CPU: what the kernels are
compared with.  Nothing here comes from the package."""
import math

import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantized(x):
    """x [..., 32 B] -> codes [..., B, 32], scale bytes [..., B]: by the definition, every magnitude's distance looked at."""
    x = x.double().unflatten(-1, (-1, 32))
    a = x.abs()
    top = a.amax(-1)                                        # (NaN if there is one)
    finite = torch.isfinite(top)
    m, e = torch.frexp(torch.where(finite & (top > 0), top, torch.ones_like(top)))     # top = m 2^e, 0.5 <= m < 1
    byte = e - 1 + 127 - 2 + (2 * m > 1.75).int()
    byte = torch.where(top > 0, byte.clamp(2, 252), torch.full_like(byte, 2))
    unit = torch.pow(2.0, (byte - 127).double()).unsqueeze(-1)
    scaled = a.nan_to_num(0.0, 0.0, 0.0) / unit
    distance = (scaled.unsqueeze(-1) - MAGNITUDES).abs()
    best = distance.amin(-1, keepdim=True)
    # of two at the same distance the even code
    code = (distance == best).int() * torch.tensor([2, 1, 2, 1, 2, 1, 2, 1], dtype=torch.int32)
    code = code.argmax(-1) + 8 * torch.signbit(x).int()
    return code.byte(), torch.where(finite, byte, torch.full_like(byte, 255)).byte()


def values(codes, scales):
    sign = torch.where(codes >= 8, -1.0, 1.0).double()
    unit = torch.where(scales == 255, torch.nan, torch.pow(2.0, scales.double() - 127))
    return (sign * MAGNITUDES[(codes & 7).long()] * unit.unsqueeze(-1)).flatten(-2)


def rounded(x):
    """x as the values of the four-bit blocks nearest to it"""
    return values(*quantized(x))


def key_place(slot):
    return 16 * (slot // 16) + 4 * (slot % 4) + slot // 4 % 4


def put(k_pages, v_pages, slot, kc, ks, vc, vs):
    """One token into pages (CPU tensors): codes [G, B, 32], scale bytes [G, B]."""
    P, G, B, _, page = k_pages.shape
    at, off = slot // page, slot % page
    flat = k_pages[at].view(G, B, 17 * page)
    flat[:, :, off * 16:off * 16 + 16] = kc[..., 0::2] | (kc[..., 1::2] << 4)
    flat[:, :, 16 * page + key_place(off)] = ks
    v_pages[at, :, :, :16, off] = vc[..., :16] | (vc[..., 16:] << 4)
    v_pages[at, :, :, 16, off] = vs


def get(k_pages, v_pages, slot):
    """[G, 32 B] keys and values of one slot"""
    P, G, B, _, page = k_pages.shape
    at, off = slot // page, slot % page
    flat = k_pages[at].reshape(G, B, 17 * page)
    two = flat[:, :, off * 16:off * 16 + 16]
    k = values(torch.stack([two & 15, two >> 4], -1).flatten(-2), flat[:, :, 16 * page + key_place(off)])
    two = v_pages[at, :, :, :16, off]
    return k, values(torch.cat([two & 15, two >> 4], -1), v_pages[at, :, :, 16, off])


def turned(x, cos, sin):
    """Heads [n, h, D] turned in pairs (i, i + D / 2) as 32-bit arithmetic does it: one product rounded, the other and the sum together."""
    half = x.shape[-1] // 2
    x0, x1 = x[..., :half].float(), x[..., half:].float()
    c, s = cos.float()[:, None], sin.float()[:, None]
    return torch.cat([(x0.double() * c.double() - (x1 * s).double()).float(), (x1.double() * c.double() + (x0 * s).double()).float()], -1)


def attention(q, q_start, q_len, pos0, tables, k_pages, v_pages, n_heads, scale, window=0):
    """(results, sum of p |v|, largest sum of |q k| scale of a row's keys), 64-bit [n, H, D], [n, H, D], [n, H]; rows of no request are NaN."""
    P, G, B, _, page = k_pages.shape
    D, rep = 32 * B, n_heads // G
    n = q.shape[0]
    q = q.double().view(n, n_heads, D)
    out, size, reach = torch.full_like(q, math.nan), torch.zeros_like(q), torch.zeros(n, n_heads, dtype=torch.float64)
    for s in range(len(q_len)):
        keys = max(0, pos0[s] + q_len[s]) if q_len[s] else 0
        k, v = torch.zeros(2, G, keys, D, dtype=torch.float64)
        known = torch.zeros(keys, dtype=torch.bool)
        for t in range(keys):
            pg = int(tables[s, t // page]) if t // page < tables.shape[1] else -1
            if 0 <= pg < P:
                k[:, t], v[:, t] = get(k_pages, v_pages, pg * page + t % page)
                known[t] = True
        for i in range(q_len[s]):
            row, p = q_start[s] + i, pos0[s] + i
            seen = known & (torch.arange(keys) <= p)
            if window:
                seen &= torch.arange(keys) > p - window
            if not seen.any():
                out[row] = 0
                continue
            for h in range(n_heads):
                ks, vs = k[h // rep, seen], v[h // rep, seen]
                w = torch.softmax(ks @ q[row, h] * scale, 0)
                out[row, h] = w @ vs
                size[row, h] = w @ vs.abs()
                reach[row, h] = (ks.abs() @ q[row, h].abs()).max() * scale
    return out, size, reach
